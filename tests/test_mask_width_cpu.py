"""Bitmasks with fewer words a row than the vocabulary needs are refused before any launch, whatever the stride of their rows: the
words behind a row's last column are not the mask's.  Nothing is launched here: the call that a launch would make is only recorded."""
import pytest
import torch

import __graft_entry__ as entry


@pytest.fixture(scope="module")
def pkg():
    entry.build()
    return entry.load_package()


class OnDevice:
    """A tensor that says it lies on a GPU."""
    is_cuda = True
    device = torch.device("cuda", 0)

    def __init__(self, tensor):
        self.tensor = tensor

    def __getattr__(self, name):
        return getattr(self.tensor, name)


VOCAB, ROWS = 1000, 3       # 32 words a row


def calls(pkg, mask):
    z, ids = OnDevice(torch.zeros(ROWS, VOCAB)), OnDevice(torch.zeros(ROWS, 4, dtype=torch.int32))
    values, out, rows = OnDevice(torch.zeros(ROWS, 4)), OnDevice(torch.zeros(ROWS, VOCAB)), OnDevice(torch.zeros(ROWS))
    stats, status = OnDevice(torch.zeros(ROWS, 4)), OnDevice(torch.zeros(ROWS, dtype=torch.int32))
    return {"constrain": lambda: pkg.constrain_logits(z, mask=mask, out=out, status=status),
            "loss": lambda: pkg._distill("ds41_b200_distill_loss", z, ids, values, 1.0, False, mask, None, rows, stats, None, status),
            "grad": lambda: pkg._distill("ds41_b200_distill_grad", z, ids, values, 1.0, False, mask, None, None, stats, out),
            "loss_grad": lambda: pkg._distill("ds41_b200_distill_loss_grad", z, ids, values, 1.0, False, mask, None, rows, None, out, status)}


@pytest.fixture
def launches(pkg, monkeypatch):
    seen = []
    monkeypatch.setattr(pkg, "_launch", lambda device, what, fn, args: seen.append(args._obj))
    return seen


@pytest.mark.parametrize("call", ["constrain", "loss", "grad", "loss_grad"])
@pytest.mark.parametrize("columns", [0, 1, 31])
@pytest.mark.parametrize("wide", [False, True])
def test_a_mask_with_too_few_words_is_refused(pkg, launches, call, columns, wide):
    mask = torch.zeros(ROWS, 64 if wide else columns, dtype=torch.int32)[:, :columns]
    with pytest.raises(RuntimeError, match="mask"):
        calls(pkg, OnDevice(mask))[call]()
    assert not launches


@pytest.mark.parametrize("call", ["constrain", "loss", "grad", "loss_grad"])
@pytest.mark.parametrize("columns,stride", [(32, 32), (32, 40), (33, 33), (40, 64)])
def test_a_mask_of_enough_words_is_taken_at_its_stride(pkg, launches, call, columns, stride):
    mask = torch.zeros(ROWS, stride, dtype=torch.int32)[:, :columns]
    calls(pkg, OnDevice(mask))[call]()
    assert [a.mask_stride for a in launches] == [stride] and launches[0].mask == mask.data_ptr()
