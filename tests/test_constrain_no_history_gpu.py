"""Histories without a single token: the lengths beside them are looked at all the same."""
import pytest
import torch

import __graft_entry__ as entry

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    entry.build()
    return entry.load_package()


@pytest.mark.parametrize("lens,status", [([0, 0, 0, 0], [0, 0, 0, 0]), ([0, 1, -1, 65535], [0, -7, -7, -7])])
def test_lengths_of_a_history_without_tokens(pkg, lens, status):
    x = torch.randn(4, 3000, device="cuda")
    history = torch.zeros(4, 0, dtype=torch.int32, device="cuda")
    out, st = pkg.constrain_logits(x, history=history, history_len=torch.tensor(lens, dtype=torch.int32, device="cuda"), repetition=1.3)
    assert st.cpu().tolist() == status
    for r, s in enumerate(status):
        assert torch.equal(out[r], x[r]) if s == 0 else out[r].isnan().all()


def test_one_sequence_and_its_drafts(pkg):
    x = torch.randn(3, 500, device="cuda")
    drafts, history = torch.tensor([[7, 499]], dtype=torch.int32, device="cuda"), torch.zeros(1, 0, dtype=torch.int32, device="cuda")
    more = {"presence": 1.0, "draft_ids": drafts, "rows_per_sequence": 3}
    want, _ = pkg.constrain_logits(x, **more)
    out, st = pkg.constrain_logits(x, history=history, history_len=torch.zeros(1, dtype=torch.int32, device="cuda"), **more)
    assert torch.equal(out, want) and st.cpu().tolist() == [0, 0, 0]
    assert torch.equal(out[2, [7, 499]], x[2, [7, 499]] - 1.0) and torch.equal(out[0], x[0])
    out, st = pkg.constrain_logits(x, history=history, history_len=torch.ones(1, dtype=torch.int32, device="cuda"), **more)
    assert out.isnan().all() and st.cpu().tolist() == [-7, -7, -7]
