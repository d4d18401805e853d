"""Argument checks of the distillation calls (all before any CUDA call; nothing is launched), and the FP64 oracle of their tests against
autograd and against differences."""
import ctypes as C

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from distill_case import bits_of, case, oracle


@pytest.fixture(scope="module")
def pkg():
    entry.build()
    return entry.load_package()


def good(pkg, **changes):
    a = pkg.DistillArgs()
    a.struct_bytes = C.sizeof(pkg.DistillArgs)
    a.rows, a.vocab, a.dtype, a.top, a.temperature = 4, 1000, 1, 20, 1.0
    a.logits, a.logits_stride, a.grad, a.grad_stride = 1 << 20, 1000, 1 << 24, 1000
    a.teacher_ids, a.ids_stride, a.teacher_values, a.values_stride = 1 << 12, 20, 1 << 13, 20
    a.loss, a.stats, a.status = 1 << 14, 1 << 15, 1 << 16
    for k, v in changes.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("call", ["loss", "grad", "loss_grad"])
@pytest.mark.parametrize("changes,message", [
    ({"struct_bytes": 16}, "ABI"), ({"rows": 0}, "out of range"), ({"vocab": 0}, "out of range"), ({"rows": 1 << 28}, "out of range"),
    ({"vocab": 131073, "logits_stride": 1 << 18, "grad_stride": 1 << 18}, "out of range"), ({"dtype": 3}, "FP32, BF16 or FP16"),
    ({"teacher_dtype": 1}, "FP32 or FP64"), ({"top": 0}, "top"), ({"top": 257, "ids_stride": 300, "values_stride": 300}, "top"),
    ({"tail": 2}, "tail"), ({"reserved": 1}, "tail"), ({"temperature": 0.0}, "temperature"), ({"temperature": float("nan")}, "temperature"),
    ({"temperature": float("inf")}, "temperature"), ({"tail": 1, "temperature": 2.0}, "temperature 1"), ({"logits": None}, "logits"),
    ({"logits_stride": 999}, "logits"), ({"logits_stride": 0}, "logits"), ({"logits": (1 << 20) + 1}, "logits"), ({"teacher_ids": None}, "teacher"),
    ({"teacher_values": None}, "teacher"), ({"ids_stride": 19}, "teacher"), ({"values_stride": 19}, "teacher"), ({"teacher_ids": 4098}, "teacher"),
    ({"teacher_values": 8196, "teacher_dtype": 3}, "teacher"), ({"mask": 1 << 12, "mask_stride": 31}, "mask"), ({"stats": (1 << 15) + 8}, "stats")])
def test_arguments_are_refused_before_any_launch(pkg, call, changes, message):
    a = good(pkg, **changes)
    if call == "loss":
        a.grad = None
    assert getattr(pkg.lib(), "ds41_b200_distill_" + call)(C.byref(a), None) == 1
    assert message in pkg.last_error(), pkg.last_error()


@pytest.mark.parametrize("call,changes,message", [
    ("loss", {"grad": None, "loss": None}, "loss"), ("loss", {"grad": None, "status": None}, "status"), ("loss", {}, "belong"),
    ("loss", {"grad": None, "row_scale": 1 << 12}, "belong"), ("grad", {"stats": None}, "stats"), ("grad", {"grad": None}, "grad"),
    ("grad", {"grad_stride": 999}, "grad"), ("loss_grad", {"grad": (1 << 24) + 1}, "grad"), ("loss_grad", {"grad": (1 << 20) + 2}, "overlaps"),
    ("loss_grad", {"grad": 1 << 20, "grad_stride": 1008}, "overlaps"), ("loss_grad", {"loss": None}, "loss"), ("loss_grad", {"status": None}, "status")])
def test_what_each_call_needs(pkg, call, changes, message):
    assert getattr(pkg.lib(), "ds41_b200_distill_" + call)(C.byref(good(pkg, **changes)), None) == 1
    assert message in pkg.last_error(), pkg.last_error()
    assert getattr(pkg.lib(), "ds41_b200_distill_" + call)(None, None) == 1


def test_tensors_without_a_device_are_refused(pkg):
    z, ids, v = torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1)
    for call in (pkg.distill_loss, pkg.distill_loss_grad, lambda *a: pkg.distill_grad(*a, torch.zeros(2, 4))):
        with pytest.raises(ValueError):
            call(z, ids, v)


@pytest.mark.parametrize("tail,temperature", [(False, 1.0), (False, 2.5), (True, 1.0)])
@pytest.mark.parametrize("share", [None, 0.3])
def test_the_oracle_against_autograd_and_differences(tail, temperature, share):
    c = case(5, 4, 200, torch.float32, 9, tail, share)
    loss, stats, grad, status, _ = oracle(c["z"], c["ids"], c["values"], temperature, tail, c.get("mask"), c["scale"])
    assert status.tolist() == [0] * 4 and loss[3] == 0 and (grad[3] == 0).all()
    for r in range(3):
        z = torch.tensor(c["z"][r], dtype=torch.float64, requires_grad=True)
        allowed = torch.from_numpy(bits_of(c["mask"][r:r + 1], 200)[0]) if share else torch.ones(200, dtype=torch.bool)
        keep = [(int(i), float(v)) for i, v in zip(c["ids"][r], c["values"][r]) if 0 <= i < 200 and allowed[i]]
        idx, val = torch.tensor([i for i, _ in keep]), torch.tensor([v for _, v in keep], dtype=torch.float64)
        log_q = (z / temperature).masked_fill(~allowed, -np.inf).log_softmax(0)
        if tail:
            p, rest = val.exp(), 1 - val.exp().sum()
            out = allowed.clone()
            out[idx] = False
            want = (p * (p.log() - log_q[idx])).sum() + rest * (rest.log() - log_q[out].logsumexp(0))
        else:
            p = (val / temperature).softmax(0)
            want = temperature ** 2 * (p * (p.log() - log_q[idx])).sum()
        (g,) = torch.autograd.grad(c["scale"][r].item() * want, z)
        assert abs(loss[r] - want.item()) < 1e-12 and np.abs(grad[r] - g.numpy()).max() < 1e-13
        for i in [int(idx[0]), int(allowed.nonzero()[-1])]:      # differences: the third derivative's term is below h^2
            step = np.zeros((1, 200))
            step[0, i] = 1e-4
            f = [oracle(c["z"][r:r + 1] + d, c["ids"][r:r + 1], c["values"][r:r + 1], temperature, tail,
                        c["mask"][r:r + 1] if share else None)[0][0] for d in (step, -step)]
            assert abs((f[0] - f[1]) / 2e-4 * c["scale"][r] - grad[r, i]) < 1e-7


def test_rows_of_the_oracle_by_hand():
    z = np.log(np.float64([[1.0, 2.0, 5.0]]))
    loss, stats, grad, status, _ = oracle(z, np.int32([[2, 1]]), np.log([[0.25, 0.25]]), tail=True)
    assert np.allclose(loss, 0.25 * np.log(0.25 / 0.625) + 0.25 * np.log(1) + 0.5 * np.log(0.5 / 0.125))
    assert np.allclose(grad, [[0.125 - 0.5, 0.0, 0.625 - 0.25]]) and np.allclose(np.exp(stats[0, [1, 3]]), [8 / 5, 1])
    loss, _, grad, status, _ = oracle(z, np.int32([[2, 2]]), np.log([[0.25, 0.25]]))       # the same id twice
    assert np.allclose(loss, -np.log(0.625)) and np.allclose(grad, [[0.125, 0.25, -0.375]])
