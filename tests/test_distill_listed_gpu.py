"""Rows whose list names every id that is allowed: nothing is outside the list, at any temperature, and ids that are not allowed get
gradient 0."""
import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from distill_bounds import compare
from distill_case import TYPES, case, gpu, oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    entry.build()
    return entry.load_package()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab,rows,masked", [(900, 6, True), (40001, 6, True), (900, 6, False), (40001, 6, False), (40001, 160, False)])
@pytest.mark.parametrize("temperature", [1e-3, 1.0, 49.0, 50.0, 64.0, 100.0, 250.0, 333.0, 500.0, 777.0, 1000.0])
def test_lists_that_name_every_allowed_id(pkg, dtype, vocab, rows, masked, temperature):
    t = TYPES[dtype]
    c = case(41, 6, vocab, t, 20)
    c["scale"] = np.float32([1.0, 0.5, -2.0, 1e-4, 300.0, 1.0])
    c["ids"][5, :] = -1                                   # (and one that names a single id)
    c["ids"][5, 0], c["values"][5, 0] = vocab - 1, -0.5
    keep = np.zeros((6, vocab), bool)
    for r in range(6):
        keep[r, c["ids"][r][c["ids"][r] >= 0]] = True
    if masked:
        bits = np.zeros((6, (vocab + 31) // 32 * 32), bool)
        bits[:, :vocab] = keep
        c["mask"] = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
    else:
        c["z"][~keep] = -np.inf
    want = oracle(c["z"], c["ids"], c["values"], temperature, False, c.get("mask"), c["scale"])
    plain = oracle(c["z"], c["ids"], c["values"], temperature, False, c.get("mask"))
    assert not want[3].any() and not want[2][~keep].any()
    order = np.arange(rows) % 6
    view, _, x = gpu({k: v[order] for k, v in c.items()}, t)
    more = {"temperature": temperature, "mask": x["mask"]}
    loss, stats, status = pkg.distill_loss(view, x["ids"], x["values"], **more)
    assert status.cpu().tolist() == [0] * rows and torch.isinf(stats[:, 2:]).all()
    compare({"loss": loss}, plain, t, temperature, order)
    loss, grad, status = pkg.distill_loss_grad(view, x["ids"], x["values"], row_scale=x["scale"], **more)
    compare({"loss": loss, "grad": grad, "status": status}, want, t, temperature, order)
    assert not grad.float().cpu().numpy()[~keep[order]].any()
    compare({"grad": pkg.distill_grad(view, x["ids"], x["values"], stats, row_scale=x["scale"], **more)}, want, t, temperature, order)
