"""The distillation on rows of finite logits far from zero, as a model's own mask or a constraint leaves them (-1e9 to the type's lowest),
at every temperature that is taken, against the FP64 definition."""
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


def run(pkg, c, dtype, temperature, tail, want, order):
    view, _, t = gpu({k: v[order] for k, v in c.items()}, dtype)
    more = {"temperature": temperature, "tail": tail, "mask": t["mask"]}
    loss, stats, status = pkg.distill_loss(view, t["ids"], t["values"], **more)
    compare({"loss": loss, "stats": stats, "status": status}, want, dtype, temperature, order)
    loss, grad, status = pkg.distill_loss_grad(view, t["ids"], t["values"], **more)
    compare({"loss": loss, "grad": grad, "status": status}, want, dtype, temperature, order)
    compare({"grad": pkg.distill_grad(view, t["ids"], t["values"], stats, **more)}, want, dtype, temperature, order)


LOW = {"fp32": [-1e9, -1e10, -1e12, -1e20, -1e30, -3.4028234663852886e38], "bf16": [-1e9, -1e10, -1e12, -1e20, -1e30, -3.3895313892515355e38],
       "fp16": [-1e4, -6e4, -65504.0]}


def rows_with(values, vocab, dtype, tail, share, teacher_seed=31):
    """For every value a row that holds it: everywhere outside the list; in its first half; in its second half; in all vectors of some
    threads, whichever kernel and alignment; at every other id by chance; everywhere; at five ids; with its sign changed at some ids."""
    kinds = 8
    c = case(teacher_seed, kinds * len(values), vocab, dtype, 24, tail, share)
    del c["scale"]
    rng, at = np.random.default_rng(32), np.arange(vocab)
    for i, m in enumerate(values):
        for kind in range(kinds):
            r = kinds * i + kind
            outside = np.ones(vocab, bool)
            outside[c["ids"][r][(c["ids"][r] >= 0) & (c["ids"][r] < vocab)]] = False
            where = [outside, outside & (at < vocab // 2), outside & (at >= vocab // 2), outside & (at // 8 % 64 < 9), outside & (rng.random(vocab) < 0.5),
                     np.ones(vocab, bool), outside & np.isin(at, rng.integers(0, vocab, 5)), outside & (rng.random(vocab) < 0.01)][kind]
            c["z"][r, where] = m if kind < 7 else min(-m, 1e30)
    c["z"] = torch.from_numpy(c["z"]).to(dtype).float().numpy()
    assert np.isfinite(c["z"]).all()
    return c


@pytest.mark.parametrize("temperature,tail", [(0.1, False), (1.0, False), (1.0, True), (50.0, False), (1000.0, False)])
@pytest.mark.parametrize("dtype,vocab,share,times", [("fp32", 20011, None, 1), ("fp32", 20011, 0.4, 1), ("fp32", 20011, None, 4),
                                                     ("bf16", 40001, None, 1), ("bf16", 40001, 0.4, 1), ("bf16", 40001, None, 4),
                                                     ("fp16", 1031, None, 1), ("fp16", 1031, 0.4, 40), ("fp16", 40001, None, 8)])
def test_finite_logits_far_from_zero(pkg, dtype, vocab, share, times, temperature, tail):
    t = TYPES[dtype]
    c = rows_with(LOW[dtype], vocab, t, tail, share)
    want = oracle(c["z"], c["ids"], c["values"], temperature, tail, c.get("mask"))
    assert not want[3].any() and np.isfinite(want[0]).all() and np.isfinite(want[2]).all()
    order = np.random.default_rng(33).permutation(np.tile(np.arange(len(c["z"])), times))
    run(pkg, c, t, temperature, tail, want, order)


@pytest.mark.parametrize("temperature", [0.01, 1.0, 30.0, 700.0])
@pytest.mark.parametrize("exponent", [8, 16, 20, 23, 24, 25, 26, 28, 30, 31, 32, 34, 40, 80, 120])
@pytest.mark.parametrize("vocab,share,rows", [(20011, None, 8), (20011, 0.5, 8), (20011, None, 160)])
def test_maxima_that_rise_across_powers_of_two(pkg, vocab, share, rows, exponent, temperature):
    """Logits whose product with log2(e) / T climbs along the row from a little beyond a power of two to a little this side of it, or
    across its negative: every thread's running maximum crosses the line, in steps that are as small as FP32 has them."""
    t = torch.float32
    c = case(34, 8, vocab, t, 16, False, share)
    del c["scale"]
    line = 2.0 ** exponent * temperature * np.log(2.0)
    if line > 3e38:
        pytest.skip("beyond FP32")
    step = np.spacing(np.float32(line)).astype(np.float64)
    climb = np.arange(vocab) / vocab - 0.5
    for r in range(8):
        # the whole way is a few powers of two, or two steps where those are more
        way = max([1.0, 6.0, 40.0, 4.0][r % 4] * temperature, 2 * step)
        c["z"][r] = ((-line if r < 4 else line) + way * climb).astype(np.float32)
        c["z"][r, c["ids"][r][c["ids"][r] < vocab]] += np.float32(way)
    assert np.isfinite(c["z"]).all()
    want = oracle(c["z"], c["ids"], c["values"], temperature, False, c.get("mask"))
    run(pkg, c, t, temperature, False, want, np.arange(rows) % 8)
