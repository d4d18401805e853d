"""The distillation's definition in FP64 (NumPy, row by row, softmax over all allowed ids), inputs for it, and how far a result in
FP32 may be off.

The student's sum over the ids outside the list is the only one in FP32.  With a the distance of an id from the row's maximum in powers
of two: the difference, the factor and the product are rounded (3 * 2^-24 * a, relative to the power's exponent, ln 2 of it in the
power), the power itself is 2 ulp off (2^-22), and a thread adds up to 66 of them before a tree of 17 (83 * 2^-24).  Ids beyond a = 27
(ln of 131072 ids and ten more) hold less than 2^-10 of the sum.  Together 3 * 27 * 0.7 * 2^-24 + 2^-22 + 83 * 2^-24 < 9e-6 = SUM, the
relative error of the sum and the absolute one of its logarithm."""
import numpy as np
import torch

from constrain_case import TYPES, bits_of, words

SUM = 9e-6
f8 = np.float64


def oracle(z, ids, values, temperature=1.0, tail=False, mask=None, scale=None):
    """(loss, stats, grad, status) in FP64, and bound [rows, vocab] of q_i + rest * r_i, the scale of a gradient's error."""
    rows, vocab = z.shape
    z = z.astype(f8)
    loss, stats, grad, status = np.zeros(rows), np.zeros((rows, 4)), np.zeros((rows, vocab)), np.zeros(rows, np.int32)
    size = np.zeros((rows, vocab))
    for r in range(rows):
        s = 1.0 if scale is None else f8(scale[r])
        if s == 0:
            continue
        allowed = (bits_of(mask[r:r + 1], vocab)[0] if mask is not None else np.ones(vocab, bool)) & ~(z[r] == -np.inf)
        entries = [(int(i), f8(v)) for i, v in zip(ids[r], values[r]) if 0 <= i < vocab]
        count = [(i, v) for i, v in entries if allowed[i]]
        if any(not v < np.inf for _, v in entries) or any(not z[r, i] < np.inf for i, _ in count):
            status[r], loss[r], stats[r], grad[r] = -1, np.nan, np.nan, np.nan
            continue
        target, on_list = np.zeros(vocab), np.zeros(vocab, bool)
        most = max([v for _, v in count], default=0.0)
        for i, v in count:
            target[i] += np.exp(v) if tail else np.exp((v - most) / temperature) if most > -np.inf else 0.0
            on_list[i] = True
        named = sum(np.exp(v) for _, v in entries)
        if tail and named > 1.01:
            status[r], loss[r], stats[r], grad[r] = -10, np.nan, np.nan, np.nan
            continue
        if not target.sum() > 0:
            status[r], stats[r] = -2, np.nan
            continue
        if not (z[r, allowed] < np.inf).all():
            status[r], loss[r], stats[r], grad[r] = -1, np.nan, np.nan, np.nan
            continue
        def statistics(ids):
            """The largest logit, the logarithm of the sum relative to it, and every id's logarithm of its share of these ids."""
            big = z[r, ids].max()
            u = np.where(ids, (z[r] - big) / temperature, -np.inf)
            log_sum = np.log(np.exp(u).sum())
            return big, log_sum, u - log_sum

        big, log_sum, log_q = statistics(allowed)
        outside = allowed & ~on_list
        rest = max(0.0, 1.0 - named) if tail and outside.any() else 0.0
        total = target.sum() + rest
        target, rest = target / total, rest / total
        listed = target > 0
        loss[r] = (target[listed] * (np.log(target[listed]) - log_q[listed])).sum()
        stats[r] = [big, log_sum, -np.inf, -np.inf]
        share = np.zeros(vocab)
        if outside.any():
            stats[r, 2:] = statistics(outside)[:2]
            share = np.exp(statistics(outside)[2])
            if rest > 0:
                loss[r] += rest * (np.log(rest) - ((stats[r, 2] - big) / temperature + stats[r, 3] - log_sum))
        loss[r] *= temperature ** 2
        q = np.exp(log_q)
        grad[r] = np.where(allowed, s * temperature * (q - target - rest * share), 0.0)
        size[r] = abs(s) * temperature * (q + rest * share)
    return loss, stats, grad, status, size


def compare(got, want, dtype=None, temperature=1.0):
    """Asserts that what the calls returned is as near to oracle()'s as the arithmetic allows.  got: dict of tensors."""
    loss, stats, grad, status, size = want
    got = {k: v.detach().cpu() for k, v in got.items()}
    if "status" in got:
        assert got["status"].tolist() == status.tolist()
    if "loss" in got:
        # both logarithms of the student's sums are off, the result is rounded once
        near = temperature ** 2 * 2 * SUM + 2.0 ** -24 * np.abs(loss)
        off = np.abs(got["loss"].double().numpy() - loss)
        assert np.array_equal(np.isnan(off), np.isnan(loss)) and not (off > near).any(), (off, near)
    if "stats" in got:
        s = got["stats"].double().numpy()
        assert np.array_equal(np.nan_to_num(s[:, ::2], nan=7e77), np.nan_to_num(stats[:, ::2], nan=7e77))     # maxima are exact
        with np.errstate(invalid="ignore"):
            off = np.abs(s[:, 1::2] - stats[:, 1::2])
        same = (s[:, 1::2] == stats[:, 1::2]) | (np.isnan(s[:, 1::2]) & np.isnan(stats[:, 1::2]))
        assert (same | (off <= SUM + 2.0 ** -23 * np.abs(stats[:, 1::2]))).all(), off
    if "grad" in got:
        g = got["grad"].double().numpy()
        # the power and the sum that it is divided by, the share q_rest (two logarithms), stats rounded once; half a step of the type, and
        # of its smallest numbers (the power's flush to zero below 2^-126 among them)
        relative = 4 * SUM + 3 * 126 * 0.7 * 2.0 ** -24 + 2.0 ** -22
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
        near = size * relative + np.abs(grad) * torch.finfo(dtype).eps / 2 * 1.01 + tiny * (1 + np.abs(size).max(1, keepdims=True, initial=0))
        off = np.abs(g - grad)
        assert np.array_equal(np.isnan(g), np.isnan(grad))
        bad = off > near
        assert not bad.any(), (np.argwhere(bad)[:5], g[bad][:5], grad[bad][:5])


def case(seed, rows, vocab, dtype, top, tail=False, share=None, wide=False, noise=1.0, teacher=np.float32):
    """A student's rows (exact in `dtype`) and the top of a teacher's near it; some lists end in padding."""
    rng = np.random.default_rng(seed)
    z = rng.normal(0, 3, (rows, vocab)) - 1.1 * np.log1p(rng.permutation(vocab))
    z = torch.from_numpy(z.astype(np.float32)).to(dtype).float().numpy()
    c = {"z": z}
    t = z + rng.normal(0, noise, z.shape)
    if share is not None:
        c["mask"] = words(rng, rows, vocab, share)
        t = np.where(bits_of(c["mask"], vocab), t, -np.inf)
    n = min(top, vocab)
    order = np.argsort(-t, 1, kind="stable")[:, :n]
    value = np.take_along_axis(t, order, 1)
    lse = np.log(np.exp(t - t.max(1, keepdims=True)).sum(1, keepdims=True)) + t.max(1, keepdims=True)
    c["ids"] = np.full((rows, top), -1, np.int32)
    c["values"] = np.full((rows, top), np.nan, teacher)
    c["ids"][:, :n] = np.where(value > -np.inf, order, vocab + 3)
    c["values"][:, :n] = value - lse
    if rows > 2 and n > 2:
        c["ids"][1, n // 2:] = -1
    c["scale"] = rng.uniform(0.2, 1.5, rows).astype(np.float32)
    if rows > 3:
        c["scale"][3] = 0.0
    return c


def gpu(c, dtype, lead=0, gap=0):
    """The arrays on the GPU; logits as rows that begin `lead` elements into a buffer with `gap` more behind each."""
    rows, vocab = c["z"].shape
    buf = torch.full((rows, lead + vocab + gap), 7.0, dtype=dtype, device="cuda")
    buf[:, lead: lead + vocab] = torch.from_numpy(c["z"]).to(dtype)
    cu = lambda k: torch.from_numpy(c[k].view(np.int32) if c[k].dtype == np.uint32 else c[k]).cuda() if k in c else None  # noqa: E731
    return buf[:, lead: lead + vocab], buf, {k: cu(k) for k in ("ids", "values", "mask", "scale")}


def want_of(c, temperature, tail, scaled=True):
    return oracle(c["z"], c["ids"], c["values"], temperature, tail, c.get("mask"), c["scale"] if scaled else None)


__all__ = ["TYPES", "SUM", "bits_of", "case", "compare", "gpu", "oracle", "want_of", "words"]
