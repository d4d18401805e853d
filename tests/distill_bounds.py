"""How far the distillation's results may be from the FP64 definition, in either of its kernels and at any temperature.

In roundings of 2^-24.  The student's sum: with a the distance of an id from the largest in powers of two, the factor log2(e) / T is
rounded (a), and each step of the chain thread, warp, CTA, row takes a difference and a product of its own part of a (2 a together,
and 1 for the power taken from the rounded product); ids beyond a = 27 hold less than 2^-10 of the sum: (3 * 27 + 1) ln 2 = 57.  The power
is 2 ulp off (4).  A thread of the streamed kernel adds 131072 / 384 / 4 = 86 numbers to each of four sums, and these (90); its maximum
can rise with each of its 22 groups (FP32; 11 in 16 bits), a power and a product each time (110); making good for the rounded
product (6), the warps' exchange and the row's (10 each).  Together 287, an ulp of slack on every 25: SUM = 300 * 2^-24, relative for the
sum, absolute for its logarithm.
A gradient's power has a up to 126: (3 * 126 + 1) ln 2 = 263; q_rest is a quotient of two sums times a power and the statistics of
the forward pass were rounded once, their exponentials' arguments again (3 * 12 * 1.45 + 3 * 4): 4 SUM and 512 * 2^-24 cover them; in
16-bit types the factor stands in the exponent, which below 512 is off by half of 2^-15."""
import numpy as np
import torch

SUM = 300 * 2.0 ** -24


def compare(got, want, dtype, temperature, order):
    """want: of the rows that `order` repeats."""
    loss, stats, grad, status, size = [w[order] for w in want]
    got = {k: v.detach().cpu() for k, v in got.items()}
    if "status" in got:
        assert got["status"].tolist() == status.tolist()
    if "loss" in got:
        near = temperature ** 2 * 2 * SUM + 2.0 ** -24 * np.abs(loss)
        off = np.abs(got["loss"].double().numpy() - loss)
        assert (off <= near).all(), (np.flatnonzero(~(off <= near))[:5], off, near)
    if "stats" in got:
        s = got["stats"].double().numpy()
        assert np.array_equal(s[:, ::2], stats[:, ::2])                       # maxima are exact
        with np.errstate(invalid="ignore"):
            off = np.abs(s[:, 1::2] - stats[:, 1::2])
        right = (s[:, 1::2] == stats[:, 1::2]) | (off <= SUM + 2.0 ** -23 * np.abs(stats[:, 1::2]))
        assert right.all(), (np.argwhere(~right)[:5], s[~right.all(1)][:5], stats[~right.all(1)][:5])
    if "grad" in got:
        g = got["grad"].double().numpy()
        relative = 4 * SUM + 512 * 2.0 ** -24 + (2.0 ** -16 if dtype != torch.float32 else 0.0)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
        near = size * relative + np.abs(grad) * torch.finfo(dtype).eps / 2 * 1.01 + tiny * (1 + size.max(1, keepdims=True))
        bad = ~(np.abs(g - grad) <= near)
        assert not bad.any(), (np.argwhere(bad)[:5], g[bad][:5], grad[bad][:5])
