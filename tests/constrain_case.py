"""The rule of ds41_b200_constrain_logits as NumPy, operation by operation in FP32 (so that results are compared bit for bit), and
inputs for it."""
import numpy as np
import torch

f4 = np.float32
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def bits_of(mask, vocab):
    """uint32 words [rows, n] -> truth values [rows, vocab]."""
    return np.unpackbits(np.ascontiguousarray(mask).view(np.uint8), axis=1, bitorder="little")[:, :vocab].astype(bool)


def expected(x, dtype, history=None, lens=None, penalties=None, drafts=None, per=1, bias_ids=None, bias_values=None, mask=None, fill=None):
    """(rows as float32 of the rounded type, status) for x float32 [rows, vocab] that the type holds exactly."""
    rows, vocab = x.shape
    info = torch.finfo(dtype)
    fill = info.min if fill is None else fill if np.isinf(fill) else min(max(fill, info.min), info.max)
    out, status = np.empty_like(x), np.zeros(rows, np.int32)
    with np.errstate(all="ignore"):
        for r in range(rows):
            s, j = divmod(r, per)
            rep, pres, freq = (f4(v) for v in (penalties[s] if penalties is not None else (1, 0, 0)))
            if not (rep > 0 and np.isfinite([rep, pres, freq]).all()):
                out[r], status[r] = np.nan, -11
                continue
            n = 0 if history is None else history.shape[1] if lens is None else int(lens[s])
            if n < 0 or (history is not None and n > history.shape[1]) or n + (j if drafts is not None else 0) > 65535:
                out[r], status[r] = np.nan, -7
                continue
            allowed = bits_of(mask[r:r + 1], vocab)[0] if mask is not None else np.ones(vocab, bool)
            if not allowed.any():
                out[r], status[r] = np.nan, -2
                continue
            ids = history[s, :n] if history is not None else np.empty(0, np.int32)
            if drafts is not None:
                ids = np.concatenate([ids, drafts[s, :j]])
            count = np.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=vocab).astype(f4)
            v = np.where(x[r] > 0, x[r] / rep, x[r] * rep)
            y = np.where(count > 0, v - (pres + freq * count), x[r]).astype(f4)
            if bias_ids is not None:
                sums = {}
                for i, b in zip(bias_ids[s].tolist(), bias_values[s]):
                    if 0 <= i < vocab:
                        sums[i] = f4(sums[i] + b) if i in sums else f4(b)
                for i, b in sums.items():
                    y[i] = f4(y[i] + b)
            y = torch.from_numpy(np.where(allowed, y, f4(fill))).to(dtype).float().numpy()
            out[r] = y
            if (allowed & ~np.isfinite(x[r])).any():
                status[r] = -1
            elif (allowed & ~np.isfinite(y)).any():
                status[r] = -3
    return out, status


def words(rng, rows, vocab, share):
    """Bitmasks in which about `share` of the ids are allowed, one at least; bits behind the last id are set, and mean nothing."""
    n = (vocab + 31) // 32
    bits = rng.random((rows, n * 32)) < share
    bits[np.arange(rows), rng.integers(0, vocab, rows)] = True
    bits[:, vocab:] = True
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def case(seed, sequences, vocab, dtype, per=1, history=0, biases=0, share=None, repeat=0.3):
    """Arrays of one call: rows that `dtype` holds exactly, Zipf-like histories with ids outside the vocabulary, bias lists with
    padding and repeated ids."""
    rng = np.random.default_rng(seed)
    rows = sequences * per
    x = torch.from_numpy(rng.normal(0, 3, (rows, vocab)).astype(f4)).to(dtype).float().numpy()
    c = {"x": x, "per": per, "penalties": np.stack([rng.uniform(0.8, 1.4, sequences), rng.uniform(-1, 1, sequences),
                                                    rng.uniform(-0.2, 0.6, sequences)], 1).astype(f4)}
    if history:
        ids = np.minimum(rng.zipf(1.3, (sequences, history)), 2 * vocab) - 1
        c["history"] = np.where(rng.random(ids.shape) < 0.1, -1 - ids, (ids * 7919) % (vocab + 3)).astype(np.int32)
        c["lens"] = rng.integers(0, history + 1, sequences).astype(np.int32)
        c["lens"][0] = history
        c["lens"][-1] = 0 if sequences > 1 else history
    if per > 1:
        c["drafts"] = rng.integers(0, vocab, (sequences, per - 1)).astype(np.int32)
    if biases:
        ids = rng.integers(-1, vocab + 1, (sequences, biases))
        again = rng.random(ids.shape) < repeat
        c["bias_ids"] = np.where(again, ids[:, :1], ids).astype(np.int32)
        c["bias_values"] = rng.normal(0, 3, ids.shape).astype(f4)
    if share is not None:
        c["mask"] = words(rng, rows, vocab, share)
    return c


def rows_at(x, dtype, lead, gap):
    """x on the GPU as a view whose rows begin `lead` elements into a buffer with `gap` more behind each row."""
    rows, vocab = x.shape
    buf = torch.full((rows, lead + vocab + gap), 7.0, dtype=dtype, device="cuda")
    view = buf[:, lead: lead + vocab]
    view.copy_(torch.from_numpy(x))
    return buf, view


def call(pkg, c, logits, **more):
    cu = lambda k: torch.from_numpy(c[k].view(np.int32) if c[k].dtype == np.uint32 else c[k]).cuda() if k in c else None  # noqa: E731
    return pkg.constrain_logits(logits, history=cu("history"), history_len=cu("lens"), penalties=cu("penalties"), draft_ids=cu("drafts"),
                                rows_per_sequence=c["per"], bias_ids=cu("bias_ids"), bias_values=cu("bias_values"), mask=cu("mask"), **more)


def same(got, want):
    """Bit for bit as float32, but for the sign of zero and the payload of NaN."""
    return np.array_equal(got, want, equal_nan=True)
