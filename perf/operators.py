"""The operators on whole logits rows that stand in front of the sampler and the verifier, and behind the score report: what they
compute in elementary torch operations, the calls that a user makes of them, and the cases they are measured on.

  constrain     penalties over the token history (and the drafts in front of a speculative row), logit biases and the
                grammar bitmask, applied to rows of logits before they are sampled, verified, scored or reported
  distill       loss and gradient of a draft head's logits against the target's top ids and log-probabilities, in one call
  distill_loss  the loss alone (evaluation, or the forward pass of a step whose upstream gradient is not known yet)
  distill_grad  the gradient from the statistics that the forward pass kept

The vocabulary is the engine's (129280) unless a case says otherwise."""
import math

import numpy as np
import torch

own = False

VOCAB = 129280
ZIPF = 1.1
NONFINITE, EMPTY = -1, -2
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user's next token: a short conversation, penalties alone.  Latency and launches
        {"name": "constrain_one", "kind": "constrain", "sequences": 1, "per_sequence": 1, "vocab": VOCAB, "dtype": "fp32", "history": 512,
         "bias": 0, "mask": False, "fill": "lowest"},
        # a server's decode batch: every conversation has its own penalties and a short list of biases
        {"name": "constrain_chat", "kind": "constrain", "sequences": 48, "per_sequence": 1, "vocab": VOCAB, "dtype": "fp32", "history": 4096,
         "bias": 16, "mask": False, "fill": "lowest"},
        # speculative verification under a grammar: two drafts and the bonus row of 32 conversations
        {"name": "constrain_verify", "kind": "constrain", "sequences": 32, "per_sequence": 3, "vocab": VOCAB, "dtype": "fp32", "history": 2048,
         "bias": 0, "mask": True, "fill": "lowest"},
        # the benchmark's constrained batch: 256 conversations with long histories, a grammar, and the longest usual bias list
        {"name": "constrain_long", "kind": "constrain", "sequences": 256, "per_sequence": 1, "vocab": VOCAB, "dtype": "fp32", "history": 32768,
         "bias": 300, "mask": True, "fill": "-inf"},
        # 16-bit rows of a model whose vocabulary is odd: every row starts at another alignment
        {"name": "constrain_bf16_odd", "kind": "constrain", "sequences": 200, "per_sequence": 1, "vocab": 65537, "dtype": "bf16", "history": 1000,
         "bias": 40, "mask": True, "fill": "-inf"},
        # a drafter's online step on one request's positions: latency
        {"name": "distill_online", "kind": "distill", "rows": 8, "vocab": VOCAB, "dtype": "bf16", "top": 20, "teacher": "fp64", "tail": True,
         "temperature": 1.0, "mask": False, "padded": 0},
        # a training micro-batch of 4096 positions
        {"name": "distill_train", "kind": "distill", "rows": 4096, "vocab": VOCAB, "dtype": "bf16", "top": 32, "teacher": "fp32", "tail": True,
         "temperature": 1.0, "mask": False, "padded": 0},
        # fp32 logits at a higher temperature, drafts that follow a grammar, an odd vocabulary, a quarter of the rows padding
        {"name": "distill_masked", "kind": "distill", "rows": 600, "vocab": 65537, "dtype": "fp32", "top": 32, "teacher": "fp32", "tail": False,
         "temperature": 2.0, "mask": True, "padded": 150},
        # evaluation over a stored set: the score report's 32 ids a position
        {"name": "loss_eval", "kind": "distill_loss", "rows": 1024, "vocab": VOCAB, "dtype": "fp32", "top": 32, "teacher": "fp64", "tail": True,
         "temperature": 1.0, "mask": False, "padded": 0},
        # many positions of a small vocabulary
        {"name": "loss_small_vocab", "kind": "distill_loss", "rows": 5000, "vocab": 1031, "dtype": "fp16", "top": 64, "teacher": "fp32", "tail": False,
         "temperature": 1.5, "mask": False, "padded": 0},
        # the backward pass of a micro-batch whose upstream gradient came from elsewhere
        {"name": "grad_train", "kind": "distill_grad", "rows": 2048, "vocab": VOCAB, "dtype": "bf16", "top": 20, "teacher": "fp32", "tail": False,
         "temperature": 1.5, "mask": False, "padded": 0},
        # the same under a grammar, at an odd vocabulary
        {"name": "grad_odd", "kind": "distill_grad", "rows": 333, "vocab": 40001, "dtype": "fp16", "top": 8, "teacher": "fp64", "tail": True,
         "temperature": 1.0, "mask": True, "padded": 33},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["constrain", "constrain", "distill", "distill", "distill_loss", "distill_grad"])
    vocab = VOCAB if rng.random() < 0.4 else _log_int(rng, 1000, 131072)
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "constrain":
        per = rng.choice([1, 1, rng.randint(2, 6)])
        return {"kind": kind, "sequences": _log_int(rng, 1, 256 // per), "per_sequence": per, "vocab": vocab, "dtype": dtype,
                "history": _log_int(rng, 16, 32768), "bias": rng.choice([0, _log_int(rng, 1, 300)]), "mask": rng.random() < 0.6,
                "fill": rng.choice(["lowest", "-inf"])}
    most = min(16384, 4096 * VOCAB * 2 // (vocab * (4 if dtype == "fp32" else 2)))
    rows = _log_int(rng, 1, most)
    tail = rng.random() < 0.5
    return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "top": rng.choice([1, rng.randint(2, 32), rng.randint(33, 100)]),
            "teacher": rng.choice(["fp32", "fp64"]), "tail": tail, "temperature": 1.0 if tail else round(rng.uniform(0.7, 4.0), 2),
            "mask": rng.random() < 0.4, "padded": rng.choice([0, int(rows * rng.uniform(0, 0.4))])}


# ---------------------------------------------------------------------------------------------------------- inputs
def _logits(gen, rows, vocab, dtype):
    """Rows as a trained model gives them: log-Zipf over an order of the ids of each row's own, plus 3 N(0, 1)."""
    out = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    ids = torch.arange(vocab, device="cuda")
    rank = torch.randperm(vocab, device="cuda", generator=gen)
    shift = torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen)
    for r in range(0, rows, 512):
        zipf = -ZIPF * torch.log1p(rank[(ids + shift[r:r + 512]) % vocab].float())
        out[r:r + 512] = zipf.add_(torch.randn(zipf.shape, device="cuda", generator=gen), alpha=3.0)
    return out


def _mask(gen, rows, vocab, share):
    """Grammar bitmasks [rows, ceil(vocab / 32)]: about `share` of the ids, in runs of 8 to 263, the first id always among them."""
    words, count = -(-vocab // 32), int(share * vocab / 136) + 1
    out = torch.empty(rows, words, dtype=torch.int32, device="cuda")
    for r in range(0, rows, 512):
        n = min(512, rows - r)
        start = (torch.rand(n, count, device="cuda", generator=gen) * vocab).long()
        end = (start + 8 + (torch.rand(n, count, device="cuda", generator=gen) * 256).long()).clamp_(max=words * 32)
        edge = torch.zeros(n, words * 32 + 1, dtype=torch.int32, device="cuda")
        edge.scatter_add_(1, start, torch.ones_like(start, dtype=torch.int32)).scatter_add_(1, end, -torch.ones_like(end, dtype=torch.int32))
        on = edge.cumsum(1)[:, :words * 32] > 0
        on[:, 0] = True
        bits = (on.view(n, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
        out[r:r + n] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()
    return out


def _bits(mask, vocab):
    """The bitmask as truth values [rows, vocab]."""
    return ((mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().flatten(1)[:, :vocab]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _prepare_constrain(case, gen) if case["kind"] == "constrain" else _prepare_distill(case, gen)
    s["case"] = case
    return s


def _prepare_constrain(c, gen):
    n, per, vocab, length, bias = c["sequences"], c["per_sequence"], c["vocab"], c["history"], c["bias"]
    # token ids of a conversation: Zipf over an order of the ids of its own; its length is 10 to 100 % of the longest
    cdf = (1.0 / torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64) ** ZIPF).cumsum(0)
    order = torch.randperm(vocab, device="cuda", generator=gen)
    shift = torch.randint(0, vocab, (n, 1), device="cuda", generator=gen)
    zipf = lambda m: order[(torch.searchsorted(cdf, torch.rand(n, m, device="cuda", generator=gen, dtype=torch.float64)  # noqa: E731
                                               * cdf[-1]).clamp_(max=vocab - 1) + shift) % vocab].int()
    lens = (length * (0.1 + 0.9 * torch.rand(n, device="cuda", generator=gen))).int() if n > 1 else \
        torch.full((1,), length, dtype=torch.int32, device="cuda")
    u = torch.rand(n, 3, device="cuda", generator=gen)
    # repetition 1 to 1.3, presence -0.5 to 1, frequency 0 to 0.5
    penalties = u * torch.tensor([0.3, 1.5, 0.5], device="cuda") + torch.tensor([1.0, -0.5, 0.0], device="cuda")
    ids = values = None
    if bias:  # distinct ids, -5 to 5; the lists' ends are padding
        first, step = torch.randint(0, vocab, (n, 1), device="cuda", generator=gen), vocab // bias
        at = torch.arange(bias, device="cuda")
        ids = ((first + at * step) % vocab).int()
        ids[(at >= (bias * (0.5 + 0.5 * torch.rand(n, 1, device="cuda", generator=gen))).ceil())] = -1
        values = 10.0 * torch.rand(n, bias, device="cuda", generator=gen) - 5.0
    dtype = TYPES[c["dtype"]]
    return {"logits": _logits(gen, n * per, vocab, dtype), "history": zipf(length), "history_len": lens, "penalties": penalties.contiguous(),
            "drafts": zipf(per - 1) if per > 1 else None, "bias_ids": ids, "bias_values": values,
            "mask": _mask(gen, n * per, vocab, 0.03) if c["mask"] else None, "fill": -math.inf if c["fill"] == "-inf" else None,
            "out": torch.empty(n * per, vocab, dtype=dtype, device="cuda"), "status": torch.empty(n * per, dtype=torch.int32, device="cuda")}


def _prepare_distill(c, gen):
    rows, vocab, top, padded = c["rows"], c["vocab"], min(c["top"], c["vocab"]), c["padded"]
    logits = _logits(gen, rows, vocab, TYPES[c["dtype"]])
    mask = _mask(gen, rows, vocab, 0.3) if c["mask"] else None
    ids = torch.empty(rows, top, dtype=torch.int32, device="cuda")
    values = torch.empty(rows, top, dtype=torch.float64 if c["teacher"] == "fp64" else torch.float32, device="cuda")
    for r in range(0, rows, 512):  # the target: the drafter's logits plus N(0, 1), under the same grammar
        t = logits[r:r + 512].double()
        t += torch.randn(t.shape, device="cuda", generator=gen)
        if mask is not None:
            t.masked_fill_(~_bits(mask[r:r + 512], vocab), -math.inf)
        best = t.topk(top, dim=1)
        ids[r:r + 512] = torch.where(best.values > -math.inf, best.indices, -1).int()
        values[r:r + 512] = best.values - t.logsumexp(1, keepdim=True)
    # each row's share of the step's loss; rows that are padding have none
    scale = (0.5 + torch.rand(rows, device="cuda", generator=gen)) / rows
    if padded:
        scale[torch.randperm(rows, device="cuda", generator=gen)[:padded]] = 0.0
    s = {"logits": logits, "ids": ids, "values": values, "mask": mask, "scale": scale}
    if c["kind"] == "distill_grad":  # what the forward pass kept
        s["stats"] = torch.empty(rows, 4, device="cuda")
        for r in range(0, rows, 512):
            s["stats"][r:r + 512] = _rows64(s, c, slice(r, r + 512))["stats"]
    if c["kind"] != "distill_loss":
        s["grad"] = torch.empty_like(logits)
    return s


# ------------------------------------------------------------------------------------------------ one pass of each
def run(s):
    return _run_constrain(s) if s["case"]["kind"] == "constrain" else _run_distill(s)


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def _run_constrain(s):
    if own:
        out, status = _package().constrain_logits(
            s["logits"], history=s["history"], history_len=s["history_len"], penalties=s["penalties"], draft_ids=s["drafts"],
            rows_per_sequence=s["case"]["per_sequence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"],
            fill=s["fill"], out=s["out"], status=s["status"])
        return {"out": out, "status": status}
    per, (rows, vocab) = s["case"]["per_sequence"], s["logits"].shape
    x, dev = s["logits"].float(), s["logits"].device
    # occurrences of every id; what is padding, behind the length, or a draft at or behind the row's place goes to a column of its own
    live = torch.arange(s["history"].shape[1], device=dev) < s["history_len"][:, None]
    ids = torch.where(live, s["history"], vocab).long()
    count = torch.zeros(rows // per, vocab + 1, device=dev).scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))
    count = count.repeat_interleave(per, 0)
    if s["drafts"] is not None:
        ahead = torch.arange(per - 1, device=dev) < torch.arange(per, device=dev)[:, None]
        ids = torch.where(ahead, s["drafts"][:, None, :], vocab).long().flatten(0, 1)
        count.scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))
    count = count[:, :vocab]
    repetition, presence, frequency = s["penalties"].repeat_interleave(per, 0)[:, :, None].unbind(1)
    y = torch.where(x > 0, x / repetition, x * repetition) - (presence + frequency * count)
    y = torch.where(count > 0, y, x)
    if s["bias_ids"] is not None:
        ids = torch.where(s["bias_ids"] >= 0, s["bias_ids"], vocab).long()
        bias = torch.zeros(rows // per, vocab + 1, device=dev).scatter_add_(1, ids, s["bias_values"])[:, :vocab]
        y = y + bias.repeat_interleave(per, 0)
    if s["mask"] is not None:
        allowed = _bits(s["mask"], vocab)
        y = torch.where(allowed, y, torch.finfo(s["logits"].dtype).min if s["fill"] is None else s["fill"])
        empty = ~allowed.any(1)
    else:
        allowed, empty = torch.ones_like(x, dtype=torch.bool), torch.zeros(rows, dtype=torch.bool, device=dev)
    status = torch.where((allowed & ~x.isfinite()).any(1), NONFINITE, 0)
    status = torch.where(empty, EMPTY, status).int()
    return {"out": torch.where(empty[:, None], math.nan, y).to(s["logits"].dtype), "status": status}


def _run_distill(s):
    c = s["case"]
    kind, t, tail = c["kind"], c["temperature"], c["tail"]
    if own:
        pkg = _package()
        if kind == "distill":
            loss, grad, status = pkg.distill_loss_grad(s["logits"], s["ids"], s["values"], row_scale=s["scale"], temperature=t, tail=tail,
                                                       mask=s["mask"], out=s["grad"])
            return {"loss": loss, "grad": grad, "status": status}
        if kind == "distill_loss":
            loss, stats, status = pkg.distill_loss(s["logits"], s["ids"], s["values"], temperature=t, tail=tail, mask=s["mask"])
            return {"loss": loss, "stats": stats, "status": status}
        return {"grad": pkg.distill_grad(s["logits"], s["ids"], s["values"], s["stats"], row_scale=s["scale"], temperature=t, tail=tail,
                                         mask=s["mask"], out=s["grad"])}
    z, vocab = s["logits"].float(), s["logits"].shape[1]
    if s["mask"] is not None:
        z = torch.where(_bits(s["mask"], vocab), z, -math.inf)
    place = s["ids"].clamp(0, vocab - 1).long()
    zt = z.gather(1, place)
    named = (s["ids"] >= 0) & (s["ids"] < vocab)
    kept = named & (zt > -math.inf)
    zt = torch.where(kept, zt, -math.inf)
    outside = torch.ones(z.shape[0], vocab + 1, dtype=torch.bool, device=z.device)
    outside = outside.scatter_(1, torch.where(kept, place, vocab), False)[:, :vocab]
    # the drafter's distribution: statistics of the ids outside the list, then of all
    if kind == "distill_grad":
        most, log_sum, most_out, log_sum_out = s["stats"].unbind(1)
    else:
        z_out = torch.where(outside, z, -math.inf)
        most_out = z_out.amax(1)
        log_sum_out = ((z_out - most_out.clamp(min=-1e30)[:, None]) / t).exp().sum(1, dtype=torch.float64).log()
        most = torch.maximum(most_out, zt.amax(1))
        log_sum = (((most_out - most) / t).double() + log_sum_out).exp() + ((zt - most[:, None]) / t).double().exp().sum(1)
        log_sum = log_sum.log()
    log_q = ((zt - most[:, None]) / t).double() - log_sum[:, None]
    log_rest = ((most_out - most) / t).double() + log_sum_out - log_sum
    # the teacher's: over the list, and with the tail over the ids outside it as one more
    if tail:
        p = torch.where(named, s["values"].double().exp(), 0.0)
        rest = torch.where(outside.any(1), (1.0 - p.sum(1)).clamp(min=0.0), 0.0)
        p = torch.where(kept, p, 0.0)
    else:
        p = torch.where(kept, s["values"].double() / t, -math.inf).softmax(1)
        rest = torch.zeros_like(log_rest)
    total = p.sum(1) + rest
    p, rest = p / total[:, None], rest / total
    out = {}
    if kind != "distill_grad":
        terms = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - log_q), 0.0).sum(1)
        terms = terms + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - log_rest), 0.0)
        out["loss"] = (t * t * terms).float()
        if kind == "distill":
            out["loss"] = torch.where(s["scale"] != 0, out["loss"], 0.0)
        else:
            out["stats"] = torch.stack([most, log_sum.float(), most_out, log_sum_out.float()], 1)
        out["status"] = torch.zeros(z.shape[0], dtype=torch.int32, device=z.device)
    if kind != "distill_loss":
        scale = t * s["scale"]
        share = ((log_rest.exp() - rest) * scale).float()
        log_sum_out = torch.where(share != 0, log_sum_out, 0.0).float()
        grad = ((z - most_out.clamp(min=-1e30)[:, None]) / t - log_sum_out[:, None]).exp() * share[:, None]
        grad = torch.cat([grad, torch.zeros_like(grad[:, :1])], 1)
        grad.scatter_(1, torch.where(kept, place, vocab), ((log_q.exp() - p) * scale[:, None]).float())
        out["grad"] = grad[:, :vocab].to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    """Every input read once and every output written once; about 12 operations an id for the statistics and as many for the gradient."""
    c, vocab = case, case["vocab"]
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "constrain":
        rows, n = c["sequences"] * c["per_sequence"], c["sequences"]
        words = 4 * rows * -(-vocab // 32) if c["mask"] else 0
        # a masked id's logit need not be read (about 3 % of the ids are allowed); every output is written
        read = rows * vocab * size * (0.03 if c["mask"] else 1.0)
        tokens = n * c["history"] * (0.55 if n > 1 else 1.0)
        return {"bytes": read + rows * vocab * size + words + 4 * tokens + 8 * n * c["bias"] + 16 * n + 4 * rows, "flops": 4.0 * rows * vocab}
    rows = c["rows"] - (c["padded"] if c["kind"] != "distill_loss" else 0)
    entry = 12 if c["teacher"] == "fp64" else 8
    read = rows * (vocab * size + entry * c["top"] + (4 * -(-vocab // 32) if c["mask"] else 0))
    if c["kind"] == "distill_loss":
        return {"bytes": read + 24 * rows, "flops": 12.0 * rows * vocab}
    if c["kind"] == "distill":
        return {"bytes": read + c["rows"] * (vocab * size + 12), "flops": 24.0 * rows * vocab}
    return {"bytes": read + c["rows"] * (vocab * size + 20), "flops": 12.0 * rows * vocab}


# ------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "constrain":
        return _exact_constrain(s)
    parts = [_rows64(s, case, slice(r, r + 256)) for r in range(0, case["rows"], 256)]
    names = {"distill": ["loss", "grad"], "distill_loss": ["loss", "stats"], "distill_grad": ["grad"]}[case["kind"]]
    got = {k: torch.cat([p[k] for p in parts]) for k in names}
    if case["kind"] == "distill":
        got["loss"][s["scale"] == 0] = 0.0
    if case["kind"] != "distill_grad":
        got["status"] = None
    return got


def _exact_constrain(s):
    """Row by row: the ids that occur, their counts, and the penalties at those places."""
    per, (rows, vocab) = s["case"]["per_sequence"], s["logits"].shape
    out = s["logits"].double()
    lowest = torch.finfo(s["logits"].dtype).min if s["fill"] is None else s["fill"]
    for r in range(rows):
        q, j = divmod(r, per)
        seen = s["history"][q, :int(s["history_len"][q])]
        if j:
            seen = torch.cat([seen, s["drafts"][q, :j]])
        ids, count = torch.unique(seen, return_counts=True)
        repetition, presence, frequency = s["penalties"][q].double()
        x = out[r, ids.long()]
        out[r, ids.long()] = torch.where(x > 0, x / repetition, x * repetition) - presence - frequency * count
        if s["bias_ids"] is not None:
            listed_ids = s["bias_ids"][q] >= 0
            out[r].index_add_(0, s["bias_ids"][q][listed_ids].long(), s["bias_values"][q][listed_ids].double())
        if s["mask"] is not None:
            words = s["mask"][r].cpu().numpy().view(np.uint8)
            on = np.unpackbits(words, bitorder="little")[:vocab].astype(bool)
            out[r, torch.from_numpy(~on).cuda()] = lowest
    return {"out": out, "status": None}


def _rows64(s, c, rows):
    """Loss, gradient and statistics of some rows: softmax over all allowed ids, the target as a whole row, their difference."""
    t, tail = c["temperature"], c["tail"]
    z = s["logits"][rows].double()
    n, vocab = z.shape
    if s["mask"] is not None:
        z[~_bits(s["mask"][rows], vocab)] = -math.inf
    entry, col = (s["ids"][rows] >= 0).nonzero(as_tuple=True)
    where = s["ids"][rows][entry, col].long()
    value = s["values"][rows][entry, col].double()
    on_list = torch.zeros(n, vocab, dtype=torch.bool, device=z.device)
    on_list[entry, where] = True
    target = torch.zeros(n, vocab, dtype=torch.float64, device=z.device)
    log_q = (z / t).log_softmax(1)
    outside = z.masked_fill(on_list, -math.inf)
    log_in_rest = (outside / t).log_softmax(1)          # an id's share of the ids outside the list; NaN where there are none
    rest_ids = (outside > -math.inf).any(1)
    log_rest = log_q.masked_fill(on_list, -math.inf).logsumexp(1)
    if tail:
        target[entry, where] = value.exp()
        rest = torch.where(rest_ids, (1.0 - target.sum(1)).clamp(min=0.0), 0.0)
    else:
        peak = torch.full((n,), -math.inf, dtype=torch.float64, device=z.device).scatter_reduce_(0, entry, value, "amax")
        target[entry, where] = ((value - peak[entry]) / t).exp()
        rest = torch.zeros(n, dtype=torch.float64, device=z.device)
    total = target.sum(1) + rest
    target, rest = target / total[:, None], rest / total
    loss = (target.xlogy(target) - torch.where(target > 0, target * log_q, 0.0)).sum(1)
    loss = loss + rest.xlogy(rest) - torch.where(rest > 0, rest * log_rest, 0.0)
    whole = target + torch.where(on_list | (rest[:, None] == 0), 0.0, rest[:, None] * log_in_rest.exp())
    stats = [z.amax(1), (z / t).logsumexp(1) - z.amax(1) / t, outside.amax(1), (outside / t).logsumexp(1) - outside.amax(1) / t]
    stats[3] = torch.where(rest_ids, stats[3], -math.inf)
    return {"loss": t * t * loss, "grad": s["scale"][rows, None].double() * t * (log_q.exp() - whole), "stats": torch.stack(stats, 1)}
