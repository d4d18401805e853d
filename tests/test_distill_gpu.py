"""The distillation calls against their FP64 definition: types, alignments, vocabularies from one id to the largest, lists from one entry
to 256, masks, duplicates, padding, values that are not finite, rows that have nothing to learn, in place and out of place."""
import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from constrain_case import expected
from distill_case import TYPES, bits_of, case, compare, gpu, oracle, want_of, words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    entry.build()
    return entry.load_package()


def check(pkg, c, dtype, temperature=1.0, tail=False, lead=0, gap=0, out_lead=0, out_gap=0, wants=None):
    rows, vocab = c["z"].shape
    view, buf, t = gpu(c, dtype, lead, gap)
    kept = buf.clone()
    more = {"temperature": temperature, "tail": tail, "mask": t["mask"]}
    want, plain = wants or (want_of(c, temperature, tail), want_of(c, temperature, tail, scaled=False))
    grads = torch.full((rows, out_lead + vocab + out_gap), 5.0, dtype=dtype, device="cuda")
    out = grads[:, out_lead: out_lead + vocab]

    def around(name):
        beside = torch.cat([grads[:, :out_lead], grads[:, out_lead + vocab:]], 1)
        assert (beside == 5.0).all(), name          # nothing beside the rows is written
        assert torch.equal(buf.view(torch.uint8), kept.view(torch.uint8)), name
    loss, stats, status = pkg.distill_loss(view, t["ids"], t["values"], **more)
    compare({"loss": loss, "stats": stats, "status": status}, plain, temperature=temperature)
    both = pkg.distill_loss_grad(view, t["ids"], t["values"], row_scale=t["scale"], out=out, **more)
    assert both[1] is out
    compare(dict(zip(("loss", "grad", "status"), both)), want, dtype, temperature)
    around("both")
    live = t["scale"] != 0
    assert torch.equal(both[0][live].view(torch.int32), loss[live].view(torch.int32))       # the same arithmetic
    out.fill_(3.0)
    compare({"grad": pkg.distill_grad(view, t["ids"], t["values"], stats, row_scale=t["scale"], out=out, **more)}, want, dtype, temperature)
    around("grad")
    again = out.clone()
    pkg.distill_grad(view, t["ids"], t["values"], stats, row_scale=t["scale"], out=view, **more)      # in place
    assert torch.equal(view.contiguous().view(torch.uint8), again.contiguous().view(torch.uint8))
    buf.copy_(kept)
    in_place = pkg.distill_loss_grad(view, t["ids"], t["values"], row_scale=t["scale"], out=view, **more)
    compare(dict(zip(("loss", "grad", "status"), in_place)), want, dtype, temperature)
    beside = torch.cat([buf[:, :lead], buf[:, lead + vocab:]], 1)
    assert (beside == 7.0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab,lead,gap,top", [(1, 0, 0, 1), (2, 1, 0, 2), (7, 3, 2, 7), (31, 0, 1, 40), (32, 0, 0, 8), (33, 7, 0, 5), (1000, 0, 0, 20),
                                                (1031, 5, 1, 256), (16385, 1, 0, 32), (32769, 2, 1, 3), (129280, 0, 0, 32), (131072, 3, 5, 100)])
def test_rows_of_every_size_type_and_alignment(pkg, dtype, vocab, lead, gap, top):
    t = TYPES[dtype]
    check(pkg, case(vocab, 5, vocab, t, top, tail=True), t, 1.0, True, lead, gap, lead, gap)
    check(pkg, case(vocab + 1, 5, vocab, t, top, share=0.5, teacher=np.float64), t, 2.0, False, lead, gap, 0, 3)   # (another alignment)


@pytest.mark.parametrize("rows,vocab,top,tail,temperature,share", [
    (1, 129280, 20, True, 1.0, None), (2, 129280, 1, False, 0.5, 0.02), (60, 40001, 64, True, 1.0, 0.3), (300, 5003, 17, False, 4.0, None),
    (150, 65537, 33, True, 1.0, None), (147, 40001, 5, True, 1.0, None), (148, 40001, 5, False, 1.3, None), (148, 36857, 9, True, 1.0, None),
    (148, 36865, 255, True, 1.0, None), (148, 36865, 256, False, 1.0, None), (444, 1031, 7, True, 1.0, 0.5), (445, 1031, 7, True, 1.0, 0.5), (1000, 257, 256, False, 1.5, 0.9), (37, 100000, 8, True, 1.0, 0.0005)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_batches(pkg, rows, vocab, top, tail, temperature, share, dtype):
    check(pkg, case(rows + vocab, rows, vocab, TYPES[dtype], top, tail, share), TYPES[dtype], temperature, tail)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tail,temperature", [(True, 1.0), (False, 1.7)])
@pytest.mark.parametrize("vocab", [900, 70001])
def test_lists_and_rows_where_it_can_go_wrong(pkg, dtype, tail, temperature, vocab):
    t = TYPES[dtype]
    c = case(11, 20, vocab, t, 30, tail, share=0.5, teacher=np.float64)
    allowed = bits_of(c["mask"], vocab)
    forbidden = [np.flatnonzero(~a) for a in allowed]
    inside = [np.setdiff1d(np.flatnonzero(a), c["ids"][r]) for r, a in enumerate(allowed)]
    c["scale"][:] = 0.7
    c["z"][0, forbidden[0][:3]] = np.nan, np.inf, -np.inf                 # masked: nothing
    c["z"][1, inside[1][4]] = np.nan                                      # allowed: rejected
    c["z"][2, inside[2][-1]] = np.inf
    c["z"][3, inside[3][:7]] = -np.inf                                    # not allowed either
    c["z"][4, c["ids"][4, 0]] = -np.inf                                   # and an entry for it is padding
    c["z"][5, c["ids"][5, 2]] = np.nan
    c["values"][6, 3] = np.nan
    c["values"][7, 3] = np.inf
    c["values"][8, 3] = -np.inf                                           # probability 0
    c["values"][9] = -np.inf                                              # all of them
    c["ids"][10] = -1                                                     # nothing but padding (NaN values there mean nothing)
    c["values"][10] = np.nan
    c["mask"][11] = 0                                                     # no id at all
    c["values"][12] += 0.5                                                # probabilities that add up to more than 1
    c["ids"][13, 5:9] = c["ids"][13, 2]                                   # one id five times
    c["ids"][13, 20] = c["ids"][13, 2]
    c["z"][14] = np.nan                                                   # padding rows are not read
    c["scale"][14] = 0.0
    c["mask"][15] = 0                                                     # the list names every allowed id
    for i in c["ids"][15, :9]:
        c["mask"][15, i // 32] |= np.uint32(1 << (i % 32))
    c["z"][16] = torch.finfo(t).min                                       # the type's lowest value everywhere
    c["z"][17] = torch.finfo(t).min                                       # ... but for the list
    c["z"][17, c["ids"][17]] = 1.0
    c["ids"][18] = c["ids"][18, 0]                                        # one id only
    c["scale"][19] = -0.3
    want = want_of(c, temperature, tail)
    assert want[3][[1, 2, 5, 6, 7, 9, 10, 11]].tolist() == [-1, -1, -1, -1, -1, -2, -2, -2] and want[3][[0, 3, 4, 8, 13, 14, 15, 16, 17, 19]].tolist() == [0] * 10
    if tail:                                                              # (1.65 times what the list holds of the smaller row, and of the larger)
        assert want[3][12] == {900: -10, 70001: 0}[vocab]
    check(pkg, c, t, temperature, tail)
    check(pkg, c, t, temperature, tail, 1, 2, 1, 2)


@pytest.mark.parametrize("dtype,vocab,tail,temperature", [("fp32", 50021, True, 1.0), ("fp32", 131072, False, 0.6), ("bf16", 50021, False, 1.7),
                                                          ("bf16", 129280, True, 1.0), ("fp16", 50024, True, 1.0), ("fp16", 98305, False, 3.0)])
def test_many_rows_where_it_can_go_wrong(pkg, dtype, vocab, tail, temperature):
    """Batches of long rows that each CTA takes several of: rows to skip, to reject and to take, in every order, at every alignment."""
    t = TYPES[dtype]
    c = case(21, 16, vocab, t, 30, tail, teacher=np.float64)
    inside = [np.setdiff1d(np.arange(vocab), c["ids"][r]) for r in range(16)]
    c["scale"][:] = np.linspace(0.5, 1.5, 16)
    c["scale"][[0, 5]] = 0.0
    c["z"][0] = np.nan                                                    # padding rows are not read
    c["z"][2, inside[2][-1]] = np.nan
    c["z"][3, inside[3][0]] = np.inf
    c["z"][4, inside[4][::2]] = -np.inf                                   # half of the ids are not allowed
    c["z"][6, c["ids"][6, 1]] = -np.inf
    c["ids"][7] = -1
    c["values"][8, 2] = np.nan
    c["ids"][9, 3:20] = c["ids"][9, 1]                                    # one id eighteen times
    c["ids"][10] = np.arange(30)                                          # ids side by side, at the row's beginning and end
    c["ids"][11] = vocab - 1 - np.arange(30)
    c["z"][12] = torch.finfo(t).min
    c["z"][13] = torch.finfo(t).min
    c["z"][13, c["ids"][13]] = 1.0
    c["scale"][14] = -1.0
    times, order = 45, np.random.default_rng(22).permutation(16 * 45)
    wants = [tuple(np.tile(w, (times,) + (1,) * (w.ndim - 1))[order] for w in want_of(c, temperature, tail, scaled)) for scaled in (True, False)]
    assert wants[0][3][np.argsort(order)][:16].tolist() == [0, 0, -1, -1, 0, 0, 0, -2, -1, 0, 0, 0, 0, 0, 0, 0]
    c = {k: np.tile(v, (times,) + (1,) * (v.ndim - 1))[order] for k, v in c.items()}
    check(pkg, c, t, temperature, tail, wants=wants)
    check(pkg, c, t, temperature, tail, 3, 2, 1, 0, wants=wants)          # (an output at another alignment)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_student_that_is_sure_of_the_list(pkg, dtype):
    """The ids outside the list hold e^-120 of the student's mass: their share is not a difference of sums near 1."""
    t = TYPES[dtype]
    c = case(12, 4, 20000, t, 16, tail=True)
    c["z"] -= 120.0
    for r in range(4):
        own = c["ids"][r][c["ids"][r] >= 0]
        c["z"][r, own] += 120.0
    c["z"] = torch.from_numpy(c["z"]).to(t).float().numpy()
    loss = want_of(c, 1.0, True)[0]
    assert (loss[:3] > 1.0).all()
    check(pkg, c, t, 1.0, True)


def test_offsets_beyond_32_bits(pkg):
    """Rows 2^30 and more elements apart, loss and gradient in place."""
    stride, vocab = (1 << 30) + 72, 3001
    c = case(13, 3, vocab, torch.bfloat16, 12, tail=True)
    buf = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((3, vocab), (stride, 1))
    view.copy_(torch.from_numpy(c["z"]))
    _, _, t = gpu(c, torch.bfloat16)
    got = pkg.distill_loss_grad(view, t["ids"], t["values"], row_scale=t["scale"], tail=True, out=view)
    compare(dict(zip(("loss", "grad", "status"), got)), want_of(c, 1.0, True), torch.bfloat16)


def test_teacher_lists_inside_wider_rows(pkg):
    """Ids and values as columns of wider buffers (the first n of a stored list)."""
    c = case(14, 6, 4097, torch.float32, 40, tail=False)
    view, _, t = gpu(c, torch.float32)
    n = dict(c, ids=c["ids"][:, :11].copy(), values=c["values"][:, :11].copy())
    loss, stats, status = pkg.distill_loss(view, t["ids"][:, :11], t["values"][:, :11], temperature=3.0)
    compare({"loss": loss, "stats": stats, "status": status}, want_of(n, 3.0, False, scaled=False), temperature=3.0)


def test_results_do_not_change_from_run_to_run(pkg):
    c = case(15, 40, 129280, torch.bfloat16, 32, tail=True)
    view, _, t = gpu(c, torch.bfloat16)
    runs = [pkg.distill_loss_grad(view, t["ids"], t["values"], tail=True) for _ in range(5)]
    for r in runs[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(r, runs[0]))


def test_other_streams_and_captured_graphs(pkg):
    """Two calls at once on two streams, and a captured step (loss, then gradient) replayed on new inputs."""
    cases = [case(16 + i, 50, 30011, torch.float32, 24, True, share=0.5) for i in range(2)]
    wants = [want_of(c, 1.0, True) for c in cases]
    plain = [want_of(c, 1.0, True, scaled=False) for c in cases]
    inputs = [gpu(c, torch.float32) for c in cases]
    streams, got = [torch.cuda.Stream() for _ in cases], []
    torch.cuda.synchronize()
    for s, (view, _, t) in zip(streams, inputs):
        with torch.cuda.stream(s):
            got.append(pkg.distill_loss_grad(view, t["ids"], t["values"], row_scale=t["scale"], tail=True, mask=t["mask"]))
    torch.cuda.synchronize()
    for g, w in zip(got, wants):
        compare(dict(zip(("loss", "grad", "status"), g)), w, torch.float32)
    x, kept = inputs[0][0].clone(), {k: v.clone() for k, v in inputs[0][2].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, stats, status = pkg.distill_loss(x, kept["ids"], kept["values"], tail=True, mask=kept["mask"])
        grad = pkg.distill_grad(x, kept["ids"], kept["values"], stats, row_scale=kept["scale"], tail=True, mask=kept["mask"])
    for i in (1, 0, 1):
        x.copy_(inputs[i][0])
        for k, v in kept.items():
            v.copy_(inputs[i][2][k])
        graph.replay()
        torch.cuda.synchronize()
        compare({"loss": loss, "stats": stats, "status": status}, plain[i])
        compare({"grad": grad}, wants[i], torch.float32)


def test_the_gradient_against_differences_of_the_loss(pkg):
    """Along the gradient's own direction d the loss falls by h |g|^2 / |g|: with h = 1/8 either way the central difference's error is
    below h^2 / 6 times the third derivative (at most 1 along a unit direction, T = 1), that of the two losses 2 * 2 SUM / (2 h)."""
    c = case(18, 3, 2000, torch.float32, 10, tail=True)
    c["scale"][:] = 1.0
    view, _, t = gpu(c, torch.float32)
    _, grad, _ = pkg.distill_loss_grad(view, t["ids"], t["values"], tail=True)
    norm = grad.double().norm(dim=1)
    h, d = 0.125, grad / grad.norm(dim=1, keepdim=True)
    up = pkg.distill_loss(view + h * d, t["ids"], t["values"], tail=True)[0].double()
    down = pkg.distill_loss(view - h * d, t["ids"], t["values"], tail=True)[0].double()
    assert ((up - down) / (2 * h) - norm).abs().max() < h * h / 6 + 1.5e-4 and norm.min() > 0.02


def test_a_draft_head_learns_from_what_the_target_reports(pkg):
    """The calls as they are used together: the target's rows are constrained, scored, and their top ids and log-probabilities teach the
    drafter's logits under the same grammar; the drafter's weights get their gradient from the rows'."""
    rows, vocab, hidden, n = 24, 129280, 64, 32
    rng = np.random.default_rng(19)
    target = torch.from_numpy(rng.normal(0, 3, (rows, vocab)).astype(np.float32)).cuda()
    history = torch.from_numpy(rng.integers(0, vocab, (rows, 200)).astype(np.int32)).cuda()
    packed = words(rng, rows, vocab, 0.2)
    mask = torch.from_numpy(packed.view(np.int32)).cuda()
    constrained, status = pkg.constrain_logits(target, history=history, repetition=1.2, mask=mask)
    assert (status == 0).all()
    want, _ = expected(target.cpu().numpy(), torch.float32, history.cpu().numpy(), None, np.tile(np.float32([1.2, 0, 0]), (rows, 1)), mask=packed)
    assert np.array_equal(constrained.cpu().numpy(), want)
    _, _, ids, logprobs, status = pkg.score_logits(constrained, n)
    assert (status == 0).all()
    x = torch.from_numpy(rng.normal(0, 1, (rows, hidden)).astype(np.float32)).cuda().requires_grad_()
    w = torch.from_numpy(rng.normal(0, 0.3, (vocab, hidden)).astype(np.float32)).cuda().requires_grad_()
    logits = x @ w.t()
    scale = torch.full((rows,), 1.0 / rows, device="cuda")
    scale[5] = 0.0
    loss, grad, status = pkg.distill_loss_grad(logits.detach(), ids, logprobs, row_scale=scale, tail=True, mask=mask)
    logits.backward(grad)
    z = logits.detach().cpu().numpy()
    ref = oracle(z, ids.cpu().numpy(), logprobs.cpu().numpy(), 1.0, True, packed, scale.cpu().numpy())
    compare({"loss": loss, "grad": grad, "status": status}, ref, torch.float32)
    want_w, want_x = ref[2].T @ x.detach().cpu().numpy().astype(np.float64), ref[2] @ w.detach().cpu().numpy().astype(np.float64)
    # products of at most 129280 terms in FP32 (or of rounded operands): 2^-9 of the sizes of what is added up covers either
    size_w, size_x = np.abs(ref[2]).T @ np.abs(x.detach().cpu().numpy()), np.abs(ref[2]) @ np.abs(w.detach().cpu().numpy())
    assert (np.abs(w.grad.cpu().numpy() - want_w) <= 2.0 ** -9 * size_w + 1e-12).all()
    assert (np.abs(x.grad.cpu().numpy() - want_x) <= 2.0 ** -9 * size_x + 1e-12).all()


def test_refusals(pkg):
    z = torch.zeros(3, 64, device="cuda")
    ids, v = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, 4, device="cuda")
    for args in [(z.cpu(), ids, v), (z.double(), ids, v), (z.t(), ids, v), (z, ids.long(), v), (z, ids, v.half()), (z, ids[:2], v), (z, ids, v[:, :3]),
                 (z, ids.t(), v.t()), (z[0], ids, v)]:
        with pytest.raises(ValueError):
            pkg.distill_loss(*args)
        with pytest.raises(ValueError):
            pkg.distill_loss_grad(*args)
    with pytest.raises(ValueError):
        pkg.distill_grad(z, ids, v, torch.zeros(3, 3, device="cuda"))
    with pytest.raises(ValueError):
        pkg.distill_loss_grad(z, ids, v, row_scale=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        pkg.distill_loss_grad(z, ids, v, out=torch.zeros(3, 64, dtype=torch.float16, device="cuda"))
    with pytest.raises(RuntimeError, match="temperature"):
        pkg.distill_loss(z, ids, v, temperature=0.0)
    with pytest.raises(RuntimeError, match="temperature 1"):
        pkg.distill_loss(z, ids, v, temperature=2.0, tail=True)
    with pytest.raises(RuntimeError, match="mask"):
        pkg.distill_loss(z, ids, v, mask=torch.zeros(3, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="top"):
        pkg.distill_loss(z, ids[:, :0], v[:, :0])
    buf = torch.zeros(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        pkg.distill_loss_grad(buf[:3], ids, v, out=buf[1:])
