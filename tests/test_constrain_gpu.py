"""ds41_b200_constrain_logits against its rule in NumPy, bit for bit: types, alignments, lengths from none to the longest, repeated ids
in the bias list, masks that leave a row empty, values that are not finite in masked and in allowed places, in place and out of
place; and in front of the sampler, the verifier and the score report."""
import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from constrain_case import TYPES, bits_of, call, case, expected, rows_at, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    entry.build()
    return entry.load_package()


def want_of(c, dtype, fill=None):
    return expected(c["x"], dtype, c.get("history"), c.get("lens"), c["penalties"], c.get("drafts"), c["per"], c.get("bias_ids"),
                    c.get("bias_values"), c.get("mask"), fill)


def check(pkg, c, dtype, lead=0, gap=0, out_lead=0, out_gap=0, fill=None):
    want, status = want_of(c, dtype, fill)
    _, view = rows_at(c["x"], dtype, lead, gap)
    buf, out = rows_at(np.zeros_like(c["x"]), dtype, out_lead, out_gap)
    got, st = call(pkg, c, view, out=out, fill=fill)
    assert got is out and st.cpu().tolist() == status.tolist()
    assert same(got.float().cpu().numpy(), want)
    around = torch.cat([buf[:, :out_lead], buf[:, out_lead + out.shape[1]:]], 1)
    assert (around == 7.0).all()                                    # nothing beside the rows is written
    assert same(view.float().cpu().numpy(), c["x"])                 # nor the input
    st.fill_(77)
    got, st = call(pkg, c, view, out=view, fill=fill, status=st)    # in place: the same rows, and the old ones are gone
    assert st.cpu().tolist() == status.tolist() and same(got.float().cpu().numpy(), want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab,lead,gap", [(1, 0, 0), (31, 1, 2), (32, 0, 0), (33, 3, 0), (1000, 0, 0), (1031, 5, 1), (16385, 7, 0), (32769, 2, 1),
                                            (129280, 0, 0), (131072, 1, 3)])
def test_rows_of_every_size_type_and_alignment(pkg, dtype, vocab, lead, gap):
    c = case(vocab + lead, 3, vocab, TYPES[dtype], per=2, history=777, biases=40, share=0.4)
    check(pkg, c, TYPES[dtype], lead, gap, lead, gap)
    check(pkg, c, TYPES[dtype], lead, gap, 0, 5, fill=-np.inf)      # (an output at another alignment)


@pytest.mark.parametrize("sequences,per,history,biases,share", [
    (1, 1, 1, 0, None), (1, 1, 0, 0, 0.5), (1, 1, 65535, 1024, None), (2, 6, 65530, 3, 0.01), (2, 6, 65531, 0, None), (5, 1, 0, 1, None), (160, 1, 100, 0, 0.9),
    (40, 4, 5000, 300, 0.02), (3, 1, 4099, 17, 0.0005)])
@pytest.mark.parametrize("dtype,vocab", [("fp32", 129280), ("bf16", 40001)])
def test_lengths_and_lists(pkg, sequences, per, history, biases, share, dtype, vocab):
    check(pkg, case(9 + history, sequences, vocab, TYPES[dtype], per, history, biases, share), TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_one_id_through_the_whole_history_and_the_whole_list(pkg, dtype):
    """The largest count (65535 occurrences), and every entry of the longest list for the same id."""
    c = case(4, 2, 3000, TYPES[dtype], history=65535, biases=1024)
    c["lens"][:] = 65535
    c["history"][0] = 2999
    c["penalties"][:, 2] = 1e-4
    c["bias_ids"][0] = 2999
    c["bias_ids"][1] = 0
    check(pkg, c, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_values_that_are_not_finite(pkg, dtype):
    """NaN and infinities are nothing in masked places and reject the row in allowed ones; so do results beyond the type's range."""
    t = TYPES[dtype]
    c = case(5, 9, 20000, t, history=300, biases=20, share=0.5)
    allowed = bits_of(c["mask"], 20000)
    inside, outside = [np.flatnonzero(a) for a in allowed], [np.flatnonzero(~a) for a in allowed]
    for r, v in enumerate([np.nan, np.inf, -np.inf]):
        c["x"][r, outside[r][[0, 9000]]] = v
        c["x"][3 + r, inside[3 + r][r * 4000]] = v
    c["x"][6, inside[6][5]] = torch.finfo(t).max
    c["history"][6, :2] = inside[6][5]
    c["lens"][6] = 2
    c["penalties"][6] = (0.5, 0, 0)              # twice the largest value
    c["bias_ids"][7, 3] = inside[7][8000]
    c["bias_values"][7, 3] = np.inf
    c["x"][8, :] = torch.finfo(t).min            # the type's lowest value everywhere: a row like any other, but for its penalties
    c["lens"][8] = 0
    c["bias_ids"][8] = -1
    want, status = want_of(c, t)
    assert status.tolist() == [0, 0, 0, -1, -1, -1, -3, -3, 0]
    check(pkg, c, t)
    check(pkg, c, t, fill=-np.inf, lead=1, gap=2, out_lead=1, out_gap=2)


def test_a_result_that_only_the_bias_brings_back_into_range(pkg):
    """Rounding to the type is the last step: 60000 twice over, less 70000."""
    c = case(6, 1, 5000, torch.float16, history=4, biases=2)
    c["x"][0, 77] = 60000.0
    c["history"][:], c["lens"][:] = 77, 4
    c["penalties"][0] = (0.5, 0.0, 0.0)
    c["bias_ids"][0], c["bias_values"][0] = (77, -1), (-70000.0, 0.0)
    want, status = want_of(c, torch.float16)
    assert status[0] == 0 and want[0, 77] == 49984.0     # (50000 lies between two values, and goes to the even one)
    check(pkg, c, torch.float16)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [100, 129280])
def test_rejected_rows_are_nan_and_the_others_stand(pkg, dtype, vocab):
    t = TYPES[dtype]
    c = case(7, 8, vocab, t, per=2, history=50, biases=4, share=0.3)
    c["penalties"][0, 0], c["penalties"][1, 0], c["penalties"][2, 1], c["penalties"][3, 2] = 0.0, -1.0, np.nan, np.inf
    c["lens"][4], c["lens"][5] = -1, 51
    c["mask"][12] = 0
    c["mask"][15, :-1] = 0                       # only what is behind the last id
    c["mask"][15, -1] = 0 if vocab % 32 == 0 else np.uint32(2 ** 32 - 2 ** (vocab % 32))
    want, status = want_of(c, t)
    assert status.tolist() == [-11] * 8 + [-7] * 4 + [-2, 0, 0, -2]
    check(pkg, c, t)


def test_without_history_list_or_mask_rows_pass_unchanged(pkg):
    c = {"x": np.random.default_rng(1).normal(0, 3, (3, 5000)).astype(np.float32), "per": 1}
    c["x"][1, 7] = -0.0
    view = torch.from_numpy(c["x"]).cuda()
    got, st = pkg.constrain_logits(view)
    assert torch.equal(got, view) and st.cpu().tolist() == [0, 0, 0]
    got, st = pkg.constrain_logits(view[:1].expand(4, -1), repetition=1.2, history=torch.zeros(4, 0, dtype=torch.int32, device="cuda"))
    assert torch.equal(got, view[:1].expand(4, -1)) and st.cpu().tolist() == [0] * 4


def test_shared_logits_rows_and_rows_without_status(pkg):
    """One row of logits for every row of the call (stride 0), each under its own constraint."""
    c = case(8, 6, 70001, torch.float32, history=200, share=0.1)
    c["x"][:] = c["x"][0]
    want, status = want_of(c, torch.float32)
    row = torch.from_numpy(c["x"][:1]).cuda()
    got, st = call(pkg, c, row.expand(6, -1))
    assert same(got.cpu().numpy(), want) and st.cpu().tolist() == status.tolist()


def test_rows_side_by_side_in_one_buffer(pkg):
    """Input and output as the two halves of the same rows."""
    c = case(9, 4, 3001, torch.bfloat16, history=100, share=0.3)
    want, _ = want_of(c, torch.bfloat16)
    buf = torch.zeros(4, 6002, dtype=torch.bfloat16, device="cuda")
    buf[:, :3001] = torch.from_numpy(c["x"])
    got, _ = call(pkg, c, buf[:, :3001], out=buf[:, 3001:])
    assert same(got.float().cpu().numpy(), want) and same(buf[:, :3001].float().cpu().numpy(), c["x"])


def test_other_streams_and_captured_graphs(pkg):
    """Two calls at once on two streams, and a captured call replayed on new inputs."""
    cases = [case(20 + i, 30, 50000, torch.float32, history=3000, biases=30, share=0.2) for i in range(2)]
    wants = [want_of(c, torch.float32) for c in cases]
    tensors = [torch.from_numpy(c["x"]).cuda() for c in cases]
    outs = [torch.empty_like(t) for t in tensors]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for s, c, t, o in zip(streams, cases, tensors, outs):
        with torch.cuda.stream(s):
            call(pkg, c, t, out=o)
    torch.cuda.synchronize()
    for (want, _), o in zip(wants, outs):
        assert same(o.cpu().numpy(), want)
    cu = [{k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in c.items() if k not in ("x", "per")} for c in cases]
    kept, x, out, status = {k: v.clone() for k, v in cu[0].items()}, tensors[0].clone(), torch.empty_like(outs[0]), torch.empty(30, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    run = lambda: pkg.constrain_logits(x, history=kept["history"], history_len=kept["lens"], penalties=kept["penalties"],  # noqa: E731
                                       bias_ids=kept["bias_ids"], bias_values=kept["bias_values"], mask=kept["mask"], out=out, status=status)
    with torch.cuda.graph(graph):
        run()
    for i in (0, 1, 0):
        x.copy_(tensors[i])
        for k, v in kept.items():
            v.copy_(cu[i][k])
        graph.replay()
        torch.cuda.synchronize()
        assert same(out.cpu().numpy(), wants[i][0]) and status.cpu().tolist() == wants[i][1].tolist()


@pytest.mark.parametrize("rows,t,top_p,top_k", [(5, 0.8, 0.95, 0), (70, 0.8, 0.95, 0), (5, 0.7, 1.0, 0), (300, 0.0, 1.0, 0), (300, 0.9, 0.9, 20)])
def test_in_front_of_the_sampler(pkg, oracle, rows, t, top_p, top_k):
    """The rows that it leaves, sampled as plain rows by whichever path the batch takes, give the ids of the sampler's own constraints."""
    vocab, n = 129280, 400
    x = torch.from_numpy(oracle.gen_logits(31, rows, vocab)).cuda()
    history = torch.from_numpy(oracle.gen_history(32, rows, vocab, n)).cuda()
    mask = torch.from_numpy(oracle.gen_mask(33, rows, vocab).view(np.int32)).cuda()
    seeds, steps = torch.arange(rows, device="cuda") * 31 + 5, torch.arange(rows, device="cuda") + 2
    want, st = pkg.sample_logits(x, t, top_p, seeds, steps, top_k=top_k, history=history, repetition=1.1, presence=0.3, frequency=0.2, mask=mask)
    assert (st >= 0).all()
    y, st = pkg.constrain_logits(x, history=history, repetition=1.1, presence=0.3, frequency=0.2, mask=mask)
    assert (st == 0).all()
    got, st = pkg.sample_logits(y, t, top_p, seeds, steps, top_k=top_k)
    assert (st >= 0).all() and torch.equal(got, want)


@pytest.mark.parametrize("sequences", [2, 30])
def test_in_front_of_the_verifier(pkg, oracle, sequences):
    """A speculative step under penalties and a grammar: every row sees its sequence's history and the drafts in front of it, target and draft
    rows alike; the records are the oracle's on the constrained rows."""
    drafts, vocab, t, top = 2, 129280, 0.7, 0.95
    per = drafts + 1
    c = case(40, sequences, vocab, torch.float32, per, history=500, share=0.05)
    c["penalties"] = np.tile(np.float32([1.1, 0.3, 0.2]), (sequences, 1))
    x = oracle.gen_logits(41, sequences * per, vocab)
    c["x"] = x
    target, st = call(pkg, c, torch.from_numpy(x).cuda())
    assert (st == 0).all()
    d = dict(c, per=drafts, drafts=c["drafts"][:, :drafts - 1].copy(), mask=c["mask"].reshape(sequences, per, -1)[:, :drafts].reshape(sequences * drafts, -1).copy())
    raw = oracle.gen_perturbed(42, x.reshape(sequences, per, vocab)[:, :drafts].reshape(-1, vocab), sigma=0.3)
    draft, st = call(pkg, d, torch.from_numpy(raw).cuda())
    assert (st == 0).all()
    want_rows, _ = expected(x, torch.float32, c["history"], c["lens"], c["penalties"], c["drafts"], per, mask=c["mask"])
    assert same(target.cpu().numpy(), want_rows)
    seeds, steps = np.arange(sequences) * 7 + 3, np.arange(sequences) + 11
    u64 = lambda a: torch.from_numpy(np.asarray(a, np.uint64).view(np.int64)).cuda()  # noqa: E731
    ids = draft.argmax(1).int()
    results, status = pkg.verify_logits(target, draft, ids, drafts, t, top, u64(seeds), u64(steps))
    want, _ = oracle.verify_rows(target.cpu().numpy(), draft.cpu().numpy(), ids.cpu().numpy(), drafts, t, top, seeds, steps, threads=8)
    got = pkg.results_to_numpy(results)
    assert (status.cpu().numpy() >= 0).all()
    for name in ("emitted", "accepted_drafts", "rejected"):
        assert got[name].tolist() == want[name].tolist(), name
    for g, w in zip(got, want):
        assert g["tokens"][:g["emitted"]].tolist() == w["tokens"][:w["emitted"]].tolist()


def test_in_front_of_the_score_report(pkg, oracle):
    c = case(50, 4, 129280, torch.float32, history=300, share=0.02)
    y, _ = call(pkg, c, torch.from_numpy(c["x"]).cuda())
    lse, top1, ids, lp, st = pkg.score_logits(y, 10)
    assert (st == 0).all()
    rows = torch.where(torch.from_numpy(bits_of(c["mask"], 129280)).cuda(), y.double(), -np.inf)
    assert torch.allclose(lse, rows.logsumexp(1), rtol=1e-12, atol=0) and torch.equal(top1.long(), rows.argmax(1))


def test_refusals(pkg):
    x = torch.zeros(2, 64, device="cuda")
    with pytest.raises(ValueError):
        pkg.constrain_logits(x.cpu())
    with pytest.raises(ValueError):
        pkg.constrain_logits(x.double())
    with pytest.raises(ValueError):
        pkg.constrain_logits(x.t())
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, rows_per_sequence=3)
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, history=torch.zeros(3, 4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, history=torch.zeros(2, 4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, history_len=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, bias_ids=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, penalties=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        pkg.constrain_logits(x, out=torch.empty(2, 64, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="mask stride"):
        pkg.constrain_logits(x, mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="overlaps"):
        buf = torch.zeros(3, 64, device="cuda")
        pkg.constrain_logits(buf[:2], out=buf[1:])
    with pytest.raises(RuntimeError, match="penalties"):
        pkg.constrain_logits(x, repetition=0.0)
    with pytest.raises(RuntimeError, match="NaN"):
        pkg.constrain_logits(x, fill=float("nan"))
