"""Argument checks of ds41_b200_constrain_logits (all before any CUDA call; nothing is launched), its rule on small rows, and the source
rules of the kernels whose rows are shared by a team of CTAs."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from constrain_case import case, expected
from test_kernel_rules_cpu import CSRC, braced, enclosing, kernels, source, without_lambdas


@pytest.fixture(scope="module")
def pkg():
    entry.build()
    return entry.load_package()


def good(pkg, **changes):
    a = pkg.ConstrainArgs()
    a.struct_bytes = C.sizeof(pkg.ConstrainArgs)
    a.sequences, a.rows_per_sequence, a.vocab, a.dtype = 2, 3, 1000, 0
    a.logits, a.logits_stride, a.out, a.out_stride = 1 << 20, 1000, 1 << 24, 1000
    a.repetition, a.fill = 1.0, -3e38
    for k, v in changes.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("changes,message", [
    ({"struct_bytes": 8}, "ABI"), ({"sequences": 0}, "out of range"), ({"rows_per_sequence": 0}, "out of range"), ({"vocab": 0}, "out of range"),
    ({"vocab": 131073, "logits_stride": 140000, "out_stride": 140000}, "out of range"), ({"sequences": 1 << 20, "rows_per_sequence": 1 << 20}, "2^27"),
    ({"dtype": 3}, "FP32, BF16 or FP16"), ({"dtype": -1}, "FP32, BF16 or FP16"), ({"logits": None}, "null"), ({"out": None}, "null"),
    ({"logits_stride": 999}, "short stride"), ({"logits_stride": -1000}, "short stride"), ({"out_stride": 0}, "short stride"),
    ({"logits": (1 << 20) + 2}, "aligned"), ({"out": (1 << 24) + 1, "dtype": 1}, "aligned"),
    ({"out": (1 << 20) + 4000}, "overlaps"), ({"out": 1 << 20, "out_stride": 1001}, "overlaps"), ({"out": 1 << 20, "logits_stride": 0}, "overlaps"),
    ({"out": (1 << 20) - 23996}, "overlaps"), ({"out": (1 << 20) + 4 * 900, "logits_stride": 2000, "out_stride": 2000}, "overlaps"),
    ({"repetition": 0.0}, "penalties"), ({"repetition": float("nan")}, "penalties"), ({"presence": float("inf")}, "penalties"),
    ({"history": 1 << 12, "history_stride": -1}, "history"), ({"history": 1 << 12, "history_stride": 65536}, "history"),
    ({"biases": -1}, "biases"), ({"biases": 1025, "bias_ids": 1, "bias_values": 1}, "biases"), ({"biases": 1, "bias_ids": 1}, "no list"),
    ({"mask": 1 << 12, "mask_stride": 31}, "mask stride"), ({"fill": float("nan")}, "NaN")])
def test_arguments_are_refused_before_any_launch(pkg, changes, message):
    assert pkg.lib().ds41_b200_constrain_logits(C.byref(good(pkg, **changes)), None) == 1
    assert message in pkg.last_error(), pkg.last_error()
    assert pkg.lib().ds41_b200_constrain_logits(None, None) == 1


def test_tensors_without_a_device_are_refused(pkg):
    with pytest.raises(ValueError):
        pkg.constrain_logits(torch.zeros(2, 8))


def test_the_rule_on_a_row_by_hand():
    x = np.float32([[2.0, -2.0, 1.0, 0.5, 3.0]])
    out, status = expected(x, torch.float32, np.int32([[0, 1, 1, 9, -3]]), np.int32([5]), np.float32([[2.0, 0.5, 0.25]]),
                           bias_ids=np.int32([[2, 2, 4, -1]]), bias_values=np.float32([[1, 2, 5, 9]]), mask=np.uint32([[0b01111]]), fill=-np.inf)
    assert out.tolist() == [[0.25, -5.0, 4.0, 0.5, -np.inf]] and status.tolist() == [0]
    out, status = expected(np.repeat(x, 3, 0), torch.float32, penalties=np.float32([[1.0, 1.0, 0.0]]), drafts=np.int32([[3, 4]]), per=3)
    assert out[:, 3:].tolist() == [[0.5, 3.0], [-0.5, 3.0], [-0.5, 2.0]] and status.tolist() == [0, 0, 0]


def test_inputs_of_the_tests_hold_what_they_say():
    c = case(3, 4, 1031, torch.bfloat16, per=2, history=600, biases=40, share=0.01)
    assert (c["history"] < 0).any() and (c["history"] >= 1031).any() and c["lens"].tolist()[0] == 600 and c["lens"].tolist()[-1] == 0
    assert any(len(set(ids[ids >= 0].tolist())) < (ids >= 0).sum() for ids in c["bias_ids"])


TEAM_READ = re.compile(r"\bteam_read\(|\bteam_address\(")


def test_team_kernels_read_between_barriers():
    """Another CTA's shared memory is read behind a barrier of the whole team, and none leaves before a later one."""
    seen = set()
    for name, kernel, _, body in kernels():
        if "team_rank()" not in body:
            assert not TEAM_READ.search(body), (name, kernel)
            continue
        seen.add(kernel)
        if kernel == "constrain_kernel":          # its variant for few rows: two barriers at the end, the reads between them
            part = braced(body, body.index("if constexpr (kTeam) {"))
            assert not TEAM_READ.search(body.replace(part, "")) and "team_barrier" not in body.replace(part, "")
            barriers = [m.start() for m in re.finditer(r"\bteam_barrier\(\);", part)]
            reads = [m.start() for m in TEAM_READ.finditer(part)]
            assert len(barriers) == 2 and not any(enclosing(part, b) for b in barriers)
            assert barriers[0] < reads[0] and reads[-1] < barriers[1] and part.strip().endswith("team_barrier();")
        else:                                     # a barrier a turn, of both kinds of warps, and one behind the last turn
            head = "for (int turn = -1; turn <= turns; ++turn) {"
            loop = braced(body, body.index(head))
            behind = body[body.index(head) + len(head) + len(loop):]
            assert behind.strip("}; \n").endswith("if (p.team > 1) team_barrier()") and not re.search(r"\b(?:return|break);", without_lambdas(loop))
            listing = braced(loop, loop.index("if (warp >= kWarps) {"))
            first = braced(loop, loop.index("} else if (!has) {"))
            computing = loop[loop.index("} else if (!has) {") + len(first):]
            calls = lambda text: re.findall(r"if \(([^()]*(?:\([^()]*\))?[^()]*)\) team_(\w+)\(\);|\bteam_(\w+)\(\);", text)  # noqa: E731
            # every thread arrives once a turn that has a row, and waits once for it: in the same turn, or (the loss alone) in the next one
            assert calls(listing) == [("together && turn > 0", "wait", ""), ("together && has", "arrive", ""),
                                      ("kMode != kDistillLoss && together && has", "wait", "")]
            assert re.search(r"if \(kMode == kDistillLoss\) \{\s*if \(together && turn > 0\) team_wait\(\);", listing)
            assert calls(first) == [("kMode == kDistillLoss && together && turn > 0", "wait", "")]
            assert re.sub(r"\s+", " ", computing[computing.index("if (kMode == kDistillLoss) { if".split(" if")[0], computing.index("float rest_max")):]
                          ).startswith("if (kMode == kDistillLoss) { if (together) { if (turn > 0) team_wait(); team_arrive(); } } else if (together) { team_barrier(); }")
            assert [c[1] or c[2] for c in calls(computing)] == ["wait", "arrive", "barrier"]
            # the words that are read are written in front of the arrival, and again four turns on, when every reader has arrived for a later row
            assert computing.index("s.sums[turn & 3][warp] = ") < computing.index("team_wait();")
            assert len(TEAM_READ.findall(body)) == 1 and "team_read(&s.sums[turn & 3]" in braced(body, body.index("auto combine = "))
            assert listing.index("team_wait();") < listing.index("combine(turn - 1)") < listing.index("team_arrive();")
            assert computing.index("team_barrier();") < computing.index("combine(turn)") and body.count("combine(turn") == 2
            assert "const bool together = p.team > 1 && (kMode != kDistillGrad || p.in_place);" in body
    assert seen == {"constrain_kernel", "distill_kernel"}
    users = {n for n in os.listdir(CSRC) if n.endswith((".cu", ".cuh")) and "team_rank()" in source(n)}
    assert users == {"constrain.cu", "distill.cu", "row_team.cuh"}
