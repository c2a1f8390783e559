"""No warp of the weights' kernel on the tensor cores waits for good for one that gave up.  Nothing makes a wait run out on the GPU: the source is read, and the one barrier without a limit
is gone through in a model of four warps, in every order of their steps."""
import glob
import os
import re

import pytest
import torch

import flash_trittention as ft
from tests.test_eviction import DEV, Weighed

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-3-way-attention_b200", "csrc")


def _source():
    text = re.sub(r"//.*", "", open(os.path.join(CSRC, "tritt_sm100_tdp_weigh.cu")).read())
    kernel = text[text.index("tdp_weigh_sm100_kernel("):text.index("int launch(")]
    return kernel[kernel.index("if (warp < 4) {"):]


def test_waits_have_limits_but_for_one_barrier_that_is_left_in_turn():
    roles = _source()
    # the block's barrier: behind all of the warps' loops, where those that gave up come too
    assert len(re.findall(r"__syncthreads\(\)", roles)) == 1
    assert roles.index("__syncthreads()") > max(m.start() for m in re.finditer(r"next_item\(", roles))
    for unbounded in ("bar.sync", "barrier.sync", "__syncthreads_", "mbar_try_wait", "while (!"):
        assert unbounded not in roles, unbounded
    # a warpgroup's: behind it the flag is looked at, and who leaves because of the flag arrives once more
    assert len(re.findall(r"named_bar_sync\(", roles)) == 1 and len(re.findall(r"named_bar_arrive\(", roles)) == 1
    assert re.search(r"named_bar_sync\(1 \+ wg, 128\);\s*if \(__any_sync\(0xffffffffu, \*abort_flag\)\) break;", roles)
    assert re.search(r"\+\+pieces;\s*}\s*if \(__any_sync\(0xffffffffu, \*abort_flag\)\) named_bar_arrive\(1 \+ wg, 128\);\s*}", roles)


def _ends(arrive, look, pieces=3, warps=4):
    """Whether all warps get to the end, in whatever order they take their steps and wherever waits run out.  A warp is (barriers behind it, what it does): it works on a piece and may give up, which sets the flag, or comes to the
    barrier; behind the barrier it looks at the flag (with `look`); it leaves after the last piece or with the flag, and then arrives once more if the flag is set (with `arrive`)."""
    start = (tuple((0, "work") for _ in range(warps)), False, 0)   # ..., flag, arrivals at the barrier
    seen, todo = {start}, [start]
    while todo:
        state, flag, arrived = todo.pop()
        following = []
        for i, (behind, what) in enumerate(state):
            def put(new, flag=flag, arrived=arrived, i=i):
                ws = list(state)
                ws[i] = new
                if arrived == warps:   # complete: who waits goes on
                    ws, arrived = [(n + 1, "look") if w == "wait" else (n, w) for n, w in ws], 0
                following.append((tuple(ws), flag, arrived))
            if what == "work":
                if behind == pieces:
                    put((behind, "leave"))
                else:
                    put((behind, "wait"), arrived=arrived + 1)
                put((behind, "leave"), flag=True)    # (its wait ran out)
                if flag:
                    put((behind, "leave"))           # (a wait that ends because of the flag; it may also end well)
            elif what == "look":
                put((behind, "leave" if flag and look else "work"))
            elif what == "leave":
                put((behind, "end"), arrived=arrived + (flag and arrive))
        if not following and any(w != "end" for _, w in state):
            return False
        for s in following:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return True


def test_every_order_of_leaving_ends():
    assert _ends(True, True)
    assert not _ends(False, False) and not _ends(True, False) and not _ends(False, True)


def test_a_kernel_that_may_start_early_waits_for_the_one_ahead():
    """(Else the next one in the stream, which waits for it alone, starts beside the one ahead.)  Who returns ahead of the wait waits first, the first block at least."""
    kernels = 0
    for path in glob.glob(os.path.join(CSRC, "*.cu")):
        text = re.sub(r"//.*", "", open(path).read())
        for body in re.split(r"\n(?=template|__global__|}  // namespace)", text):
            if "__global__" not in body or "wait_for_previous();" not in body:
                continue
            kernels += 1
            last = body.rindex("wait_for_previous();")
            early = [m.start() for m in re.finditer(r"\breturn;", body[:last])]
            for at in early:
                assert re.search(r"(wait_for_previous\(\);\s*)$", body[:at]), (path, body[max(0, at - 100):at + 7])
    assert kernels >= 5


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 32])
def test_free_slots_alone_and_then_others_in_a_graph(D):
    """A call of a batch that has no sequence in use, and one whose scratch follows it."""
    idle, bt = Weighed(3, 2, 2, D, "bf16", "e4m3", 16, [-1, -1, -1], length=40), Weighed(2, 2, 2, D, "bf16", "e4m3", 16, [90, 41])
    table = torch.nn.functional.pad(bt.table, (0, 200), value=0)
    args = [(b.before.to(DEV), b.q.to(DEV), b.sums.to(DEV), b) for b in (idle, bt)]
    outs = [torch.full_like(a[0], 5.0) for a in args]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        for _ in range(3):
            for (before, q, sums, b), out in zip(args, outs):
                ft.tdp_weigh(before, q, sums, b.cache, table if b is bt else torch.zeros(3, 200, dtype=torch.int32, device=DEV), b.context, b.alpha, out=out)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    ft.check_status(DEV)
    assert bool((outs[0] == 5.0).all())
    bt.check(outs[1], stale=torch.full_like(bt.before, 5.0))
