"""Workspaces of the paged-cache operators: what grows, and graphs captured before."""
import ctypes as C

import pytest

from test_gpu_ops import Attention, torch  # noqa: F401

from lrrt_b200 import native as N
from lrrt_b200.qwen import Runtime

pytestmark = pytest.mark.gpu


def frees():
    stats = N.MemoryStats()
    N.check(N.runtime().lr_get_memory_stats(Runtime.open_device(0), C.byref(stats)),
            "lr_get_memory_stats")
    return stats.free_count


def compact_many(torch, ops, pages):
    """A plan over `pages` pages of one row: its workspace takes 28 bytes for each."""
    keys, values = (torch.zeros(1, pages, 1, 1, 2, dtype=torch.float16, device="cuda")
                    for _ in range(2))
    table = torch.tensor([[pages - 1, 3]], dtype=torch.int32, device="cuda")
    got, status = ops.compact_pages(keys, values, table)
    assert got.tolist() == [[1, 0]] and status.tolist() == [2, 2]


def attend_many(torch, ops, sequences, heads=8):
    """Attention of `sequences` rows of one token: a counter for each of their heads."""
    keys, values = (torch.ones(1, 1, heads, 64, dtype=torch.float16, device="cuda")
                    for _ in range(2))
    q = torch.ones(sequences, heads, 64, dtype=torch.float16, device="cuda")
    table = torch.zeros(sequences, 1, dtype=torch.int32, device="cuda")
    lengths = torch.ones(sequences, dtype=torch.int32, device="cuda")
    return lambda: ops.paged_attention(q, keys, values, table, lengths)[0]


def test_growing_frees_nothing(gpu, torch):
    """Larger calls replace workspace and counters; nothing that a captured graph
    may use is freed before the operators are closed."""
    from lrrt_b200 import ops as module
    with module.Ops(0) as ops:
        before = frees()
        compact_many(torch, ops, 1000000)
        assert (attend_many(torch, ops, 6000)() == 1).all()
        compact_many(torch, ops, 3000000)
        assert frees() == before
    assert frees() == before + 5  # two sizes of counters, three of the workspace


def test_replay_after_growing(gpu, torch):
    """A graph of small steps, replayed after calls that outgrew the workspace
    and the counters, between further ones."""
    from lrrt_b200 import ops as module
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), module.Ops(0) as ops:
        case = Attention(torch, "bf16", [9000, 5, 4000, 777], 16, 2, 128, 32, seed=51)
        logits = torch.randn(2, 4, 30000, device="cuda")
        scores = torch.zeros(2, 4, device="cuda")

        def step():
            out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
            return (out, lse, *ops.beam_select(logits, scores, 4))

        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
        large = attend_many(torch, ops, 6000)
        for seed in range(4):
            compact_many(torch, ops, 400000 * (seed + 1))
            assert (large() == 1).all()
            torch.manual_seed(seed)
            logits.copy_(torch.randn(2, 4, 30000, device="cuda"))
            case.q.copy_(torch.randn_like(case.q))
            want = [t.clone() for t in step()]
            for t in captured:
                t.zero_()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(captured, want))
            assert (large() == 1).all()
        side.synchronize()
        del graph


def test_capture_that_would_grow(gpu, torch):
    """Refused while captured, and the stream and the operators are as before;
    with counters reserved the same call is captured."""
    from lrrt_b200 import ops as module
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), module.Ops(0) as ops:
        call = attend_many(torch, ops, 5000)
        attend_many(torch, ops, 2)()  # the kernel is loaded
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            torch.zeros(4, device="cuda")
            with pytest.raises(N.LrrtError, match="reserve"):
                call()
        ops.reserve(1 << 20, counters=5000 * 8)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call()
        for _ in range(2):
            out.zero_()
            graph.replay()
            assert (out == 1).all()
        side.synchronize()
        del graph
    queue, capturing = C.c_void_p(), C.c_uint32(7)
    N.check(N.runtime().lr_queue_is_capturing(Runtime.open_device(0), queue, C.byref(capturing)),
            "lr_queue_is_capturing")
    assert capturing.value == 0


def test_threads_share_operators(gpu, torch):
    """Threads that call one Ops on its stream, with sizes that outgrow its
    workspace and its counters on the way: each gets what it gets alone."""
    from concurrent.futures import ThreadPoolExecutor

    from lrrt_b200 import ops as module
    cases = [Attention(torch, kind, [9000, 5, 777], 16, 2, 64, 32, seed=53)
             for kind in ("f32", "bf16", "f16")]
    logits = torch.randn(2, 4, 30000, device="cuda")
    scores = torch.zeros(2, 4, device="cuda")

    def attend(case):
        return lambda ops: ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)

    calls = [attend(case) for case in cases]
    calls += [lambda ops: ops.beam_select(logits, scores, 4),
              lambda ops: (attend_many(torch, ops, 3000)(),),
              lambda ops: (attend_many(torch, ops, 7000)(),),
              lambda ops: (compact_many(torch, ops, 500000),),
              lambda ops: (ops.reserve(1 << 24, 70000),)]
    with module.Ops(0) as ops:
        want = [call(ops) for call in calls]
        torch.cuda.synchronize()
    with module.Ops(0) as ops, ThreadPoolExecutor(len(calls)) as pool:
        def run(i):
            return [[t if t is None else t.clone() for t in calls[i](ops)] for _ in range(15)]

        for got, expected in zip(pool.map(run, range(len(calls))), want):
            for each in got:
                assert all(a is b or torch.equal(a, b) for a, b in zip(each, expected))
    with pytest.raises(ValueError, match="closed"):
        ops.reserve(1)
