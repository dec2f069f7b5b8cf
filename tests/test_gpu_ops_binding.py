"""The paged-cache operators' torch binding: what it refuses, and what it leaves alone."""
import pytest

from test_gpu_ops import Attention, ops, rope_case, torch  # noqa: F401

from lrrt_b200 import native as N

pytestmark = pytest.mark.gpu


def test_gradients_are_refused(ops, torch):
    """Inputs that require gradients, where these are recorded; not under no_grad."""
    case = Attention(torch, "f32", [5, 6], 4, 2, 64, 16)
    slopes = torch.zeros(4, device="cuda")
    rope = rope_case(torch, "f32", 3, 4, 2, 64, 64, 16)
    names = ("q", "k", "v", "keys", "values", "table", "sequences", "positions", "cos", "sin")
    logits, scores = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    own = lambda t: t.clone().requires_grad_()  # noqa: E731

    def attend(**changed):
        given = dict(q=case.q, keys=case.keys, values=case.values, slopes=slopes)
        return ops.paged_attention(table=case.table, lengths=case.n, **{**given, **changed})

    calls = [lambda name=name, t=t: attend(**{name: own(t)})
             for name, t in (("q", case.q), ("keys", case.keys), ("values", case.values),
                             ("slopes", slopes))]
    calls += [lambda name=name: ops.rope_append(*({**rope, name: own(rope[name])}[n]
                                                  for n in names))
              for name in ("q", "k", "v", "cos", "sin")]
    calls += [lambda: ops.beam_select(own(logits), scores, 3),
              lambda: ops.beam_select(logits, own(scores), 3)]
    for call in calls:
        with pytest.raises(ValueError, match="requires gradients"):
            call()
        with torch.no_grad():
            call()
    assert not attend()[0].requires_grad


def test_the_current_device_stays(gpu, torch):
    """Operators of one device, made and called while another is current."""
    from lrrt_b200 import ops as module
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    logits = torch.randn(1, 2, 500, device="cuda:1")
    scores = torch.zeros(1, 2, device="cuda:1")
    with torch.cuda.device(0):
        with module.Ops(1) as second:
            assert torch.cuda.current_device() == 0
            first = second.beam_select(logits, scores, 2)
            assert torch.cuda.current_device() == 0
            second.reserve(1 << 26, 100000)
            assert torch.cuda.current_device() == 0
            again = second.beam_select(logits, scores, 2)
        assert torch.cuda.current_device() == 0
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert torch.zeros(1, device="cuda").device.index == 0


def test_outputs_that_share_memory_are_refused(ops, torch):
    """Expanded outputs, rows that run into one another, tables inside tables."""
    case = Attention(torch, "bf16", [5, 6], 4, 2, 64, 16)
    attend = lambda out: ops.paged_attention(case.q, case.keys, case.values, case.table,  # noqa: E731
                                             case.n, out=out)
    rope = rope_case(torch, "f32", 3, 4, 2, 64, 64, 16)
    names = ("q", "k", "v", "keys", "values", "table", "sequences", "positions", "cos", "sin")

    def append(out=None, **changed):
        return ops.rope_append(*({**rope, **changed}[n] for n in names), out=out)

    pools = [torch.zeros(1, 8, 4, 2, 8, device="cuda") for _ in range(2)]
    tables = torch.zeros(6, 8, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(4, dtype=torch.int32, device="cuda")
    fork = lambda table, out: ops.fork_pages(*pools, table, lengths, lengths, table_out=out)  # noqa: E731
    compact = lambda table, out: ops.compact_pages(*pools, table, table_out=out)  # noqa: E731
    b16 = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    f32 = lambda *shape: torch.zeros(*shape, device="cuda")  # noqa: E731
    keys = rope["keys"]
    for call, text in [
        (lambda: attend(b16(1, 4, 64).expand(2, 4, 64)), "share memory"),
        (lambda: attend(b16(2, 1, 64).expand(2, 4, 64)), "share memory"),
        (lambda: attend(b16(1000).as_strided((2, 4, 64), (200, 64, 1))), "share memory"),
        (lambda: append(f32(1, 4, 64).expand(3, 4, 64)), "share memory"),
        (lambda: append(f32(2000).as_strided((3, 4, 64), (256, 60, 1))), "share memory"),
        (lambda: append(keys=keys[:1].expand_as(keys)), "keys share memory"),
        (lambda: append(values=keys[:, :, :1].expand_as(keys)), "values share memory"),
        (lambda: fork(tables[:4], tables[1:5]), "share memory"),
        (lambda: fork(tables[:4, :5], tables[:4, 3:8]), "share memory"),
        (lambda: fork(tables[:4, :5], tables.flatten()[4:24].reshape(4, 5)), "share memory"),
        (lambda: fork(tables[:4], tables.new_zeros(1, 8).expand(4, 8)), "share memory"),
        (lambda: compact(tables[:4], tables[2:6]), "shares memory"),
        (lambda: compact(tables[:4], tables.new_zeros(1, 8).expand(4, 8)), "share memory"),
    ]:
        with pytest.raises((N.LrrtError, ValueError), match=text):
            call()
    rows = b16(3, 4, 64)
    with pytest.raises(ValueError, match="partly in q"):
        ops.paged_attention(rows[:2], case.keys, case.values, case.table, case.n, out=rows[1:])
    packed = f32(4, 4, 64)
    with pytest.raises(ValueError, match="partly in q"):
        append(packed[1:], q=packed[:3])


def test_outputs_beside_inputs(ops, torch):
    """Halves of one buffer, woven and turned layouts, and q itself are no overlap."""
    case = Attention(torch, "bf16", [9000, 40, 0, 700, 5], 16, 2, 64, 16, seed=55)
    call = lambda q, out: ops.paged_attention(q, case.keys, case.values, case.table,  # noqa: E731
                                              case.n, out=out)[0]
    want = call(case.q, None)
    both = torch.zeros(5, 32, 64, dtype=torch.bfloat16, device="cuda")
    both[:, :16] = case.q
    assert torch.equal(call(both[:, :16], both[:, 16:]), want)
    woven = torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    woven[:, :, 0] = case.q
    assert torch.equal(call(woven[:, :, 0], woven[:, :, 1]), want)
    turned = torch.zeros(16, 5, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(call(case.q, turned), want)
    for _ in range(3):
        mine = case.q.clone()
        assert call(mine, mine) is mine and torch.equal(mine, want)
    pools = [torch.zeros(1, 8, 4, 2, 8, device="cuda") for _ in range(2)]
    table = torch.zeros(4, 10, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(4)
    lengths = torch.full((4,), 3, dtype=torch.int32, device="cuda")
    got, _, _ = ops.fork_pages(*pools, table[:, :5], lengths, torch.arange(4).int().cuda(),
                               table_out=table[:, 5:])
    assert got[:, 0].tolist() == [0, 1, 2, 3] and (got[:, 1:] == -1).all()
    got, _ = ops.compact_pages(*pools, table[:, 5:], table_out=table[:, 5:])
    assert got[:, 0].tolist() == [0, 1, 2, 3]


def test_pools_whose_pages_share_memory_are_refused(ops, torch):
    """Expanded layers or pages; pages of one layer, and pages woven with others'
    by layer, are as they were."""
    one = torch.randn(2, 8, 4, 2, 8, device="cuda")
    table = torch.tensor([[7, 2], [5, -1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([8, 3], dtype=torch.int32, device="cuda")
    both = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for pool in (one[:1].expand(2, 8, 4, 2, 8), one[:, :1].expand(2, 8, 4, 2, 8)):
        for call in (lambda p: ops.fork_pages(p, p, table, lengths, both),
                     lambda p: ops.compact_pages(p, p, table),
                     lambda p: ops.copy_pages(p, p, both, both + 2)):
            with pytest.raises(N.LrrtError, match="share memory"):
                call(pool)
    woven = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    for view in (torch.clone, woven, lambda x: woven(x)[:, ::2], lambda x: x.clone()[:, :, :2],
                 lambda x: x[:1].clone()):  # woven: [pages][layers] in memory
        keys, values = view(one), view(one)
        want = keys.clone()
        want[:, 2:4] = keys[:, :2]
        ops.copy_pages(keys, values, both, both + 2)
        assert torch.equal(keys, want) and torch.equal(values, want)
