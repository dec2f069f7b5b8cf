"""The paged-cache operators on a B200 against plain implementations in 64 bits.

Bounds are derived from the arithmetic, not from runs: ROUND is half a unit in
the last place of an output's type (relative), FLOAT that of 32 bits.
"""
import math

import numpy as np
import pytest

from lrrt_b200 import native as N

pytestmark = pytest.mark.gpu

FLOAT = 2.0 ** -24
ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# Below the smallest normal number of f16 its rounding is absolute.
LEAST = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def torch(gpu):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(gpu, torch):
    from lrrt_b200 import ops as module
    with module.Ops(0) as handle:
        yield handle


def dtype_of(torch, kind):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]


def close(actual, want, bound, what=""):
    """|actual - want| <= bound everywhere; infinities have to be equal."""
    actual, want = actual.double().cpu(), want.double().cpu()
    finite = want.isfinite()
    assert (actual[~finite] == want[~finite]).all(), what
    error = (actual - want).abs()[finite]
    limit = bound.double().cpu().expand_as(want)[finite]
    worst = (error - limit).max().item() if error.numel() else 0.0
    assert worst <= 0 and not error.isnan().any(), f"{what}: over the bound by {worst}"


# --- attention ----------------------------------------------------------------

class Attention:
    """A paged cache whose unread rows, and pages that no table names, are NaN."""

    def __init__(self, torch, kind, lengths, heads, kv_heads, dim, page, layout="token", seed=0,
                 spread=1.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        dtype = dtype_of(torch, kind)
        self.torch, self.kind, self.page, self.kv_heads = torch, kind, page, kv_heads
        self.heads, self.dim, self.lengths = heads, dim, lengths
        width = max([1] + [-(-n // page) for n in lengths]) + 1
        used = sum(-(-n // page) for n in lengths)
        pages = used + 2
        order = torch.randperm(pages, generator=g, device="cuda")
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
        at = 0
        shape = (pages, page, kv_heads, dim) if layout == "token" else (pages, kv_heads, page, dim)
        self.keys, self.values = (torch.full(shape, math.nan, dtype=dtype, device="cuda")
                                  for _ in range(2))
        if layout == "head":
            self.keys, self.values = self.keys.transpose(1, 2), self.values.transpose(1, 2)
        for row, n in enumerate(lengths):
            count = -(-n // page)
            mine = order[at:at + count]
            at += count
            self.table[row, :count] = mine.int()
            # Past the pages: numbers that are out of range, or of other rows' pages.
            self.table[row, count:] = -7 if row % 2 else pages
            j = torch.arange(n, device="cuda")
            for pool in (self.keys, self.values):
                x = torch.randn(n, kv_heads, dim, generator=g, device="cuda") * spread
                pool[mine[j // page], j % page] = x.to(dtype)
        self.q = (torch.randn(len(lengths), heads, dim, generator=g, device="cuda")
                  * spread).to(dtype)
        self.n = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def expected(self, scale=None, softcap=0.0, slopes=None, window=0):
        """(out, lse, bound of out, bound of lse) in 64 bits.

        A score is off by at most e = 2^-19 of the sum of its products'
        magnitudes (the products' own rounding, 2^-21 in 32 bits, and the sums
        in 32 bits of at most 256 of them in any order), plus 2^-22 of its
        size for the steps that follow; its weight then by a factor of exp(e).
        The weights' own arithmetic and rounding adds 2^-16 where they are
        held in 16-bit pieces, 2^-20 in 32 bits. The output is off by at most
        twice the relative error of the weights times the largest value, and
        its rounding.
        """
        torch = self.torch
        outs, sums, bounds, sum_bounds = [], [], [], []
        scale = self.dim ** -0.5 if scale is None else scale
        group = self.heads // self.kv_heads
        pieces = 2.0 ** -20 if self.kind == "f32" else 2.0 ** -16
        for row, n in enumerate(self.lengths):
            j = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
            page = self.table[row, j // self.page].long()
            there = (page >= 0) & (page < self.keys.shape[0])
            j, page = j[there], page[there]
            k = self.keys[page, j % self.page].double().repeat_interleave(group, 1)
            v = self.values[page, j % self.page].double().repeat_interleave(group, 1)
            q = self.q[row].double()
            x = torch.einsum("hd,jhd->hj", q, k) * scale
            size = torch.einsum("hd,jhd->hj", q.abs(), k.abs()) * abs(scale)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - slopes.double()[:, None] * (n - 1 - j)
            lse = torch.logsumexp(x, -1) if j.numel() else torch.full((self.heads,), -math.inf)
            out = torch.einsum("hj,jhd->hd", torch.softmax(x, -1), v)
            e = (2.0 ** -19 * size + 2.0 ** -22 * x.abs()).amax(-1) if j.numel() else \
                torch.zeros(self.heads, dtype=torch.float64, device="cuda")
            most = v.abs().amax(0).amax(-1) if j.numel() else torch.zeros_like(e)
            outs.append(out)
            sums.append(lse.cuda())
            bounds.append((2 * (e + pieces) * most)[:, None] + ROUND[self.kind] * out.abs() * 1.01 +
                          LEAST[self.kind])
            sum_bounds.append(e + pieces + 4 * FLOAT * lse.cuda().abs().nan_to_num(posinf=0))
        return [torch.stack(x) for x in (outs, sums, bounds, sum_bounds)]

    def check(self, ops, **options):
        out, lse = ops.paged_attention(self.q, self.keys, self.values, self.table, self.n,
                                       **options)
        want, want_lse, bound, lse_bound = self.expected(**options)
        close(out, want, bound, "out")
        close(lse, want_lse, lse_bound, "lse")
        return out, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 0, 255, 256, 257, 511, 700]


@pytest.mark.parametrize("kind,dim,heads,kv_heads,page", [
    ("f32", 64, 14, 2, 16), ("f32", 64, 24, 2, 32), ("f32", 128, 8, 1, 20), ("f32", 96, 3, 3, 1),
    ("f32", 128, 24, 2, 64), ("bf16", 64, 16, 2, 16), ("bf16", 64, 12, 1, 64),
    ("bf16", 128, 32, 8, 64), ("bf16", 128, 16, 1, 7), ("bf16", 256, 8, 2, 16),
    ("bf16", 256, 20, 1, 128), ("bf16", 80, 10, 2, 24), ("f16", 128, 5, 5, 1),
    ("f16", 64, 40, 2, 48), ("f16", 8, 4, 4, 16), ("f16", 200, 17, 1, 33),
])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_attention_shapes(ops, torch, kind, dim, heads, kv_heads, page, layout):
    Attention(torch, kind, EDGES, heads, kv_heads, dim, page, layout).check(ops)


@pytest.mark.parametrize("kind,dim,heads,kv_heads,page", [
    ("f32", 72, 10, 2, 8), ("f32", 96, 24, 2, 16), ("f32", 88, 8, 1, 48), ("bf16", 72, 16, 1, 16),
    ("bf16", 96, 14, 2, 8), ("f16", 88, 36, 3, 32), ("f16", 80, 3, 3, 1), ("bf16", 104, 12, 1, 24),
])
def test_attention_between_widths(ops, torch, kind, dim, heads, kv_heads, page):
    """Heads of 65 to 127 elements, tiles of one page and of several."""
    Attention(torch, kind, EDGES, heads, kv_heads, dim, page, seed=23).check(ops, window=300)


@pytest.mark.parametrize("kind,dim", [("f32", 128), ("f32", 64), ("bf16", 64), ("f16", 256)])
@pytest.mark.parametrize("page", [8, 16, 32])
def test_attention_repeated_pages(ops, torch, kind, dim, page):
    """A page that a sequence names twice, side by side: the same rows again."""
    case = Attention(torch, kind, [100, 400, 64], 8, 2, dim, page, seed=25)
    case.table[:, 1] = case.table[:, 0]
    case.table[1, 3:6] = case.table[1, 2]
    case.check(ops)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("spread", [0.01, 1.0, 12.0])
def test_attention_wide_cap(ops, torch, kind, spread):
    """Scores far below the cap and far above it. Beside the other errors a
    capped score has that of 1 - 2 / (1 + e^2x): two units in the last place of
    the exponential (2^-22), one of the reciprocal (2^-23), twice over: at most
    2^-20 of the cap."""
    cap = 50.0
    case = Attention(torch, kind, [1, 40, 700, 2500], 16, 2, 96, 16, seed=27, spread=spread)
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n, softcap=cap)
    want, want_lse, bound, lse_bound = case.expected(softcap=cap)
    most = case.values[~case.values.isnan()].abs().max().double()
    close(out, want, bound + 2 * 2.0 ** -20 * cap * most, "out")
    close(lse, want_lse, lse_bound + 2.0 ** -20 * cap, "lse")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("options", [
    dict(softcap=5.0), dict(window=1), dict(window=33), dict(window=100000), dict(scale=0.7),
    dict(scale=0.0), dict(scale=-0.3), "slopes", "all",
])
def test_attention_scores(ops, torch, kind, options):
    case = Attention(torch, kind, EDGES, 14, 2, 64, 16, seed=3)
    if isinstance(options, str):
        # Some of the slopes are negative: distance may raise a score too.
        slopes = torch.linspace(-0.01, 0.5, 14, device="cuda")
        options = dict(slopes=slopes) if options == "slopes" else \
            dict(slopes=slopes, softcap=3.0, window=200, scale=0.5)
    case.check(ops, **options)


@pytest.mark.parametrize("kind,lengths", [
    ("f32", [40000]), ("bf16", [70001, 3]), ("f16", [0, 33333, 1, 20000]),
    ("bf16", [5] * 700), ("bf16", [0] * 50), ("f32", [1]),
    ("bf16", [4096] * 37), ("f16", list(range(0, 1300, 7))),
])
def test_attention_splits(ops, torch, kind, lengths):
    """Rows split over many blocks, blocks over many rows, and both."""
    Attention(torch, kind, lengths, 8, 2, 128, 64, seed=5).check(ops)


def test_attention_large_scores(ops, torch):
    """Scores far apart: the running maximum has to be followed."""
    for kind in ("f32", "bf16", "f16"):
        Attention(torch, kind, [1, 50, 700, 3000], 8, 1, 64, 16, seed=7, spread=6.0).check(ops)


def test_attention_missing_pages(ops, torch):
    """Entries out of range inside a sequence are skipped, a row of nothing
    else sees no token."""
    case = Attention(torch, "bf16", [100, 300, 64, 2000], 8, 2, 128, 16, seed=9)
    case.table[0, 2] = -1
    case.table[1, :] = -1
    case.table[2, 0] = 10 ** 9
    case.table[3, 3::5] = case.keys.shape[0]
    out, lse = case.check(ops)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_attention_lengths_are_clamped(ops, torch):
    case = Attention(torch, "f16", [64, 64], 4, 2, 64, 16, seed=11)
    case.table = case.table[:, :4].contiguous()
    want, _ = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    n = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, n)
    assert torch.equal(out[0], want[0])
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_attention_infinite_and_nan_values(ops, torch):
    """A NaN that is read shows in its heads and rows alone; one past the end
    does not (every case's unread rows are NaN)."""
    case = Attention(torch, "bf16", [40, 40], 8, 2, 64, 16, seed=13)
    case.keys[case.table[0, 1].long(), 3, 1] = math.nan
    out, _ = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    assert out[0, 4:].isnan().all() and out[0, :4].isfinite().all() and out[1].isfinite().all()


def test_attention_strides(ops, torch):
    """Queries inside packed rows, the output into a wider one, keys and values
    in one pool with different strides, a table with a stride of its own."""
    case = Attention(torch, "bf16", [100, 33, 0, 257], 8, 2, 64, 16, seed=15)
    pages = case.keys.shape[0]
    both = torch.full((pages, 2, 16, 2, 72), math.nan, dtype=torch.bfloat16, device="cuda")
    both[:, 0, :, :, :64], both[:, 1, :, :, :64] = case.keys, case.values
    case.keys, case.values = both[:, 0, :, :, :64], both[:, 1, :, :, :64]
    packed = torch.zeros(4, 12, 65, dtype=torch.bfloat16, device="cuda")
    packed[:, 1:9, 1:] = case.q
    case.q = packed[:, 1:9, 1:]
    wide = torch.full((4, case.table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 3:-2] = case.table
    case.table = wide[:, 3:-2]
    out = torch.full((4, 9, 65), 7.0, dtype=torch.bfloat16, device="cuda")
    case.check(ops, **{})
    ops.paged_attention(case.q, case.keys, case.values, case.table, case.n, out=out[:, :8, :64])
    want, _, bound, _ = case.expected()
    close(out[:, :8, :64], want, bound)
    assert (out[:, 8] == 7).all() and (out[:, :, 64] == 7).all()


def test_attention_repeats(ops, torch):
    """The same bits again, with other calls between: nothing depends on timing
    or is left behind."""
    case = Attention(torch, "bf16", [9000, 5, 0, 4000, 777], 16, 2, 128, 32, seed=17)
    other = Attention(torch, "f32", [3000, 1], 14, 2, 64, 16, seed=18)
    first, first_lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    for _ in range(20):
        ops.paged_attention(other.q, other.keys, other.values, other.table, other.n)
        out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


def test_attention_offsets_past_32_bits(ops, torch):
    """A pool of more than 2^32 elements; the pages in use lie at its end."""
    pages, page, kv_heads, dim = 66000, 64, 8, 128
    keys, values = (torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
                    for _ in range(2))
    assert keys.numel() > 2 ** 32
    case = Attention(torch, "bf16", [200, 129], 16, 8, 128, 64, seed=19)
    high = torch.arange(pages - case.keys.shape[0], pages, device="cuda")
    keys[high], values[high] = case.keys, case.values
    inside = (case.table >= 0) & (case.table < case.keys.shape[0])
    case.table = torch.where(inside, case.table + (pages - case.keys.shape[0]), -1).int()
    case.keys, case.values = keys, values
    case.check(ops)


def test_attention_without_rows(ops, torch):
    case = Attention(torch, "bf16", [5], 4, 2, 64, 16)
    out, lse = ops.paged_attention(case.q[:0], case.keys, case.values, case.table[:0], case.n[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_attention_refuses(ops, torch):
    case = Attention(torch, "bf16", [5, 6], 4, 2, 64, 16)
    call = lambda **k: ops.paged_attention(**{**dict(q=case.q, keys=case.keys, values=case.values,  # noqa: E731
                                                     table=case.table, lengths=case.n), **k})
    for bad, text in [
        (dict(q=case.q.float()), "q is"), (dict(q=case.q.cpu()), "on cpu"),
        (dict(q=case.q[:1]), "rows"), (dict(lengths=case.n.long()), "lengths"),
        (dict(lengths=case.n[:1]), "lengths has"), (dict(values=case.values[:1]), "differ"),
        (dict(values=case.values.half()), "values is"), (dict(window=-1), "window"),
        (dict(q=case.q[..., :32]), "head_dim"), (dict(table=case.table.long()), "table"),
        (dict(q=case.q.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
        (dict(slopes=torch.zeros(3, device="cuda")), "slopes"),
        (dict(keys=case.keys.to(torch.float64)), "a cache of"),
    ]:
        with pytest.raises(ValueError, match=text):
            call(**bad)
    odd = torch.zeros(4, 16, 2, 68, dtype=torch.bfloat16, device="cuda")[..., :64]
    wide = torch.zeros(4, 16, 2, 264, dtype=torch.bfloat16, device="cuda")
    for bad, text in [
        (dict(softcap=-1.0), "softcap"), (dict(softcap=math.inf), "softcap"),
        (dict(scale=math.nan), "scale"), (dict(q=case.q[:, :3]), "multiple of kv_heads"),
        (dict(keys=odd, values=odd), "16 bytes"),
        (dict(keys=wide, values=wide, q=torch.zeros(2, 4, 264, dtype=torch.bfloat16,
                                                    device="cuda")), "head_dim"),
    ]:
        with pytest.raises(N.LrrtError, match=text):
            call(**bad)
    large = torch.zeros(2, 16, 2, 136, device="cuda")
    with pytest.raises(N.LrrtError, match="128 in 32 bits"):
        call(q=torch.zeros(2, 4, 136, device="cuda"), keys=large, values=large)


# --- rotary positions and append ------------------------------------------------

def rope_case(torch, kind, tokens, heads, kv_heads, dim, rotary, page, batch=3, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = dtype_of(torch, kind)
    from lrrt_b200 import ops as module
    longest = tokens + 50
    width = -(-longest // page)
    pages = batch * width + 1
    case = {
        "packed": torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g,
                              device="cuda").to(dtype),
        "keys": torch.zeros(pages, page, kv_heads, dim, dtype=dtype, device="cuda"),
        "values": torch.zeros(pages, page, kv_heads, dim, dtype=dtype, device="cuda"),
        "table": torch.randperm(pages, generator=g, device="cuda")[:batch * width].int()
        .reshape(batch, width).contiguous(),
    }
    sequence = torch.randint(0, batch, (tokens,), generator=g, device="cuda")
    # Distinct places: position t + offset of its sequence.
    case["positions"] = (torch.arange(tokens, device="cuda") +
                         torch.tensor([0, 7, 50], device="cuda")[sequence % 3]).int()
    case["sequences"] = sequence.int()
    case["cos"] = case["sin"] = None
    if rotary:
        cos, sin = module.rope_tables(longest, rotary, 1e4)
        case["cos"], case["sin"] = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    case["q"], case["k"], case["v"] = case["packed"].split([heads, kv_heads, kv_heads], 1)
    return case


def rope_expected(torch, case, x, rotary, interleaved, kind):
    """(turned, bound) in 64 bits: three roundings of 32 bits of the two products' size."""
    at = case["positions"].long()
    y = x.double().clone()
    bound = y.abs() * 0
    if rotary:
        cos, sin = (case[n].double()[at][:, None, :] for n in ("cos", "sin"))
        first, second = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else \
            (slice(0, rotary // 2), slice(rotary // 2, rotary))
        a, b = x[..., first].double(), x[..., second].double()
        y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
        size = (a.abs() + b.abs())
        bound[..., first] = bound[..., second] = 3 * FLOAT * size
        bound += ROUND[kind] * 1.01 * y.abs() + LEAST[kind]
        bound[..., rotary:] = 0  # copied
    return y, bound


@pytest.mark.parametrize("kind,tokens,heads,kv_heads,dim,rotary,page", [
    ("f32", 1, 14, 2, 64, 64, 16), ("f32", 33, 14, 2, 64, 32, 1), ("f32", 7, 3, 1, 30, 14, 5),
    ("f32", 5, 2, 2, 64, 0, 16), ("bf16", 1, 32, 8, 128, 128, 64), ("bf16", 300, 8, 2, 128, 64, 20),
    ("bf16", 17, 10, 2, 80, 40, 24), ("bf16", 9, 4, 1, 66, 22, 3), ("f16", 257, 4, 4, 96, 48, 16),
    ("f16", 64, 7, 1, 256, 256, 32), ("f16", 3, 1, 1, 2, 2, 1), ("bf16", 2048, 28, 4, 64, 64, 16),
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append(ops, torch, kind, tokens, heads, kv_heads, dim, rotary, page, interleaved):
    case = rope_case(torch, kind, tokens, heads, kv_heads, dim, rotary, page)
    q = ops.rope_append(case["q"], case["k"], case["v"], case["keys"], case["values"],
                        case["table"], case["sequences"], case["positions"], case["cos"],
                        case["sin"], interleaved=interleaved)
    want, bound = rope_expected(torch, case, case["q"], rotary, interleaved, kind)
    close(q, want, bound, "q")
    keys, values = (torch.zeros_like(case["keys"], dtype=torch.float64) for _ in range(2))
    limit = torch.zeros_like(keys)
    at = case["positions"].long()
    place = (case["table"].long()[case["sequences"].long(), at // page], at % page)
    want, bound = rope_expected(torch, case, case["k"], rotary, interleaved, kind)
    keys[place], limit[place], values[place] = want, bound, case["v"].double()
    close(case["keys"], keys, limit, "keys")
    assert torch.equal(case["values"].double(), values)


@pytest.mark.parametrize("kind,heads,kv_heads,dim,rotary", [
    ("bf16", 6, 2, 40, 40), ("f16", 4, 1, 72, 24), ("bf16", 3, 3, 56, 8), ("f16", 2, 1, 96, 88),
    ("f16", 5, 1, 20, 8),
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_halves_of_odd_vectors(ops, torch, kind, heads, kv_heads, dim, rotary, interleaved):
    """Halves of a multiple of four elements beside copies of a multiple of eight."""
    test_rope_append(ops, torch, kind, 37, heads, kv_heads, dim, rotary, 12, interleaved)



def test_rope_append_in_place_and_padding(ops, torch):
    case = rope_case(torch, "bf16", 12, 8, 2, 64, 64, 16, seed=2)
    case["sequences"][3] = -1          # no sequence
    case["sequences"][4] = 3           # past the table
    case["positions"][5] = -2          # no position
    case["positions"][6] = 10 ** 6     # past the tables
    case["table"][case["sequences"][7].long(), case["positions"][7].long() // 16] = -1
    padding = torch.zeros(12, dtype=torch.bool, device="cuda")
    padding[3:8] = True
    for other in range(12):            # others may share the page that is gone
        s, p = case["sequences"][other].item(), case["positions"][other].item()
        if 0 <= s < 3 and 0 <= p < case["cos"].shape[0] and case["table"][s, p // 16] < 0:
            padding[other] = True
    source = case["packed"].clone()
    q = ops.rope_append(case["q"], case["k"], case["v"], case["keys"], case["values"],
                        case["table"], case["sequences"], case["positions"], case["cos"],
                        case["sin"], out=case["q"])
    assert q is case["q"]
    assert torch.equal(case["packed"][:, 8:], source[:, 8:])  # keys and values are as they were
    keep = ~padding
    case["positions"] = torch.where(keep, case["positions"], 0)
    want, bound = rope_expected(torch, case, source[:, :8], 64, False, "bf16")
    close(q[keep], want[keep], bound[keep])
    assert (q[padding] == 0).all()
    written = (case["keys"] != 0).any(-1).any(-1).sum().item()
    assert written == keep.sum().item()


def test_rope_append_without_sequences(ops, torch):
    """One token per sequence: their numbers may be left out."""
    case = rope_case(torch, "f32", 3, 4, 2, 64, 64, 16, seed=4)
    case["sequences"] = torch.arange(3, dtype=torch.int32, device="cuda")
    arguments = [case[n] for n in ("q", "k", "v")]
    pools = [[torch.zeros_like(case[n]) for n in ("keys", "values")] for _ in range(2)]
    rest = [case[n] for n in ("positions", "cos", "sin")]
    a = ops.rope_append(*arguments, *pools[0], case["table"], case["sequences"], *rest)
    b = ops.rope_append(*arguments, *pools[1], case["table"], None, *rest)
    assert torch.equal(a, b)
    assert all(torch.equal(x, y) for x, y in zip(*pools))


def test_rope_append_no_tokens(ops, torch):
    case = rope_case(torch, "f32", 3, 4, 2, 64, 64, 16)
    q = ops.rope_append(*(case[n][:0] for n in ("q", "k", "v")), case["keys"], case["values"],
                        case["table"], case["sequences"][:0], case["positions"][:0], case["cos"],
                        case["sin"])
    assert q.shape == (0, 4, 64)


def test_rope_append_refuses(ops, torch):
    case = rope_case(torch, "f32", 3, 4, 2, 64, 64, 16)
    names = ("q", "k", "v", "keys", "values", "table", "sequences", "positions", "cos", "sin")
    call = lambda **k: ops.rope_append(*({**case, **k}[n] for n in names))  # noqa: E731
    for bad, text in [
        (dict(q=case["q"].half()), "q is"), (dict(k=case["k"][:2]), "k has"),
        (dict(v=case["v"][:, :1]), "v has"), (dict(sin=case["sin"][:4]), "one shape"),
        (dict(positions=case["positions"][:1]), "positions has"),
        (dict(sequences=case["sequences"].long()), "sequences is"),
    ]:
        with pytest.raises(ValueError, match=text):
            call(**bad)
    wide = torch.zeros(60, 40, device="cuda")
    with pytest.raises(N.LrrtError, match="rotary_dim"):
        call(cos=wide, sin=wide)


# --- pages ----------------------------------------------------------------------

def fork_expected(pool, table, lengths, parents, room, held=None):
    """The rules of lro_pages_fork, one row after another."""
    pages, page, columns = pool.shape[1], pool.shape[2], table.shape[1]
    pool = pool.copy()
    rows = []
    for p in parents:
        alive = 0 <= p < len(lengths)
        n = min(max(int(lengths[p]), 0), columns * page) if alive else 0
        have = -(-n // page)
        entries = [int(x) if 0 <= x < pages else -1 for x in (table[p, :have] if alive else [])]
        rows.append((alive, n, entries))
    whole = set(np.nonzero(held)[0].tolist()) if held is not None else set()
    for _, n, entries in rows:
        whole |= set(entries[:n // page]) - {-1}
    owner = {}
    for s, (_, n, entries) in enumerate(rows):
        if n % page and entries[-1] >= 0:
            owner.setdefault(entries[-1], s)
    free = [x for x in range(pages) if x not in whole and x not in owner]
    missing, moves, out = 0, [], np.full((len(parents), columns), -1, np.int32)
    taken = 0
    for s, (alive, n, entries) in enumerate(rows):
        entries = list(entries)
        copy = bool(n % page and entries[-1] >= 0 and
                    (entries[-1] in whole or owner[entries[-1]] != s))
        need = min(-(-(n + room) // page), columns) if alive else 0
        wanted = list(range(len(entries), need))
        if copy:
            wanted.insert(0, len(entries) - 1)
        source = entries[-1] if entries else -1
        entries += [-1] * (need - len(entries))
        for column in wanted:
            got = free[taken] if taken < len(free) else -1
            missing += got < 0
            taken += 1
            entries[column] = got
        if copy and entries[n // page] >= 0:
            moves.append((source, entries[n // page], n % page))
        out[s, :len(entries)] = entries
    before = pool.copy()
    for source, target, count in moves:
        pool[:, target, :count] = before[:, source, :count]
    return pool, out, np.array([n for _, n, _ in rows], np.int32), \
        np.array([missing, max(0, len(free) - taken)], np.int32)


def page_pool(torch, kind, layers, pages, page, heads, dim, layout="token"):
    shape = (layers, pages, page, heads, dim) if layout == "token" else \
        (layers, pages, heads, page, dim)
    pools = [torch.randn(shape, device="cuda").to(dtype_of(torch, kind)) for _ in range(2)]
    return [p.transpose(2, 3) if layout == "head" else p for p in pools]


def random_table(rng, lengths, page, pages, columns, sharing):
    """Rows of distinct pages; with `sharing`, some begin as an earlier row does."""
    order = list(rng.permutation(pages))
    table = np.full((len(lengths), columns), -1, np.int32)
    for row, n in enumerate(lengths):
        count = -(-n // page)
        first = 0
        if sharing and row and rng.random() < 0.7:
            other = rng.integers(row)
            first = min(lengths[other] // page, n // page)
            table[row, :first] = table[other, :first]
        table[row, first:count] = [order.pop() for _ in range(first, count)]
    return table


@pytest.mark.parametrize("page,layout,kind,heads,dim", [
    (16, "token", "f32", 2, 64), (1, "token", "bf16", 2, 8), (20, "head", "bf16", 3, 72),
    (7, "head", "f16", 1, 2), (33, "token", "f16", 5, 24),
])
@pytest.mark.parametrize("room", [0, 1, 40])
def test_fork(ops, torch, page, layout, kind, heads, dim, room):
    rng = np.random.default_rng(page + room)
    for trial in range(4):
        count, columns = int(rng.integers(1, 40)), 12
        lengths = rng.integers(0, (columns - 1) * page + 1, count).astype(np.int32)
        lengths[rng.random(count) < 0.3] //= page  # whole pages, and none
        lengths[rng.random(count) < 0.3] *= 1
        pages = int(sum(-(-lengths // page))) + [0, 3, 50, 400][trial]
        pages = max(pages, 1)
        table = random_table(rng, lengths, page, pages, columns, True)
        rows_out = [count, 1, 2 * count, count + 3][trial]
        parents = rng.integers(-1, count, rows_out).astype(np.int32)
        if trial == 3:
            parents[0] = count + 5
        held = (rng.random(pages) < 0.1).astype(np.uint8) if trial >= 2 else None
        keys, values = page_pool(torch, kind, 2, pages, page, heads, dim, layout)
        before = [p.float().cpu().numpy() for p in (keys, values)]
        to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        got, got_lengths, status = ops.fork_pages(
            keys, values, to(table), to(lengths), to(parents), room=room,
            held=None if held is None else to(held))
        for pool, was in zip((keys, values), before):
            want, want_table, want_lengths, want_status = fork_expected(
                was, table, lengths, parents, room, held)
            assert np.array_equal(pool.float().cpu().numpy(), want)
        assert np.array_equal(got.cpu().numpy(), want_table)
        assert np.array_equal(got_lengths.cpu().numpy(), want_lengths)
        assert np.array_equal(status.cpu().numpy(), want_status)


def test_fork_shared_unfinished_pages(ops, torch):
    """A last page that another row holds whole, or that is held outside, is
    copied by everyone who goes on in it."""
    page, columns = 8, 4
    table = np.array([[5, 1, -1, -1], [5, 1, 2, -1], [3, -1, -1, -1]], np.int32)
    lengths = np.array([12, 20, 5], np.int32)  # row 0 ends in page 1, row 1 holds it whole
    parents = np.array([0, 0, 1, 2, 2], np.int32)
    held = np.zeros(12, np.uint8)
    held[3] = 1
    keys, values = page_pool(torch, "f32", 3, 12, page, 2, 4)
    before = keys.cpu().numpy()
    to = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got, _, status = ops.fork_pages(keys, values, to(table), to(lengths), to(parents), room=1,
                                    held=to(held))
    want, want_table, _, want_status = fork_expected(before, table, lengths, parents, 1, held)
    assert np.array_equal(got.cpu().numpy(), want_table)
    assert np.array_equal(keys.cpu().numpy(), want)
    assert np.array_equal(status.cpu().numpy(), want_status)
    ends = [want_table[0, 1], want_table[1, 1], want_table[3, 0], want_table[4, 0]]
    assert len(set(ends)) == 4 and not {1, 3} & set(ends) and columns == 4


def test_fork_many_rows_and_pages(ops, torch):
    """More rows, columns and pages than the plan has threads and warps."""
    rng = np.random.default_rng(3)
    page, columns, count = 4, 70, 5000
    lengths = rng.integers(0, columns * page - 1, count).astype(np.int32)
    pages = int(sum(-(-lengths // page))) + 9000
    table = random_table(rng, lengths, page, pages, columns, False)
    parents = rng.integers(-1, count, count).astype(np.int32)
    keys, values = page_pool(torch, "f16", 1, pages, page, 1, 2)
    before = values.float().cpu().numpy()
    to = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got, got_lengths, status = ops.fork_pages(keys, values, to(table), to(lengths), to(parents))
    want, want_table, want_lengths, want_status = fork_expected(before, table, lengths, parents, 1)
    assert np.array_equal(got.cpu().numpy(), want_table)
    assert np.array_equal(got_lengths.cpu().numpy(), want_lengths)
    assert np.array_equal(status.cpu().numpy(), want_status)
    assert np.array_equal(values.float().cpu().numpy(), want)


def test_fork_frees_everything(ops, torch):
    keys, values = page_pool(torch, "f32", 1, 9, 4, 1, 4)
    table = torch.tensor([[3, 4], [7, -1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([8, 2], dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    got, _, status = ops.fork_pages(keys, values, table, lengths, none)
    assert got.shape == (0, 2) and status.tolist() == [0, 9]
    gone = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    got, n, status = ops.fork_pages(keys, values, table, lengths, gone)
    assert (got == -1).all() and n.tolist() == [0, 0] and status.tolist() == [0, 9]


@pytest.mark.parametrize("page,layout,kind,heads,dim", [
    (16, "token", "f32", 2, 64), (1, "token", "bf16", 2, 8), (20, "head", "bf16", 3, 72),
    (5, "token", "f16", 1, 2),
])
def test_compact(ops, torch, page, layout, kind, heads, dim):
    rng = np.random.default_rng(page)
    for trial in range(5):
        count, columns = int(rng.integers(1, 60)), 9
        lengths = rng.integers(0, columns * page + 1, count).astype(np.int32)
        used = int(sum(-(-lengths // page)))
        pages = max(1, used + [0, 1, 30, 500, 6000][trial])
        table = random_table(rng, lengths, page, pages, columns, True)
        held = (rng.random(pages) < 0.2).astype(np.uint8) if trial % 2 else None
        keys, values = page_pool(torch, kind, 2, pages, page, heads, dim, layout)
        before = keys.float().cpu().numpy()
        live = np.zeros(pages, bool)
        live[table[table >= 0]] = True
        kept = held.astype(bool) if held is not None else np.zeros(pages, bool)
        live &= ~kept
        total = int((live | kept).sum())
        sources = [x for x in np.nonzero(live)[0] if x >= total]
        targets = [x for x in range(total) if not live[x] and not kept[x]][:len(sources)]
        want = before.copy()
        want[:, targets] = before[:, sources]
        place = np.arange(pages)
        place[sources] = targets
        want_table = np.where(table >= 0, place[table.clip(0)], -1)
        device_table = torch.from_numpy(table).cuda()
        in_place = trial == 4
        got, status = ops.compact_pages(keys, values, device_table,
                                        held=None if held is None else torch.from_numpy(held).cuda(),
                                        table_out=device_table if in_place else None)
        assert (got is device_table) == in_place
        assert np.array_equal(got.cpu().numpy(), want_table)
        assert status.tolist() == [total, len(sources)]
        assert np.array_equal(keys.float().cpu().numpy(), want)


def test_compact_many_rows_and_pages(ops, torch):
    """More rows and pages than one block plans for; some pages held."""
    rng = np.random.default_rng(4)
    page, columns, count = 2, 60, 900
    lengths = rng.integers(0, columns * page + 1, count).astype(np.int32)
    used = int(sum(-(-lengths // page)))
    for pages in (used + 25000, used):
        table = random_table(rng, lengths, page, pages, columns, False)
        held = (rng.random(pages) < 0.05).astype(np.uint8)
        keys, values = page_pool(torch, "f16", 1, pages, page, 1, 2)
        before = values.float().cpu().numpy()
        live = np.zeros(pages, bool)
        live[table[table >= 0]] = True
        kept = held.astype(bool)
        live &= ~kept
        total = int((live | kept).sum())
        sources = np.nonzero(live)[0]
        sources = sources[sources >= total]
        targets = np.nonzero(~live & ~kept)[0][:len(sources)]
        want = before.copy()
        want[:, targets] = before[:, sources]
        place = np.arange(pages)
        place[sources] = targets
        got, status = ops.compact_pages(keys, values, torch.from_numpy(table).cuda(),
                                        held=torch.from_numpy(held).cuda())
        assert np.array_equal(got.cpu().numpy(), np.where(table >= 0, place[table.clip(0)], -1))
        assert status.tolist() == [total, len(sources)]
        assert np.array_equal(values.float().cpu().numpy(), want)


def test_copy_pages(ops, torch):
    for kind, dim, layout in (("bf16", 8, "token"), ("f16", 2, "head"), ("f32", 3, "token")):
        keys, values = page_pool(torch, kind, 3, 20, 5, 2, dim, layout)
        before = [p.clone() for p in (keys, values)]
        sources = torch.tensor([3, 3, -1, 7, 25], dtype=torch.int32, device="cuda")
        targets = torch.tensor([10, 19, 11, 20, 12], dtype=torch.int32, device="cuda")
        ops.copy_pages(keys, values, sources, targets)
        for pool, was in zip((keys, values), before):
            want = was.clone()
            want[:, 10] = want[:, 19] = was[:, 3]
            assert torch.equal(pool, want)
        ops.copy_pages(keys, values, sources[:0], targets[:0])


def test_pages_refuse(ops, torch):
    keys, values = page_pool(torch, "f32", 2, 6, 4, 2, 8)
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call, text in [
        (lambda: ops.fork_pages(keys, values[:1], table, lengths, lengths), "differ"),
        (lambda: ops.fork_pages(keys[..., :4], values[..., :4], table, lengths, lengths),
         "contiguous"),
        (lambda: ops.fork_pages(keys, values, table, lengths, lengths, room=-1), "room"),
        (lambda: ops.fork_pages(keys, values, table, lengths[:1], lengths), "lengths has"),
        (lambda: ops.fork_pages(keys, values, table, lengths, lengths,
                                held=torch.zeros(5, dtype=torch.uint8, device="cuda")), "held"),
        (lambda: ops.compact_pages(keys, values, table, table_out=table[:1]), "table_out"),
        (lambda: ops.copy_pages(keys, values, lengths, lengths[:1]), "targets"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(N.LrrtError, match="must not be the table"):
        ops.fork_pages(keys, values, table, lengths, lengths, table_out=table)
    odd = [p[..., :1] for p in page_pool(torch, "f16", 1, 6, 1, 1, 2)]
    with pytest.raises((N.LrrtError, ValueError)):
        ops.copy_pages(*odd, lengths, lengths)


# --- beam selection ---------------------------------------------------------------

def beam_expected(logits, scores, count, finished, end_token):
    """Candidates one after another in 64 bits; the cases keep scores that are
    not equal at least 1e-3 apart. (scores, parents, tokens, finished)"""
    groups, beams, vocab = logits.shape
    outs = []
    for g in range(groups):
        found = []
        for k in range(beams):
            if finished is not None and finished[g, k]:
                found.append((-float(scores[g, k]), k, 0.0, end_token))
                continue
            x = logits[g, k].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            top = x.max()
            if not np.isfinite(top):
                continue
            lse = top + np.log(np.exp(x - top).sum())
            order = np.argsort(-x, kind="stable")[:count]
            found += [(-(float(scores[g, k]) + x[t] - lse), k, -x[t], int(t)) for t in order
                      if np.isfinite(x[t])]
        # Equal scores: exactly equal logits of a beam, or nothing else by design.
        found = sorted((c for c in found if c[0] < np.inf), key=lambda c: (round(c[0], 6), *c[1:]))
        found = found[:count]
        row = [(-c[0], g * beams + c[1], c[3],
                int(c[3] == end_token or bool(finished is not None and finished[g, c[1]])))
               for c in found]
        row += [(-np.inf, -1, -1, 1)] * (count - len(row))
        outs.append(row)
    return [np.array([[r[i] for r in row] for row in outs]) for i in range(4)]


def beam_case(rng, groups, beams, vocab, ended=0.2):
    """Logits on a grid of 1/16; scores that set the beams 1/16/beams apart."""
    logits = np.round(rng.normal(0, 3, (groups, beams, vocab)) * 16) / 16
    logits = logits.clip(-15, 15)
    finished = (rng.random((groups, beams)) < ended).astype(np.uint8)
    lse = np.log(np.exp(logits).sum(-1))
    lse = np.where(finished, np.round(lse * 16) / 16, lse)
    shift = np.argsort(rng.random((groups, beams)), -1)
    scores = (lse - 20 + (2 * shift + 1) / (32 * beams)).astype(np.float32)
    return logits, scores, finished


def beam_check(ops, torch, kind, logits, scores, count, finished=None, end_token=-1, device=None):
    if device is None:
        device = torch.from_numpy(logits).to(dtype_of(torch, kind)).cuda()
    got = ops.beam_select(device, torch.from_numpy(scores).cuda(), count,
                          finished=None if finished is None else torch.from_numpy(finished).cuda(),
                          end_token=end_token)
    want = beam_expected(device.double().cpu().numpy(), scores, count, finished, end_token)
    # A log-sum in 32 bits (relative 2^-18 of a sum of positive numbers, so
    # that absolutely), and the roundings of two sums of numbers below 64.
    close(got[0], torch.from_numpy(want[0]), torch.tensor(2.0 ** -18 + 4 * 64 * FLOAT), "scores")
    for g, w, name in zip(got[1:], want[1:], ("parents", "tokens", "finished")):
        assert np.array_equal(g.cpu().numpy(), w), name
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 4, 1000, 4), (3, 2, 4095, 7), (1, 8, 4097, 16),
    (5, 3, 8193, 6), (1, 32, 2000, 64), (2, 64, 333, 32), (1, 4, 151936, 4), (1, 1, 70000, 64),
    (9, 5, 64, 1),
])
def test_beam_select(ops, torch, kind, groups, beams, vocab, count):
    rng = np.random.default_rng(vocab + count)
    logits, scores, finished = beam_case(rng, groups, beams, vocab)
    beam_check(ops, torch, kind, logits, scores, count)
    beam_check(ops, torch, kind, logits, scores, count, finished, end_token=0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_beam_select_equal_logits(ops, torch, kind):
    """All equal, two values, sorted either way: ties go to the lower token, and
    orders that defeat the pre-selection are still right."""
    vocab, scores = 9000, np.array([[0.0, -0.01]], np.float32)
    index = np.arange(vocab)
    for row in (index * 0.0, (index % 2) * 1.0, index // 64 / 16.0, -(index // 64) / 16.0,
                (index >= vocab - 3) * 2.0, (index % 2000 == 5) * -1.0,
                # One group of threads holds the small ones of each round.
                np.where(index % 1024 < 128, 0.0, 8 + (index * 7919 % 97) / 16.0)):
        logits = np.broadcast_to(row, (1, 2, vocab)).copy()
        for count in (1, 2, 16, 64):
            beam_check(ops, torch, kind, logits, scores, count)


def test_beam_select_infinities(ops, torch):
    """Banned tokens, dead beams, NaN, and too few candidates."""
    rng = np.random.default_rng(5)
    logits, scores, _ = beam_case(rng, 4, 3, 500)
    logits[0, 0, 3:] = -np.inf          # three tokens left
    logits[0, 1] = -np.inf              # none
    logits[0, 2, 1:] = np.nan           # one
    logits[1, 0, 7] = np.nan
    scores[1, 1] = -np.inf              # a beam that has not begun
    scores[2] = -np.inf
    got = beam_check(ops, torch, "f32", logits, scores, 8)
    assert got[2][0, 4:].tolist() == [-1] * 4 and got[0][2].tolist() == [-math.inf] * 8
    finished = np.zeros((4, 3), np.uint8)
    finished[3] = 1                     # all have ended
    beam_check(ops, torch, "f32", logits, scores, 8, finished, end_token=4)


def test_beam_select_strides(ops, torch):
    """Rows that begin off 16 bytes, and rows with space between them."""
    rng = np.random.default_rng(6)
    logits, scores, _ = beam_case(rng, 2, 2, 3001)
    for kind in ("f32", "bf16"):
        wide = torch.full((2, 2, 3333), 9.0, dtype=dtype_of(torch, kind), device="cuda")
        view = wide[:, :, 1:3002]
        view.copy_(torch.from_numpy(logits))
        beam_check(ops, torch, kind, None, scores, 5, device=view)


def test_beam_select_repeats(ops, torch):
    rng = np.random.default_rng(8)
    logits, scores, finished = beam_case(rng, 16, 4, 20000)
    device = torch.from_numpy(logits).bfloat16().cuda()
    s, f = torch.from_numpy(scores).cuda(), torch.from_numpy(finished).cuda()
    first = ops.beam_select(device, s, 8, finished=f, end_token=2)
    for _ in range(20):
        again = ops.beam_select(device, s, 8, finished=f, end_token=2)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_beam_select_no_groups_and_refusals(ops, torch):
    x = torch.zeros(2, 3, 50, device="cuda")
    s = torch.zeros(2, 3, device="cuda")
    assert ops.beam_select(x[:0], s[:0], 3)[0].shape == (0, 3)
    for call, text in [
        (lambda: ops.beam_select(x.double(), s, 3), "logits of"),
        (lambda: ops.beam_select(x, s[:1], 3), "scores must"),
        (lambda: ops.beam_select(x, s, 3, finished=torch.zeros(2, 3, device="cuda")), "finished"),
        (lambda: ops.beam_select(x[..., ::2], s, 3), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    for call, text in [
        (lambda: ops.beam_select(x, s, 0), "1 to 64"), (lambda: ops.beam_select(x, s, 65), "1 to 64"),
        (lambda: ops.beam_select(x[..., :2], s, 3), "vocab"),
    ]:
        with pytest.raises(N.LrrtError, match=text):
            call()


# --- streams ------------------------------------------------------------------------

def test_another_stream(gpu, torch, ops):
    """Operators made on a side stream run there, and refuse any other."""
    from lrrt_b200 import ops as module
    case = Attention(torch, "bf16", [500, 20], 8, 2, 64, 16, seed=21)
    want, _ = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        with module.Ops(0) as mine:
            q = case.q * 1  # on the side stream, without a wait of the host's
            got, _ = mine.paged_attention(q, case.keys, case.values, case.table, case.n)
            assert torch.equal(got, want)
            with pytest.raises(ValueError, match="stream"):
                ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    with pytest.raises(ValueError, match="closed"):
        mine.beam_select(torch.zeros(1, 1, 4, device="cuda"), torch.zeros(1, 1, device="cuda"), 1)


def test_captured_step(gpu, torch):
    """A step of beam search as a CUDA graph, replayed with other inputs."""
    from lrrt_b200 import ops as module
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), module.Ops(0) as mine:
        mine.reserve(16 << 20)
        case = Attention(torch, "f16", [40, 90], 4, 2, 64, 16, seed=23)
        logits = torch.randn(1, 2, 5000, device="cuda")
        scores = torch.zeros(1, 2, device="cuda")

        def step():
            out, _ = mine.paged_attention(case.q, case.keys, case.values, case.table, case.n)
            chosen = mine.beam_select(logits, scores, 2)
            forked = mine.fork_pages(case.keys[None], case.values[None], case.table, case.n,
                                     chosen[1].flatten(), room=0)
            return (out, *chosen, *forked)

        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
        for seed in range(3):
            torch.manual_seed(seed)
            logits.copy_(torch.randn(1, 2, 5000, device="cuda"))
            case.q.copy_(torch.randn_like(case.q))
            before = [case.keys.clone(), case.values.clone()]  # a fork reuses freed pages
            graph.replay()
            got = [t.clone() for t in captured] + [case.keys.clone(), case.values.clone()]
            case.keys.copy_(before[0])
            case.values.copy_(before[1])
            want = [*step(), case.keys, case.values]
            got[-2:], want[-2:] = ([t.nan_to_num() for t in x[-2:]] for x in (got, want))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        side.synchronize()
        del graph
