"""The paged-cache operators where numbers are at the ends of their ranges.
Bounds are derived as in test_gpu_ops.py."""
import math

import numpy as np
import pytest

from test_gpu_ops import (FLOAT, LEAST, ROUND, Attention, beam_case, beam_check, close,  # noqa: F401
                          dtype_of, ops, torch)

pytestmark = pytest.mark.gpu


def same(actual, want, bound, what=""):
    """close(), and NaN in the same places."""
    actual, want = actual.double().cpu(), want.double().cpu()
    assert (actual.isnan() == want.isnan()).all(), f"{what}: NaN elsewhere"
    clean = lambda x: x.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf)  # noqa: E731
    close(clean(actual), clean(want), bound.nan_to_num(0.0, 0.0, 0.0), what)


# --- weights far below the largest ------------------------------------------------

def dominated(torch, kind, n, gap, first, equal, dim=64):
    """One key whose score is `gap` above the rest, with the value `first`, and
    n more keys; scores are exact in every type: q is (1, 0, ...), keys are
    (score, 0, ...), the rest's scores below 1."""
    case = Attention(torch, kind, [n + 1], 8, 1, dim, 64, seed=31)
    case.q.zero_()
    case.q[..., 0] = 1
    j = torch.arange(n + 1, device="cuda")
    place = (case.table[0, j // 64].long(), j % 64)
    score = torch.zeros(n + 1, device="cuda") if equal else (j * 7 % 16) / 16.0
    score[0] = gap + 1
    keys = torch.zeros(n + 1, 1, dim, device="cuda")
    keys[:, 0, 0] = score
    case.keys[place] = keys.to(case.keys.dtype)
    values = torch.rand(n + 1, 1, dim, device="cuda") + 0.5
    if equal:
        values[1:] = values[1:2]
    values[0] = first
    case.values[place] = values.to(case.values.dtype)
    return case, score.double(), case.values[place][:, 0].double()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("first", [0.0, 1.0])
@pytest.mark.parametrize("n,gap,equal", [
    (40, 6, False), (3500, 13.875, True), (8191, 17, True), (30000, 16, False), (30000, 9, True),
    (131071, 17, False), (2000, 25, True),
])
def test_attention_below_a_dominating_key(ops, torch, kind, first, n, gap, equal):
    """A key that has nearly all the weight and a value of 0 or 1: the rest is
    small, and with a value of 0 it is all that there is to see.

    Scores are exact; a weight's error is below 2^-18 (the exponential 2^-22, its
    argument up to 26 times log2 e, rounded twice and with a rounded constant:
    2.5 * 2^-24 * 26), that of its two pieces 2^-16 in bf16 (the first cut off
    after 8 bits, the rest rounded to 8) and 2^-20 in f16 and f32, whose values
    are split too; f16 pieces end at 2^-39 of the largest weight, and two of
    them may be amiss. A sum of positive terms in 32 bits whose roundings all go
    one way is off by 2^-23 of it for each addition: two for each tile of 16
    keys in a unit's share of the row (of at least 592 units), and the joins'
    (148 blocks' parts, eight of a block). The log-sum is off by the share of
    the weights below the first that is, and by its sum's roundings."""
    case, x, v = dominated(torch, kind, n, gap, first, equal)
    p = torch.exp(x - x.max())
    total = p.sum()
    want = (p[:, None] * v).sum(0) / total
    pieces = {"f32": 2.0 ** -20, "bf16": 2.0 ** -16, "f16": 2.0 ** -20}[kind]
    tiles = n // 16 // 592 + 2
    relative = 2 * (2.0 ** -18 + pieces) + 2 * (2 * tiles + 156) * 2.0 ** -23
    lost = n * 2.0 ** -38 * v.abs().max() / total if kind == "f16" else 0.0
    bound = relative * want.abs() + lost + 1.01 * ROUND[kind] * want.abs() + LEAST[kind]
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n, scale=1.0)
    close(out[0], want.expand(8, -1), bound.expand(8, -1), "out")
    want_lse = torch.logsumexp(x, 0).expand(1, 8)
    sums = (2.0 ** -18 * (1 - 1 / total) + (2 * tiles + 156) * FLOAT).cpu()
    close(lse, want_lse, sums + 4 * FLOAT * want_lse.abs().cpu(), "lse")


# --- infinities and NaN -----------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths", [[5, 40], [700, 3], [20000, 16]])
def test_attention_nan_rows(ops, torch, kind, lengths):
    """A NaN in a query: outputs and log-sums of its head are NaN, and no others."""
    case = Attention(torch, kind, lengths, 8, 2, 64, 16, seed=33)
    case.q[0, 2, 5] = math.nan
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    nan = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    nan[0, 2] = True
    assert torch.equal(lse.isnan(), nan)
    assert torch.equal(out.isnan().all(-1), nan) and torch.equal(out.isnan().any(-1), nan)
    assert lse[~nan].isfinite().all()


@pytest.mark.parametrize("kind,dim,heads,kv_heads", [
    ("f32", 64, 14, 2), ("f32", 128, 24, 2), ("f32", 128, 8, 2), ("f32", 96, 3, 3),
    ("bf16", 128, 32, 8), ("bf16", 64, 24, 2), ("bf16", 256, 20, 1), ("f16", 128, 16, 2),
    ("f16", 256, 17, 1), ("f16", 80, 4, 4),
])
@pytest.mark.parametrize("lengths", [[1, 37], [300, 1000], [20000, 0]])
def test_attention_infinite_values(ops, torch, kind, dim, heads, kv_heads, lengths):
    """An infinite value makes its column infinite, of both signs NaN, a NaN
    NaN; every other column is as it would be."""
    case = Attention(torch, kind, lengths, heads, kv_heads, dim, 16, seed=35)
    bound = case.expected()[2]  # with the finite values: the largest one is the same

    def put(row, j, head, column, value):
        case.values[int(case.table[row, j // 16]), j % 16, head, column] = value

    for row, n in enumerate(lengths):
        if n:
            put(row, n // 2, 0, 1, math.inf)
            put(row, n - 1, 0, 2, -math.inf)
            put(row, 0, kv_heads - 1, 5, math.inf)
            put(row, n // 3, kv_heads - 1, 7, math.nan)
        if n > 30:
            put(row, n - 9, 0, 3, math.inf)
            put(row, 4, 0, 3, -math.inf)
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    want, want_lse, _, lse_bound = case.expected()
    same(out, want, bound, "out")
    same(lse, want_lse, lse_bound, "lse")
    if lengths[0] > 30:
        assert (out[0, :heads // kv_heads, 1] == math.inf).all()
        assert (out[0, :heads // kv_heads, 2] == -math.inf).all()
        assert out[0, :heads // kv_heads, 3].isnan().all()


@pytest.mark.parametrize("kind,dim,heads,kv_heads", [
    ("f32", 64, 14, 2), ("f32", 128, 24, 2), ("f32", 128, 8, 2), ("f32", 96, 3, 3),
    ("bf16", 128, 8, 2), ("bf16", 256, 20, 1), ("f16", 64, 24, 2),
])
@pytest.mark.parametrize("lengths", [[3, 37], [300, 1000], [20000, 50]])
def test_attention_infinite_keys(ops, torch, kind, dim, heads, kv_heads, lengths):
    """A key whose score is -infinity weighs nothing, one of infinity leaves NaN."""
    case = Attention(torch, kind, lengths, heads, kv_heads, dim, 16, seed=37)
    case.q[:, :, 3] = case.q[:, :, 3].abs() + 0.5
    _, _, bound, lse_bound = case.expected()  # an infinity has no error of its own

    def put(row, j, heads, value):
        case.keys[int(case.table[row, j // 16]), j % 16, heads, 3] = value

    for j in {0, lengths[0] // 2}:
        put(0, j, slice(None), -math.inf)
    put(1, lengths[1] - 1, 0, math.inf)
    want, want_lse, _, _ = case.expected()
    group = heads // kv_heads
    assert want[0].isfinite().all() and want[1, :group].isnan().all()
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    same(out, want, bound + 1.01 * ROUND[kind] * want.abs(), "out")
    want_lse[1, :group] = math.nan  # infinity - infinity, as the weights are
    same(lse, want_lse, lse_bound + 4 * FLOAT * want_lse.abs(), "lse")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_attention_nothing_weighs(ops, torch, kind):
    """Every score is -infinity: as a row that sees no token."""
    case = Attention(torch, kind, [1, 20, 5000], 8, 2, 64, 16, seed=39)
    case.q[:, :, 0] = 1
    case.keys[..., 0] = -math.inf
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_attention_largest_numbers(ops, torch):
    """Keys and values next to the largest of 32 bits: what rounds to an infinity
    on its way is still the number that it is."""
    most = torch.finfo(torch.float32).max
    lengths = [1, 33, 900]
    case = Attention(torch, "f32", lengths, 8, 2, 64, 16, seed=41)
    case.keys[..., 2] = most
    case.q[..., 2] = 2.0 ** -122
    want, want_lse, bound, lse_bound = case.expected()
    case.values[..., 1] = most
    out, lse = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    others = [i for i in range(64) if i != 1]
    close(out[..., others], want[..., others], bound[..., others], "out")
    close(lse, want_lse, lse_bound, "lse")
    # One key: its value, split in two (2^-20). More of them may leave 32 bits.
    assert ((out[0, :, 1].double() / most - 1).abs() <= 2.0 ** -19).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 16)])
def test_attention_long_sums(ops, torch, kind, dim, heads):
    """Rows of 100000 keys, so many that a warp has nearly all of one, with the
    same value at each key: the output is that value. Rounded to nearest, the
    tiles' sums are off by a random walk of 6250 roundings of 2^-24 (3e-6), less
    than half a unit in the last place of 16 bits; rounded one way, by 4e-4."""
    g = torch.Generator(device="cuda")
    g.manual_seed(43)
    n, batch, page = 100000, 1200, 64
    pages = -(-n // page)
    dtype = dtype_of(torch, kind)
    keys = (torch.randn(pages, page, 1, dim, generator=g, device="cuda") * 0.3).to(dtype)
    value = (1 + torch.arange(dim, device="cuda") / 128).to(dtype)
    values = value.expand(pages, page, 1, dim).contiguous()
    q = torch.randn(batch, heads, dim, generator=g, device="cuda").to(dtype)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, -1)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out, _ = ops.paged_attention(q, keys, values, table, lengths)
    if kind == "f32":
        close(out, value.expand_as(out), 2.0 ** -16 * value.expand_as(out), "out")
    else:
        assert torch.equal(out, value.expand_as(out))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("softcap", [0.5, 50.0, 1.0e3, 1.0e4, 1.0e6])
@pytest.mark.parametrize("spread", [0.01, 1.0, 12.0])
def test_attention_caps(ops, torch, kind, softcap, spread):
    """Caps below the scores and far above them. A capped score has the relative
    error of two products and of tanhf, below 2^-21,
    which the bound of every score (2^-19 of its products' sizes) holds."""
    case = Attention(torch, kind, [1, 40, 700, 2500], 16, 2, 96, 16, seed=45, spread=spread)
    case.check(ops, softcap=softcap)


# --- rows of masked logits --------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["lowest", -1.0e10, -1.0e30, 1.0e10, "largest", -60000.0])
@pytest.mark.parametrize("vocab", [70, 5000, 151936])
def test_beam_select_masked_rows(ops, torch, kind, mask, vocab):
    """A row of one value throughout, as masks of a type's lowest value leave it, is
    uniform: its best are the lowest tokens, at -log vocab. Beside it a row where
    the mask leaves three tokens, and one that it leaves as it is.

    Scores are off by the roundings of 32 bits and by the sum's (2^-18, as in
    test_gpu_ops.py); a beam's logits are exact in each type."""
    dtype = dtype_of(torch, kind)
    info = torch.finfo(dtype)
    value = {"lowest": info.min, "largest": info.max}.get(mask, mask)
    value = min(max(value, info.min), info.max)
    g = torch.Generator(device="cuda")
    g.manual_seed(47)
    rows = torch.randn(3, vocab, generator=g, device="cuda").mul_(48).round_().div_(16)
    rows[0] = value
    if value < 0:
        rows[1, 3:] = value
    logits = rows.to(dtype)
    assert (logits[0] == logits[0, 0]).all() and logits.isfinite().all()
    scores = torch.tensor([-3.0, -30.0, -60.0], device="cuda")
    got = ops.beam_select(logits[None], scores[None], 16)
    x = logits.double()
    above = x - x.amax(-1, keepdim=True)
    score = scores.double()[:, None] + above - above.exp().sum(-1, keepdim=True).log()
    order = score.flatten().sort(descending=True, stable=True)
    close(got[0][0], order.values[:16], torch.tensor(2.0 ** -18 + 4 * 64 * FLOAT), "scores")
    alone = ops.beam_select(logits[None, :1], scores[None, :1], 16)
    assert alone[2].tolist() == [list(range(16))] and alone[1].tolist() == [[0] * 16]
    close(alone[0][0], torch.full((16,), -3.0 - math.log(vocab)),
          torch.tensor(2.0 ** -18 + 4 * 64 * FLOAT), "scores")


# --- every number of candidates ---------------------------------------------------

@pytest.mark.parametrize("beams", [1, 2, 3, 5, 7, 8, 13, 16])
def test_beam_select_any_number_of_candidates(ops, torch, beams):
    """Few candidates are ranked by one, two or four threads each, whatever remains
    of the last warp: all numbers of them up to 17 beams' worth."""
    rng = np.random.default_rng(beams)
    for count in range(1, 18):
        logits, scores, finished = beam_case(rng, 3, beams, 200)
        beam_check(ops, torch, "f32", logits, scores, count, finished, end_token=1)
        beam_check(ops, torch, "bf16", logits, scores, count)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("below", [0, 1, 2 ** 10, 2 ** 12, 2 ** 13 - 1])
def test_attention_largest_values(ops, torch, sign, below):
    """The value of a single key at either end of 32 bits, some units in the last
    place inside it, is the output, to 2^-20 of it."""
    most = torch.finfo(torch.float32).max
    case = Attention(torch, "f32", [1, 1], 8, 2, 128, 16, seed=49)
    value = torch.tensor(most).view(torch.int32).sub(below).view(torch.float32).item() * sign
    case.values[..., 7] = value
    out, _ = ops.paged_attention(case.q, case.keys, case.values, case.table, case.n)
    assert ((out[:, :, 7].double() / value - 1).abs() <= 2.0 ** -20).all()
