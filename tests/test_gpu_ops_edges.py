"""The paged-cache operators where numbers are at the ends of their ranges.
Bounds are derived as in test_gpu_ops.py."""
import math

import pytest

from test_gpu_ops import FLOAT, LEAST, ROUND, Attention, close, ops, torch  # noqa: F401

pytestmark = pytest.mark.gpu


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
