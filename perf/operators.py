"""Cases of the paged-cache operators: what one step of serving many sequences
from a paged key-value cache runs besides its matrix products.

  rope    rotary positions of a step's queries and keys, appended to the pages
  attn    attention of one new token per sequence over the paged cache
  fork    sequences reordered, shared and split copy-on-write (a beam step)
  compact live pages moved to the front of the pool, tables rewritten
  beam    the best continuations over the beams and the vocabulary

``run`` computes an operator in its plain form with elementary torch
operations in 32 bits, or, where ``own`` is true, through lrrt_b200.ops.
Lengths, parents and positions follow from the case alone, so that ``work`` can
count them; values, page numbers and flags follow from the seed.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # One stream early in its answer: this framework's decode shape (14
        # query heads over 2, 64 wide, 32 bits). Latency is all there is.
        dict(name="attn one stream", op="attn", type="f32", batch=1, heads=14, kv_heads=2, dim=64,
             page=16, longest=160, spread="near", cap=0.0, bias=False, window=0, layout="token"),
        # The batched decode of this framework's benchmark: 32 streams around
        # a context of 1024.
        dict(name="attn 32 streams", op="attn", type="f32", batch=32, heads=14, kv_heads=2, dim=64,
             page=16, longest=1152, spread="near", cap=0.0, bias=False, window=0, layout="token"),
        # A busy server: 64 conversations of very different lengths, some just
        # begun, a 16-bit cache with grouped heads.
        dict(name="attn ragged server", op="attn", type="bf16", batch=64, heads=32, kv_heads=8,
             dim=128, page=64, longest=8192, spread="ragged", cap=0.0, bias=False, window=0,
             layout="token"),
        # Two very long documents, capped scores with a distance bias, pages
        # stored head by head; few rows, so the work is in the length.
        dict(name="attn long capped", op="attn", type="f16", batch=2, heads=16, kv_heads=2, dim=128,
             page=128, longest=131071, spread="near", cap=30.0, bias=True, window=0, layout="head"),
        # One decode step of 32 streams at this framework's shape.
        dict(name="rope step", op="rope", type="f32", tokens=32, batch=32, heads=14, kv_heads=2,
             dim=64, rotary=64, page=16, longest=1152, pairs="half", scaled=False),
        # Five prompts of a middling size in one pass, interleaved pairs on
        # part of the head.
        dict(name="rope prompts", op="rope", type="f16", tokens=2047, batch=5, heads=16, kv_heads=16,
             dim=96, rotary=48, page=24, longest=1000, pairs="interleaved", scaled=False),
        # A long prompt's chunk far into its document, with the frequencies
        # scaled for long contexts.
        dict(name="rope long chunk", op="rope", type="bf16", tokens=16384, batch=3, heads=32,
             kv_heads=8, dim=128, rotary=128, page=64, longest=40000, pairs="half", scaled=True),
        # A beam step over this framework's cache: 8 prompts with 4 beams, 24
        # layers of 2 heads, 64 wide, 32 bits.
        dict(name="fork 32 beams", op="fork", type="f32", prompts=8, beams=4, layers=24, kv_heads=2,
             dim=64, page=16, longest=300, room=1),
        # A beam step of a server: 16 prompts with 8 beams over a 16-bit cache.
        dict(name="fork 128 beams", op="fork", type="bf16", prompts=16, beams=8, layers=16,
             kv_heads=8, dim=128, page=32, longest=500, room=1),
        # A pool that finished sequences left full of holes.
        dict(name="compact", op="compact", type="bf16", batch=48, layers=16, kv_heads=4, dim=128,
             page=32, longest=700, holes=0.5),
        # One prompt with 4 beams over this framework's vocabulary.
        dict(name="beam 1 x 4", op="beam", type="f32", batch=1, beams=4, vocab=151936, count=4),
        # 32 prompts with 8 beams, twice as many candidates as beams.
        dict(name="beam 32 x 8", op="beam", type="bf16", batch=32, beams=8, vocab=151936, count=16),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rope", "fork", "compact", "beam"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "attn":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
        dim = rng.choice([64, 96, 128] if kind == "f32" else [64, 80, 128, 256])
        longest = _log(rng, 2, 100000)
        row = kv_heads * dim * 2 * SIZES[kind]
        batch = max(1, min(_log(rng, 1, 128), int(500e6 // (row * longest))))
        longest = min(longest, int(500e6 // (row * batch)))
        return dict(op=op, type=kind, batch=batch, heads=kv_heads * group, kv_heads=kv_heads,
                    dim=dim, page=rng.choice([1, 8, 16, 20, 32, 64, 128]) if longest < 20000
                    else rng.choice([16, 48, 64, 128]), longest=longest,
                    spread=rng.choice(["near", "ragged"]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    bias=rng.random() < 0.3, window=rng.choice([0, 0, 0, _log(rng, 1, longest)]),
                    layout=rng.choice(["token", "head"]))
    if op == "rope":
        kv_heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 128, 256])
        heads = kv_heads * rng.choice([1, 3, 4, 7])
        row = dim * SIZES[kind]
        tokens = min(_log(rng, 1, 16384), int(200e6 // ((heads + 2 * kv_heads) * row)))
        batch = min(tokens, _log(rng, 1, 64))
        return dict(op=op, type=kind, tokens=tokens, batch=batch, heads=heads, kv_heads=kv_heads,
                    dim=dim, rotary=rng.choice([dim, dim // 2]), page=rng.choice([1, 16, 20, 64]),
                    longest=min(_ceil(tokens, batch) + _log(rng, 1, 30000),
                                int(400e6 // (batch * kv_heads * row))),
                    pairs=rng.choice(["half", "interleaved"]), scaled=rng.random() < 0.5)
    if op == "fork":
        return dict(op=op, type=kind, prompts=_log(rng, 1, 16), beams=_log(rng, 1, 8),
                    layers=_log(rng, 1, 12), kv_heads=rng.choice([1, 2, 4, 5]),
                    dim=rng.choice([64, 72, 128]), page=rng.choice([1, 16, 20, 32]),
                    longest=_log(rng, 2, 400), room=rng.choice([0, 1, 1, 9]))
    if op == "compact":
        return dict(op=op, type=kind, batch=_log(rng, 1, 64), layers=_log(rng, 1, 12),
                    kv_heads=rng.choice([1, 2, 4, 5]), dim=rng.choice([64, 72, 128]),
                    page=rng.choice([1, 16, 20, 32]), longest=_log(rng, 2, 500),
                    holes=rng.choice([0.1, 0.5, 0.8]))
    beams = _log(rng, 1, 16)
    return dict(op=op, type=kind, batch=max(1, min(_log(rng, 1, 48), 200 // beams)), beams=beams,
                vocab=_log(rng, 1000, 151936), count=rng.choice([beams, 2 * beams]))


# --- what follows from the case alone ----------------------------------------

def _chance(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case, count):
    """Lengths of `count` sequences: around the longest, or from none to it."""
    r, top = _chance(case), case["longest"]
    if case.get("spread", "ragged") == "near":
        return [top] + [r.randint(max(1, top - max(1, top // 8)), top) for _ in range(count - 1)]
    return [top] + [r.randint(0, top) if r.random() < 0.7 else r.randint(0, max(1, top // 16))
                    for _ in range(count - 1)]


def _tokens(case):
    """(sequence, position) of every token: each sequence gets a run of new
    positions at its end."""
    r = _chance(case)
    n, b = case["tokens"], case["batch"]
    share = [n // b + (i < n % b) for i in range(b)]
    ends = [r.randint(s, max(s, case["longest"])) for s in share]
    sequence = [i for i, s in enumerate(share) for _ in range(s)]
    position = [e - s + j for s, e in zip(share, ends) for j in range(s)]
    return sequence, position, ends


def _parents(case):
    """A beam step's parents: beams of the same prompt, the better ones taken
    more often; a finished prompt's rows are given up."""
    r = _chance(case)
    parents = []
    for p in range(case["prompts"]):
        gone = case["prompts"] > 4 and r.random() < 0.1
        for _ in range(case["beams"]):
            k = min(r.randrange(case["beams"]), r.randrange(case["beams"]))
            parents.append(-1 if gone else p * case["beams"] + k)
    return parents


def _ceil(a, b):
    return -(-a // b)


# --- inputs --------------------------------------------------------------------

def _table(lengths, page, pages, width, g):
    """Page numbers of each sequence in a random order over the pool."""
    need = torch.tensor([_ceil(n, page) for n in lengths])
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width)[None, :]
    first = (torch.cumsum(need, 0) - need)[:, None]
    index = torch.where(column < need[:, None], first + column, -1).cuda()
    return torch.where(index >= 0, order[index.clamp(min=0)], -1).to(torch.int32).contiguous()


def _inverse_frequencies(case):
    """Rotary frequencies; scaled: the long wavelengths divided by 8, the short
    ones kept, a linear blend of the two between (for a model trained at 8192
    positions and used at eight times as many)."""
    f = 1e6 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
    if not case["scaled"]:
        return f
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
    return f * keep + f / 8 * (1 - keep)


def _noise(g, kind, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(TYPES[kind])


def _pool(g, case, pages):
    """All layers' pages, filled layer by layer (some pools are large)."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    pools = []
    for _ in range(2):
        pool = torch.empty((case["layers"],) + shape, dtype=TYPES[case["type"]], device="cuda")
        for layer in range(case["layers"]):
            pool[layer] = _noise(g, case["type"], *shape)
        pools.append(pool)
    return pools


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] == "attn":
        lengths = _lengths(c, c["batch"])
        width = _ceil(c["longest"], c["page"])
        pages = sum(_ceil(n, c["page"]) for n in lengths) + 3
        s["q"] = _noise(g, c["type"], c["batch"], c["heads"], c["dim"])
        # Pages are stored token by token, or head by head and seen through a
        # transposed view.
        shape = [pages, c["page"], c["kv_heads"], c["dim"]]
        if c["layout"] == "head":
            shape[1], shape[2] = shape[2], shape[1]
        s["keys"], s["values"] = (_noise(g, c["type"], *shape) for _ in range(2))
        if c["layout"] == "head":
            s["keys"], s["values"] = s["keys"].transpose(1, 2), s["values"].transpose(1, 2)
        s["table"] = _table(lengths, c["page"], pages, width, g)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["slopes"] = None
        if c["bias"]:
            s["slopes"] = 0.02 * torch.rand(c["heads"], generator=g, device="cuda")
    elif c["op"] == "rope":
        sequence, position, ends = _tokens(c)
        heads, kv = c["heads"], c["kv_heads"]
        pages = sum(_ceil(n, c["page"]) for n in ends) + 3
        # Queries, keys and values lie side by side, as one product wrote them.
        packed = _noise(g, c["type"], c["tokens"], heads + 2 * kv, c["dim"])
        s["q"], s["k"], s["v"] = packed.split([heads, kv, kv], dim=1)
        s["keys"], s["values"] = (torch.zeros(pages, c["page"], kv, c["dim"], device="cuda",
                                              dtype=TYPES[c["type"]]) for _ in range(2))
        s["table"] = _table(ends, c["page"], pages, _ceil(max(ends), c["page"]), g)
        s["sequence"] = torch.tensor(sequence, dtype=torch.int32, device="cuda")
        s["position"] = torch.tensor(position, dtype=torch.int32, device="cuda")
        angle = torch.arange(max(ends), dtype=torch.float64)[:, None] * _inverse_frequencies(c)
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    elif c["op"] in ("fork", "compact"):
        count = c["prompts"] * c["beams"] if c["op"] == "fork" else c["batch"]
        lengths = _lengths(c, count)
        if c["op"] == "fork":  # a prompt's beams have the same length
            lengths = [lengths[i - i % c["beams"]] for i in range(count)]
        used = sum(_ceil(n, c["page"]) for n in lengths)
        spare = count * (1 + _ceil(c["room"], c["page"])) if c["op"] == "fork" else \
            int(used * c["holes"] / (1 - c["holes"])) + 1
        pages = used + spare
        width = _ceil(c["longest"] + c.get("room", 0), c["page"])
        s["keys"], s["values"] = _pool(g, c, pages)
        table = _table(lengths, c["page"], pages, width, g)
        if c["op"] == "fork":
            # Beams share the first half of their prompt's full pages.
            first = table[torch.arange(count, device="cuda") // c["beams"] * c["beams"]]
            shared = torch.tensor([n // c["page"] // 2 for n in lengths], device="cuda")[:, None]
            table = torch.where(torch.arange(width, device="cuda") < shared, first, table)
            s["parents"] = torch.tensor(_parents(c), dtype=torch.int32, device="cuda")
        s["table"] = table.contiguous()
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    else:
        b, k, v = c["batch"], c["beams"], c["vocab"]
        # Logits on a grid of 1/16, as a 16-bit output gives them near its
        # top: equal ones are common and go to the lower token. The beams'
        # scores put candidates of different beams 1/16/beams apart, so that
        # the rounding of the log-sum decides no order.
        x = torch.randn(b, k, v, generator=g, device="cuda").mul_(48).round_().div_(16)
        s["logits"] = x.to(TYPES[c["type"]])
        total = s["logits"].double().logsumexp(-1)
        s["finished"] = torch.rand(b, k, generator=g, device="cuda") < 0.1
        total = torch.where(s["finished"], (total * 16).round() / 16, total)
        shift = torch.rand(b, k, generator=g, device="cuda").argsort(-1)
        s["scores"] = (total - 24 + (2 * shift + 1) / (32 * k)).float()
        s["finished"] = s["finished"].to(torch.uint8)
    return s


# --- the plain forms -------------------------------------------------------------

def _plain_attention(s):
    c, q, lengths = s["case"], s["q"].float(), s["lengths"].long()
    b, heads, dim = q.shape
    kv = c["kv_heads"]
    position = torch.arange(c["longest"], device="cuda")
    page = s["table"].long()[:, position // c["page"]].clamp(min=0)
    row = position % c["page"]
    keys = s["keys"][page, row].float()  # [batch, longest, kv_heads, dim]
    scores = torch.matmul(q.view(b, kv, heads // kv, dim), keys.permute(0, 2, 3, 1))
    del keys
    scores = (scores * dim ** -0.5).view(b, heads, -1)
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    distance = (lengths[:, None] - 1 - position)[:, None, :]
    if s["slopes"] is not None:
        scores = scores - s["slopes"][None, :, None] * distance
    seen = distance >= 0
    if c["window"]:
        seen = seen & (distance < c["window"])
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    values = s["values"][page, row].float().permute(0, 2, 1, 3)
    out = torch.matmul(weights.view(b, kv, heads // kv, -1), values).view(b, heads, dim)
    out = torch.where(total > 0, out / total, 0.0)
    return {"out": out.to(s["q"].dtype), "lse": (top + torch.log(total))[..., 0]}


def _rotate(x, cos, sin, c):
    """The first `rotary` columns of x turned by the angles of its tokens."""
    r = c["rotary"]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if c["pairs"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_rope(s):
    c = s["case"]
    position, sequence = s["position"].long(), s["sequence"].long()
    cos, sin = s["cos"][position], s["sin"][position]
    page = s["table"].long()[sequence, position // c["page"]]
    row = position % c["page"]
    s["keys"][page, row] = _rotate(s["k"].float(), cos, sin, c).to(s["keys"].dtype)
    s["values"][page, row] = s["v"].to(s["values"].dtype)
    q = _rotate(s["q"].float(), cos, sin, c).to(s["q"].dtype)
    return {"q": q, "keys": s["keys"], "values": s["values"]}


def _plain_fork(s):
    c, page = s["case"], s["case"]["page"]
    table, parents = s["table"].long(), s["parents"].long()
    pages, width = s["keys"].shape[1], table.shape[1]
    count = parents.numel()
    kept = parents >= 0
    lengths = torch.where(kept, s["lengths"].long()[parents.clamp(min=0)], 0)
    rows = table[parents.clamp(min=0)]
    have = (lengths + page - 1) // page
    need = torch.where(kept, (lengths + c["room"] + page - 1) // page, 0)
    column = torch.arange(width, device="cuda")[None, :]
    full = lengths // page
    # A page is in use where a row holds it whole; a row's last, unfinished
    # page stays with the first row that has it, and the others get copies.
    whole = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    whole[torch.where(column < full[:, None], rows, pages).flatten()] = True
    part = lengths % page
    last = rows.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0]
    last = torch.where(part > 0, last, pages)
    index = torch.arange(count, device="cuda")
    owner = torch.full((pages + 1,), count, device="cuda")
    owner.scatter_reduce_(0, last, index, "amin")
    mine = (owner[last] == index) & ~whole[last]
    copies = (part > 0) & ~mine
    taken = whole.clone()
    taken[torch.where((part > 0) & mine, last, pages)] = True
    free = torch.sort(taken[:pages], stable=True)[1]  # the free pages, lowest first
    wanted = copies.long() + need - have
    first = torch.cumsum(wanted, 0) - wanted
    fresh = torch.where(column < have[:, None], 0, column - have[:, None] + copies[:, None].long())
    new = free[(first[:, None] + fresh).clamp(max=pages - 1)]
    is_new = ((column >= have[:, None]) | (copies[:, None] & (column == have[:, None] - 1))) & \
        (column < need[:, None])
    out = torch.where(is_new, new, torch.where(column < have[:, None], rows, -1))
    # The copies, rows of a page after one another.
    source, target = last[copies], out.gather(1, (have - 1).clamp(min=0)[:, None])[copies, 0]
    copied = torch.arange(page, device="cuda") < part[copies][:, None]
    for pool in (s["keys"], s["values"]):
        pool[:, target] = torch.where(copied[None, :, :, None, None], pool[:, source],
                                      pool[:, target])
    left = pages - taken[:pages].sum() - wanted.sum()
    return {"table": out.int(), "lengths": lengths.int(), "free": left.int(), "keys": s["keys"],
            "values": s["values"]}


def _plain_compact(s):
    table = s["table"].long()
    pages = s["keys"].shape[1]
    live = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    live[torch.where(table >= 0, table, pages).flatten()] = True
    live = live[:pages]
    count = live.sum()
    index = torch.arange(pages, device="cuda")
    high, low = live & (index >= count), ~live & (index < count)
    source, target = index[high], index[low]  # as many of the one as of the other
    place = index.clone()
    place[source] = target
    for pool in (s["keys"], s["values"]):
        pool[:, target] = pool[:, source]
    out = torch.where(table >= 0, place[table.clamp(min=0)], -1)
    return {"table": out.int(), "used": count.int(), "keys": s["keys"], "values": s["values"]}


def _plain_beam(s):
    c = s["case"]
    b, k, v, n = c["batch"], c["beams"], c["vocab"], c["count"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    # The best `count` of each beam, equal logits in the tokens' order ...
    best, token = torch.sort(x, dim=-1, descending=True, stable=True)
    best, token = best[..., :n], token[..., :n]
    score = s["scores"][..., None] + (best - total)
    # ... a finished beam goes on as itself, with the end token alone ...
    done = s["finished"][..., None] != 0
    rank = torch.arange(n, device="cuda")
    score = torch.where(done, torch.where(rank == 0, s["scores"][..., None], -math.inf), score)
    token = torch.where(done, 0, token)
    # ... and of all those the best, equal scores in the beams' order.
    score, pick = torch.sort(score.flatten(1), dim=-1, descending=True, stable=True)
    score, pick = score[:, :n], pick[:, :n]
    parent = pick // n
    token = token.flatten(1).gather(1, pick)
    finished = (s["finished"].gather(1, parent) != 0) | (token == 0)
    none = score == -math.inf
    row = torch.arange(b, device="cuda")[:, None] * k + parent
    return {"scores": score, "parents": torch.where(none, -1, row).int(),
            "tokens": torch.where(none, -1, token).int(),
            "finished": torch.where(none, True, finished).to(torch.uint8)}


# --- the framework's operators ------------------------------------------------

_handle = None


def _ops():
    """The handle that a program keeps: the operators on the current stream."""
    global _handle
    if _handle is None:
        import sys
        sys.path.insert(0, "light-rocm-runtime_b200")
        from lrrt_b200 import ops
        _handle = ops.Ops(0)
    return _handle


def _own(s):
    c, ops = s["case"], _ops()
    if c["op"] == "attn":
        out, lse = ops.paged_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"],
                                       softcap=c["cap"], slopes=s["slopes"], window=c["window"])
        return {"out": out, "lse": lse}
    if c["op"] == "rope":
        q = ops.rope_append(s["q"], s["k"], s["v"], s["keys"], s["values"], s["table"],
                            s["sequence"], s["position"], s["cos"], s["sin"],
                            interleaved=c["pairs"] == "interleaved")
        return {"q": q, "keys": s["keys"], "values": s["values"]}
    if c["op"] == "fork":
        table, lengths, status = ops.fork_pages(s["keys"], s["values"], s["table"], s["lengths"],
                                                s["parents"], room=c["room"])
        return {"table": table, "lengths": lengths, "free": status[1], "keys": s["keys"],
                "values": s["values"]}
    if c["op"] == "compact":
        table, status = ops.compact_pages(s["keys"], s["values"], s["table"])
        return {"table": table, "used": status[0], "keys": s["keys"], "values": s["values"]}
    scores, parents, tokens, finished = ops.beam_select(s["logits"], s["scores"], c["count"],
                                                        finished=s["finished"], end_token=0)
    return {"scores": scores, "parents": parents, "tokens": tokens, "finished": finished}


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attention, "rope": _plain_rope, "fork": _plain_fork,
            "compact": _plain_compact, "beam": _plain_beam}[state["case"]["op"]](state)


# --- what a pass cannot do without -----------------------------------------------

def work(case):
    c, size = case, SIZES[case["type"]]
    if c["op"] == "attn":
        seen = sum(min(n, c["window"] or n) for n in _lengths(c, c["batch"]))
        rows = c["batch"] * c["heads"]
        return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * size + 2 * rows * c["dim"] * size +
                4 * rows + 4 * _ceil(seen, c["page"]), "flops": 4 * seen * c["heads"] * c["dim"]}
    if c["op"] == "rope":
        row = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        table = 4 * c["rotary"] * len(set(_tokens(c)[1]))
        return {"bytes": 2 * c["tokens"] * row * size + table + 8 * c["tokens"],
                "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    if c["op"] in ("fork", "compact"):
        token = 2 * c["layers"] * c["kv_heads"] * c["dim"] * size
        if c["op"] == "fork":
            count = c["prompts"] * c["beams"]
            lengths, moved, seen = _lengths(c, count), 0, set()
            for p in _parents(c):
                if p >= 0:
                    moved += (lengths[p - p % c["beams"]] % c["page"]) * (p in seen)
                    seen.add(p)
            table = sum(_ceil(lengths[p - p % c["beams"]], c["page"]) for p in _parents(c)
                        if p >= 0)
        else:
            table = sum(_ceil(n, c["page"]) for n in _lengths(c, c["batch"]))
            pages = table + int(table * c["holes"] / (1 - c["holes"])) + 1
            moved = c["page"] * table * (pages - table) / pages  # of the live pages, those above
        return {"bytes": 2 * token * moved + 8 * table + 64, "flops": 0}
    rows = c["batch"] * c["beams"]
    return {"bytes": rows * c["vocab"] * size + 9 * rows + 13 * c["batch"] * c["count"],
            "flops": 3 * rows * c["vocab"]}


# --- 64 bits, from the definitions ---------------------------------------------

def exact(case, seed):
    c = case
    if c["op"] in ("fork", "compact"):
        return None  # nothing is computed: pages move, tables are whole numbers
    s = prepare(case, seed)
    if c["op"] == "attn":
        outs, sums = [], []
        group = c["heads"] // c["kv_heads"]
        for i, n in enumerate(s["lengths"].tolist()):
            low = max(0, n - c["window"]) if c["window"] else 0
            out = torch.zeros(c["heads"], c["dim"], dtype=torch.float64, device="cuda")
            lse = torch.full((c["heads"],), -math.inf, dtype=torch.float64, device="cuda")
            at = torch.arange(low, n, device="cuda")
            pages = s["table"][i].long()[at // c["page"]]
            for h in range(c["kv_heads"] if n > low else 0):
                mine = slice(h * group, (h + 1) * group)
                k = s["keys"][pages, at % c["page"], h].double()
                v = s["values"][pages, at % c["page"], h].double()
                x = s["q"][i, mine].double() @ k.T / math.sqrt(c["dim"])
                if c["cap"]:
                    x = torch.tanh(x / c["cap"]) * c["cap"]
                if s["slopes"] is not None:
                    x = x + s["slopes"][mine].double()[:, None] * (at - (n - 1))
                lse[mine] = torch.logsumexp(x, -1)
                out[mine] = torch.softmax(x, -1) @ v
            outs.append(out)
            sums.append(lse)
        return {"out": torch.stack(outs), "lse": torch.stack(sums)}
    if c["op"] == "rope":
        # Pairs of columns as complex numbers, turned by e^(i angle) with the
        # tables' cosines and sines.
        r = c["rotary"]
        at = s["position"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None, :]
        done = []
        for x in (s["q"].double(), s["k"].double()):
            y = x.clone()
            first, second = (slice(0, r // 2), slice(r // 2, r)) if c["pairs"] == "half" else \
                (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            done.append(y)
        keys, values = torch.zeros_like(s["keys"], dtype=torch.float64), \
            torch.zeros_like(s["values"], dtype=torch.float64)
        place = (s["table"].long()[s["sequence"].long(), at // c["page"]], at % c["page"])
        keys.index_put_(place, done[1])
        values.index_put_(place, s["v"].double())
        return {"q": done[0], "keys": keys, "values": values}
    # The best scores: each beam's log-probabilities added to its score.
    x = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    done = s["finished"] != 0
    x[done] = -math.inf
    x[..., 0] = torch.where(done, s["scores"].double(), x[..., 0])
    return {"scores": torch.topk(x.flatten(1), c["count"], -1)[0], "parents": None, "tokens": None,
            "finished": None}
