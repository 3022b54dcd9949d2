"""What the attention and eviction operators over the paged cache are measured on.

Four operators of ``ekv.runtime``: ``attend`` (attention over the block table, with prefixes that groups of
rows share read once), ``attend_scored`` (the same for rows whose tokens accumulate the attention weight they
receive), ``select_tokens`` (which tokens of a row to keep by that weight) and ``compact_tokens`` (the kept
tokens moved to the front of the row's blocks). Each case runs one of them; with ``own`` false the same
results come from elementary torch operations.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DECAY = 0.9375


# ---- the cases ---------------------------------------------------------------------------------------


def _attend(name, rows, longest, groups=0, prefix=0, queries=1, q_heads=32, kv_heads=8, dim=128, block=16,
            dtype="bf16", shortest=0.5, empty=0):
    return dict(name=name, op="attend", rows=rows, longest=longest, groups=groups, prefix=prefix, queries=queries,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, block=block, dtype=dtype, shortest=shortest, empty=empty)


def _scored(name, rows, longest, queries=1, q_heads=32, kv_heads=8, dim=128, block=16, dtype="bf16", shortest=0.5,
            empty=0, decay=False, prompt=False):
    return dict(name=name, op="scored", rows=rows, longest=longest, groups=0, prefix=0, queries=queries,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, block=block, dtype=dtype, shortest=shortest, empty=empty,
                decay=decay, prompt=prompt)


def _evict(op, name, rows, longest, keep, first=4, recent=64, kv_heads=8, dim=128, block=16, dtype="bf16",
           shortest=0.5, empty=0):
    return dict(name=name, op=op, rows=rows, longest=longest, groups=0, prefix=0, keep=keep, first=first,
                recent=recent, kv_heads=kv_heads, dim=dim, block=block, dtype=dtype, shortest=shortest, empty=empty)


def listed():
    return [
        # one short request on a small model: latency is all there is
        _attend("attend one short row", 1, 333, q_heads=8, kv_heads=2),
        # an ordinary decode step: 64 requests of up to 8192 tokens, nothing shared
        _attend("attend 64 rows", 64, 8192),
        # 32 samples of one prompt: 8192 shared tokens, a few hundred of their own
        _attend("attend 32 rows one prefix", 32, 700, groups=1, prefix=8192, shortest=0.0),
        # six system prompts, four drafted tokens a request, 64-wide heads
        _attend("attend drafts six prefixes", 48, 301, groups=6, prefix=2000, queries=4, q_heads=64, dim=64,
                dtype="fp16", shortest=0.0),
        # a large batch on one long document
        _attend("attend 256 rows long prefix", 256, 1024, groups=1, prefix=32768, shortest=0.0),
        # a bounded cache in its smallest use
        _scored("scored two short rows", 2, 251, q_heads=8, kv_heads=2),
        # a decode step of 64 requests whose caches are bounded at 4096 tokens
        _scored("scored 64 rows", 64, 4096, decay=True),
        # the last 32 tokens of four prompts score the whole prompt before its first eviction
        _scored("scored prompt windows", 4, 16001, queries=32, q_heads=64, dtype="fp16", prompt=True),
        # the smallest choice: four short rows of a small model
        _evict("select", "select four short rows", 4, 700, 512, kv_heads=2),
        # long prompts cut to an eighth
        _evict("select", "select eight prompts", 8, 65536, 8192, shortest=0.9),
        # the smallest move
        _evict("compact", "compact four short rows", 4, 700, 512, kv_heads=2),
        # a batch cut to half: 64 requests of up to 8192 tokens
        _evict("compact", "compact 64 rows", 64, 8192, 4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "scored", "scored", "select", "compact"])
    q_heads, kv_heads = rng.choice([(8, 2), (32, 8), (64, 8), (40, 8), (8, 8)])
    dim, block, dtype = rng.choice([64, 128, 128]), rng.choice([16, 16, 32]), rng.choice(["bf16", "fp16"])
    rows = _log(rng, 1, 256)
    longest = min(_log(rng, 1, 65536), 64 * 4096 // rows)
    shortest, empty = rng.choice([0.0, 0.5, 0.9]), rng.choice([0, 0, min(3, rows - 1)])
    shape = dict(kv_heads=kv_heads, dim=dim, block=block, dtype=dtype, shortest=shortest, empty=empty)
    if op == "attend":
        queries = rng.choice([1, 1, 1, 2, 5])
        groups = rng.choice([0, 1, 1, rng.randint(1, rows)])
        prefix = min(_log(rng, 1, 32768), 64 * 4096 // groups) if groups else 0
        while 4.0 * dim * q_heads * rows * queries * (prefix + longest) > 1.2e11:
            prefix, longest = prefix // 2, max(1, longest // 2)
        case = _attend("", rows, longest, groups, prefix, queries, q_heads, **shape)
    elif op == "scored":
        queries = rng.choice([1, 1, 1, 3, 16, _log(rng, 1, 64)])
        while 4.0 * dim * q_heads * rows * queries * longest > 3e10:
            longest = max(1, longest // 2)
            queries = queries if longest > 1 else 1
        case = _scored("", rows, longest, queries, q_heads, decay=rng.random() < 0.5, prompt=rng.random() < 0.3, **shape)
    else:
        first, recent, longest = rng.choice([0, 4, 17]), rng.choice([0, 32, 128]), max(longest, 200)
        case = _evict(op, "", rows, longest, rng.randint(first + recent + 1, longest - 1), first, recent, **shape)
    del case["name"]
    return case


# ---- sizes that follow from a case alone ------------------------------------------------------------------


def _sizes(case):
    """Each row's own tokens and each group's first row and shared blocks, the same for every seed."""
    rng = random.Random("%(rows)d %(longest)d %(prefix)d %(block)d" % case)
    rows, queries = case["rows"], case.get("queries", 1)
    own_len = [max(1, queries, round(case["longest"] * rng.uniform(case["shortest"], 1.0))) for _ in range(rows)]
    own_len[0] = max(queries, case["longest"])
    groups = case["groups"]
    starts = [g * rows // groups for g in range(groups)] + [rows] if groups else [0, rows]
    blocks = [max(1, round(case["prefix"] / case["block"] * rng.uniform(0.5, 1.0))) for _ in range(groups)] if groups else [0]
    if groups:
        blocks[0] = -(-case["prefix"] // case["block"])
    shared = [b for g, b in enumerate(blocks) for _ in range(starts[g], starts[g + 1])]  # of each row's prefix
    # a padded batch ends with rows that have nothing in their cache
    lens = [0 if r >= rows - case["empty"] else shared[r] * case["block"] + own_len[r] for r in range(rows)]
    return lens, starts, blocks, shared


def _kept_len(n, case):
    return n if case["keep"] >= n else max(case["keep"], min(n, case["first"] + case["recent"]))


def work(case):
    lens, starts, blocks, shared = _sizes(case)
    heads, dim, block = case["kv_heads"], case["dim"], case["block"]
    if case["op"] in ("attend", "scored"):
        q, qh = case["queries"], case["q_heads"]
        once = sum(b * block for g, b in enumerate(blocks) if starts[g + 1] > starts[g])
        tokens = once + sum(max(0, n - s * block) for n, s in zip(lens, shared))
        seen = sum(q * n - q * (q - 1) // 2 for n in lens if n)
        moved = tokens * heads * dim * 4 + 2 * case["rows"] * q * qh * dim * 2 + case["rows"] * q * qh * 4
        if case["op"] == "scored":
            moved += (8 if not case["prompt"] else 4) * heads * tokens
        return {"bytes": moved + 4 * (tokens // block), "flops": 4 * dim * qh * seen}
    width = -(-max(lens) // block) * block
    if case["op"] == "select":
        return {"bytes": 4 * heads * (sum(lens) + case["rows"] * width) + 8 * case["rows"], "flops": heads * sum(lens)}
    short = [(n, _kept_len(n, case)) for n in lens]
    moved = sum(max(0, k - case["first"]) for n, k in short if k < n)
    return {"bytes": moved * heads * (2 * 2 * dim * 2 + 8 + 4) + 8 * case["rows"], "flops": 0}


# ---- what a caller has in hand --------------------------------------------------------------------------------


def _fill(gen, shape, dtype):
    """Standard normal values, made in slices so that a large cache needs no float32 copy of itself."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    x.normal_(generator=gen)
    return x


def prepare(case, seed):
    lens, starts, blocks, shared = _sizes(case)
    rows, block, heads, dim = case["rows"], case["block"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    width = max(1, -(-max(lens) // block))
    used = [-(-n // block) for n in lens]
    pool = 5 + sum(blocks) + sum(max(0, u - b) for u, b in zip(used, shared))
    if case["op"] != "select":
        ids = torch.randperm(pool, generator=gen, device="cuda").cpu().tolist()
        table, at = [], sum(blocks)
        for g in range(len(blocks)):
            common = ids[sum(blocks[:g]):sum(blocks[:g + 1])]
            for r in range(starts[g], starts[g + 1]):
                mine = max(0, used[r] - len(common))
                row = (common + ids[at:at + mine]) if used[r] else []
                table.append(row + [ids[-1]] * (width - len(row)))  # a block of no row
                at += mine
        s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
        s["cache"] = _fill(gen, (pool, 2, block, heads, dim), dtype)
    if case["op"] in ("attend", "scored"):
        q = case["queries"]
        query = torch.randn(rows * q, case["q_heads"], dim, generator=gen, device="cuda")
        # some keys draw much of the attention, as a prompt's first tokens and its names do: they and the
        # queries lean the same way
        lean = 0.3 * torch.randn(heads, dim, generator=gen, device="cuda")
        s["query"] = (query + lean.repeat_interleave(case["q_heads"] // heads, 0)).to(dtype)
        hot = torch.randint(0, pool * block, (max(1, pool * block // 64),), generator=gen, device="cuda")
        s["cache"][hot // block, 0, hot % block] += (4 * lean).to(dtype)
        s["start"] = torch.arange(0, rows * q + 1, q, dtype=torch.int32, device="cuda")
        s["scale"] = 1 / math.sqrt(dim)
        if case["groups"]:
            s["group_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
            s["prefix_blocks"] = torch.tensor(blocks, dtype=torch.int32, device="cuda")
    if case["op"] != "attend":
        # the weight a token has received falls off steeply from the few heavy ones
        weight = torch.rand(rows, heads, width * block, generator=gen, device="cuda")
        s["scores"] = 0.05 / (weight + 1e-3)
        # the rows' places in the score table are not the batch's order
        s["slots"] = torch.randperm(rows, generator=gen, device="cuda").to(torch.int32)
    if case["op"] == "scored":
        # a prompt's tokens have no scores yet; in a decode step only the step's own tokens have none
        s["fresh"] = s["lens"].clone() if case["prompt"] else None
    if case["op"] == "compact":
        s["kept"], s["new_lens"] = _plain_select(s["scores"], s["lens"], s["slots"], case)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _tokens(cache, table, part, count):
    """[rows, count, heads, dim] in 32 bits: the first `count` tokens' keys (part 0) or values (1) of each table row."""
    block = cache.shape[2]
    blocks = table[:, : -(-count // block)].long()
    x = cache[:, part][blocks]
    return x.reshape(x.shape[0], -1, x.shape[3], x.shape[4])[:, :count].float()


def _weights(q, k, visible, scale):
    """exp(score - max), its row sums and maxima: q [B, M, heads, G, dim], k [B, T, heads, dim], visible [B, M, T]."""
    x = torch.einsum("bmhgd,bthd->bhmgt", q, k) * scale
    x = x.masked_fill(~visible[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.clamp_min(torch.finfo(torch.float32).min))
    return p, p.sum(-1), top[..., 0]


def _values(p, v):
    return torch.einsum("bhmgt,bthd->bmhgd", p, v)


def _plain_attention(s):
    """Output, log-sum-exp and (for one part) the normalised weights: the shared part per group, each row's own part,
    and the two joined."""
    case, cache, table, lens = s["case"], s["cache"], s["table"], s["lens"].long()
    lens_h, starts, blocks, shared = _sizes(case)
    rows, nq, block, heads = case["rows"], case["queries"], case["block"], case["kv_heads"]
    group = case["q_heads"] // heads
    q = s["query"].float().view(rows, nq, heads, group, -1)
    limit = lens[:, None] - nq + 1 + torch.arange(nq, device="cuda")  # positions each query token sees
    before = torch.tensor(shared, device="cuda") * block
    # each row's own tokens: the table from its first unshared block on
    own_blocks = max(1, max(-(-n // block) - b for n, b in zip(lens_h, shared)))
    column = (before // block)[:, None] + torch.arange(own_blocks, device="cuda")
    mine = table.long().gather(1, column.clamp_max(table.shape[1] - 1))
    count = own_blocks * block
    pos = before[:, None] + torch.arange(count, device="cuda")
    inside = pos < lens[:, None]
    k, v = _tokens(cache, mine, 0, count), _tokens(cache, mine, 1, count)
    v = v.masked_fill(~inside[..., None, None], 0.0)
    p, total, top = _weights(q, k, pos[:, None] < limit[..., None], s["scale"])
    out = _values(p, v)
    top_, total_ = top.permute(0, 2, 1, 3), total.permute(0, 2, 1, 3)  # [rows, nq, heads, G]
    if case["groups"]:
        first = torch.tensor(starts[:-1], device="cuda")
        size = max(b - a for a, b in zip(starts, starts[1:]))
        member = (first[:, None] + torch.arange(size, device="cuda")).clamp_max(rows - 1)  # [groups, size]
        common = max(blocks) * block
        lead = first.clamp_max(rows - 1)
        lead = torch.where(lens[lead] > 0, lead, torch.zeros_like(lead))
        kc, vc = _tokens(cache, table[lead], 0, common), _tokens(cache, table[lead], 1, common)
        ends = torch.tensor(blocks, device="cuda") * block
        at = torch.arange(common, device="cuda")
        vc = vc.masked_fill((at >= ends[:, None])[..., None, None], 0.0)
        seen = (at < ends[:, None])[:, None, None] & (at < limit[member][..., None])  # [groups, size, nq, common]
        pc, tc, mc = _weights(q[member].flatten(1, 2), kc, seen.flatten(1, 2), s["scale"])
        oc = _values(pc, vc).view(len(blocks), size, nq, heads, group, -1)
        tc = tc.permute(0, 2, 1, 3).reshape(len(blocks), size, nq, heads, group)
        mc = mc.permute(0, 2, 1, 3).reshape(len(blocks), size, nq, heads, group)
        which = torch.bucketize(torch.arange(rows, device="cuda"), torch.tensor(starts[1:], device="cuda"), right=True)
        place = torch.arange(rows, device="cuda") - first[which]
        oc, tc, mc = oc[which, place], tc[which, place], mc[which, place]
        both = torch.maximum(top_, mc).clamp_min(torch.finfo(torch.float32).min)
        a, c = torch.exp(top_ - both), torch.exp(mc - both)
        out = out * a[..., None] + oc * c[..., None]
        total_ = total_ * a + tc * c
        top_ = both
    some = total_ > 0
    lse = torch.where(some, top_ + torch.log(total_), -math.inf)
    out = torch.where(some[..., None], out / total_[..., None], 0.0)
    out = out.reshape(rows * nq, case["q_heads"], -1).to(s["query"].dtype)
    weights = p / total.clamp_min(torch.finfo(torch.float32).tiny)[..., None]
    return out, lse.reshape(rows * nq, case["q_heads"]), weights


def _plain_scored(s):
    case, lens = s["case"], s["lens"].long()
    out, lse, p = _plain_attention(s)
    received = p.sum((2, 3))  # [rows, heads, count]
    count = received.shape[2]
    at = torch.arange(count, device="cuda")
    fresh = s["fresh"].long() if s["fresh"] is not None else torch.full_like(lens, case["queries"])
    scores, slots = s["scores"], s["slots"].long()
    old = scores[slots][..., :count]
    added = old * (DECAY if case["decay"] else 1.0) + received
    new = torch.where((at >= (lens - fresh)[:, None])[:, None], received, added)
    new = torch.where((at < lens[:, None])[:, None], new, old)
    scores[slots, :, :count] = new
    return out, lse, scores


def _plain_select(scores, lens, slots, case):
    x = scores[slots.long()].nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    n = lens.long()[:, None]
    at = torch.arange(x.shape[2], device="cuda")[None]
    pinned = (at < case["first"]) | (at >= n - case["recent"])
    kind = torch.where(at >= n, 2, torch.where(pinned, 0, 1))  # kept anyway, to choose from, not of the row
    pins = n.clamp_max(case["first"] + case["recent"])
    new = torch.where(case["keep"] >= n, n, pins.clamp_min(case["keep"]))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    kinds = kind[:, None].expand_as(x).gather(-1, order)
    order = order.gather(-1, torch.sort(kinds, dim=-1, stable=True).indices)
    taken = (at < new)[:, None].expand_as(x)
    keep = torch.zeros_like(taken).scatter(-1, order, taken)
    kept = torch.sort((~keep).to(torch.uint8), dim=-1, stable=True).indices
    return torch.where(taken, kept, -1).to(torch.int32), new[:, 0].to(torch.int32)


def _plain_compact(s):
    case, cache, table = s["case"], s["cache"], s["table"].long()
    block, heads = case["block"], case["kv_heads"]
    kept, scores, slots = s["kept"].long(), s["scores"], s["slots"].long()
    at = torch.arange(kept.shape[2], device="cuda").expand_as(kept)
    # what is not moved is read from its own place
    source = torch.where(kept >= 0, kept, at)
    r = torch.arange(kept.shape[0], device="cuda")[:, None, None]
    h = torch.arange(heads, device="cuda")[None, :, None]
    scores[slots] = scores[slots].gather(2, source)
    cache[table[r, at // block], :, at % block, h] = cache[table[r, source // block], :, source % block, h]
    return cache, scores


# ---- one pass --------------------------------------------------------------------------------------------------------


def _modules():
    package = os.path.join(ROOT, "sigmod-kvscope_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ekv.runtime import attention, eviction

    return attention, eviction


def run(s):
    case = s["case"]
    if own:
        attention, eviction = _modules()
        if case["op"] == "attend":
            more = dict(prefix_blocks=s["prefix_blocks"], group_start=s["group_start"]) if case["groups"] else {}
            return attention.attend(s["query"], s["cache"], s["table"], s["lens"], s["scale"], query_start=s["start"], **more)
        if case["op"] == "scored":
            out, lse = attention.attend_scored(
                s["query"], s["cache"], s["table"], s["lens"], s["scale"], s["scores"], query_start=s["start"],
                slots=s["slots"], fresh=s["fresh"], decay=DECAY if case["decay"] else 1.0)
            return out, lse, s["scores"]
        if case["op"] == "select":
            return eviction.select_tokens(s["scores"], s["lens"], case["keep"], first_tokens=case["first"],
                                          recent_tokens=case["recent"], slots=s["slots"])
        eviction.compact_tokens(s["cache"], s["table"], s["lens"], s["kept"], s["new_lens"],
                                first_tokens=case["first"], scores=s["scores"], slots=s["slots"])
        return s["cache"], s["scores"]
    if case["op"] == "attend":
        return _plain_attention(s)[:2]
    if case["op"] == "scored":
        return _plain_scored(s)
    if case["op"] == "select":
        return _plain_select(s["scores"], s["lens"], s["slots"], case)
    return _plain_compact(s)


# ---- the definitions, row by row in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    lens, block = s["lens"].tolist(), case["block"]
    heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "select":
        return None
    if case["op"] == "compact":
        cache, scores = s["cache"].double(), s["scores"].double()
        for r, n in enumerate(lens):
            m, slot, row = int(s["new_lens"][r]), int(s["slots"][r]), s["table"][r].long()
            new = torch.arange(m, device="cuda")
            for h in range(heads if m < n else 0):
                old = s["kept"][r, h, :m].long()
                cache[row[new // block], :, new % block, h] = cache[row[old // block], :, old % block, h]
                scores[slot, h, :m] = scores[slot, h, old]
        return cache, scores
    nq, group = case["queries"], case["q_heads"] // heads
    out = torch.zeros(case["rows"] * nq, case["q_heads"], dim, dtype=torch.float64, device="cuda")
    lse = torch.full((case["rows"] * nq, case["q_heads"]), -math.inf, dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if case["op"] == "scored" else None
    for r, n in enumerate(lens):
        if n == 0:
            continue
        row = s["table"][r, : -(-n // block)].long()
        k = s["cache"][row, 0].reshape(-1, heads, dim)[:n].double()
        v = s["cache"][row, 1].reshape(-1, heads, dim)[:n].double()
        q = s["query"][r * nq:(r + 1) * nq].double().view(nq, heads, group, dim)
        x = torch.matmul(q.permute(1, 0, 2, 3).reshape(heads, nq * group, dim), k.permute(1, 2, 0)) * s["scale"]
        x = x.view(heads, nq, group, n)
        for i in range(nq):
            x[:, i, :, n - nq + 1 + i:] = -math.inf
        total = torch.logsumexp(x, -1)
        p = torch.exp(x - total[..., None])
        o = torch.matmul(p.view(heads, nq * group, n), v.permute(1, 0, 2)).view(heads, nq, group, dim)
        out[r * nq:(r + 1) * nq] = o.permute(1, 0, 2, 3).reshape(nq, -1, dim)
        lse[r * nq:(r + 1) * nq] = total.permute(1, 0, 2).reshape(nq, -1)
        if scores is not None:
            slot, fresh = int(s["slots"][r]), n if case["prompt"] else nq
            got = p.sum((1, 2))
            scores[slot, :, : n - fresh] *= DECAY if case["decay"] else 1.0
            scores[slot, :, n - fresh:n] = 0.0
            scores[slot, :, :n] += got
    return (out, lse) if scores is None else (out, lse, scores)
