"""Token selection and compaction against the oracle: whole numbers and moved bits, so everything is equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as oat

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check_select(scores, lens, keep, first=0, recent=0, slots=None):
    from ekv.runtime.eviction import select_tokens

    rows = len(lens)
    counts = [keep] * rows if isinstance(keep, int) else keep
    got = select_tokens(scores.cuda(), ints(lens), keep if isinstance(keep, int) else ints(keep), first_tokens=first,
                        recent_tokens=recent, slots=None if slots is None else ints(slots))
    want = oat.select(scores.numpy(), np.array(lens), counts, first, recent, slots or list(range(rows)))
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    return got


@pytest.mark.parametrize("keep, first, recent", [(0, 0, 0), (1, 0, 0), (40, 4, 16), (3, 4, 16), (511, 0, 0), (10**9, 4, 16),
                                                 (-1, 0, 0), (64, 0, 64), (64, 64, 0)])
def test_select_over_lengths(cuda_lib, keep, first, recent):
    lens = [0, 1, 2, 16, 17, 40, 41, 511, 512, 513, 1023, 1200]
    scores = torch.rand(len(lens), 3, 1200, generator=torch.Generator().manual_seed(1))
    check_select(scores, lens, keep, first, recent)


def test_select_ties_and_values_that_are_not_numbers(cuda_lib):
    gen = torch.Generator().manual_seed(2)
    scores = torch.randint(-2, 3, (4, 2, 700), generator=gen).float()
    scores[1] = 0.5  # every token ties
    scores[1, 1, ::2] = -0.0
    scores[1, 1, 1::2] = 0.0  # and the two zeros do
    scores[2, :, ::3] = float("nan")
    scores[2, :, 1::7] = float("-inf")
    scores[2, :, 5::11] = float("inf")
    scores[3] = float("nan")
    for keep in (1, 100, 350, 699):
        check_select(scores, [700, 700, 699, 650], keep, 2, 5)


def test_select_per_row_counts_and_slots(cuda_lib):
    scores = torch.rand(6, 2, 90, generator=torch.Generator().manual_seed(3))
    check_select(scores, [90, 80, 70, 60, 50], [10, -1, 0, 60, 49], 1, 3, slots=[5, 0, 0, -1, 2])


def test_select_reports_what_it_clamps(cuda_lib):
    import ekv._lib as L
    from ekv.runtime.eviction import select_tokens

    scores = torch.rand(2, 1, 50, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept, new = select_tokens(scores, ints([60, 30]), 20, slots=ints([0, 2]), status=status)
    assert int(status) == L.STATUS_LEN_OVER_WIDTH | L.STATUS_BAD_SLOT
    assert new.tolist() == [20, 30] and kept[1, 0, :30].tolist() == list(range(30)) and torch.all(kept[0] < 50)


@pytest.mark.parametrize("n", [8192, 40000, 131072])
def test_select_from_long_rows(cuda_lib, n):
    scores = torch.rand(2, 2, n, generator=torch.Generator().manual_seed(n))
    scores[1] = (scores[1] * 50).floor()  # many ties
    check_select(scores, [n, n - 3], n // 3, 4, 128)


# ---- compaction --------------------------------------------------------------------------------------


def batch(seed, lens, heads=2, dim=128, block=16, dtype=torch.bfloat16, width=None):
    gen = torch.Generator().manual_seed(seed)
    width = width or max(1, max(-(-n // block) for n in lens))
    pool = len(lens) * width + 3
    table = torch.randperm(pool, generator=gen)[: len(lens) * width].reshape(len(lens), width).to(torch.int32)
    cache = torch.randint(0, 1 << 15, (pool, 2, block, heads, dim), generator=gen).to(torch.int16).view(dtype)
    scores = torch.rand(len(lens) + 1, heads, width * block, generator=gen)
    return cache, scores, table


def check_compact(cache, scores, table, lens, kept, new_lens, slots, first=0, with_scores=True):
    from ekv.runtime.eviction import compact_tokens

    got, got_scores = cache.cuda(), scores.cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    compact_tokens(got, table.cuda(), ints(lens), kept.cuda(), new_lens.cuda(), first_tokens=first, status=status,
                   **(dict(scores=got_scores, slots=ints(slots)) if with_scores else {}))
    # moved bits: compared as whole numbers
    want, want_scores = oat.compact(cache.view(torch.uint8).numpy(), scores.numpy(), table.numpy(), lens, kept.cpu().numpy(),
                                    new_lens.tolist(), slots)
    assert int(status) == 0
    np.testing.assert_array_equal(got.cpu().view(torch.uint8).numpy(), want)
    if with_scores:
        np.testing.assert_array_equal(got_scores.cpu().numpy(), want_scores)


@pytest.mark.parametrize("dtype, dim, block, heads", [(torch.bfloat16, 128, 16, 2), (torch.float16, 64, 8, 3),
                                                      (torch.float32, 96, 32, 1), (torch.uint8, 128, 16, 2)])
@pytest.mark.parametrize("keep", [1, 63, 200, 499])
def test_compact_what_select_kept(cuda_lib, dtype, dim, block, heads, keep):
    from ekv.runtime.eviction import select_tokens

    lens = [0, 1, 64, 65, 200, 500, 777]
    if dtype == torch.uint8:
        cache, scores, table = batch(1, lens, heads, dim // 2, block, torch.float16)
        cache = cache.view(torch.uint8)
    elif dtype == torch.float32:
        cache, scores, table = batch(1, lens, heads, dim * 2, block, torch.float16)
        cache = cache.view(torch.float32)
    else:
        cache, scores, table = batch(1, lens, heads, dim, block, dtype)
    slots = [3, 7, 0, 1, 6, 2, 5]
    kept, new = select_tokens(scores.cuda(), ints(lens), keep, first_tokens=3, recent_tokens=20, slots=ints(slots))
    check_compact(cache, scores, table, lens, kept.cpu(), new.cpu(), slots, first=3)
    check_compact(cache, scores, table, lens, kept.cpu(), new.cpu(), slots, with_scores=False)


def test_compact_one_token_fewer(cuda_lib):
    """Every later token moves by one place, onto its neighbour's."""
    lens = [1000, 333]
    cache, scores, table = batch(2, lens)
    kept = torch.stack([torch.tensor([[i for i in range(1008) if i != hole] for hole in pair]) for pair in ((0, 998), (5, 100))])
    check_compact(cache, scores, table, lens, kept.to(torch.int32), torch.tensor([999, 332], dtype=torch.int32), [0, 1])


def refused(status_name, cache, table, lens, kept, new, first=0, scores=None, slots=None, moved=()):
    """The status, and that every row but those in `moved` is left as it was: with a small table, and with one so wide that its
    blocks are not compared with one another."""
    import ekv._lib as L
    from ekv.runtime.eviction import compact_tokens

    if table.shape[1] < 300 and scores is None:
        wide = torch.full((len(table), 300), -1, dtype=torch.int32)
        wide[:, : table.shape[1]] = table
        refused(status_name, cache, wide, lens, kept, new, first, moved=moved)
    got = cache.cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    extra = {} if scores is None else dict(scores=scores, slots=slots)
    compact_tokens(got, table.cuda(), ints(lens), kept.cuda(), ints(new), first_tokens=first, status=status, **extra)
    assert int(status) == getattr(L, status_name)
    want, _ = oat.compact(cache.view(torch.uint8).numpy(), None, table.numpy(), lens, kept.numpy(),
                          [m if r in moved else -1 for r, m in enumerate(new)], list(range(len(lens))))
    np.testing.assert_array_equal(got.cpu().view(torch.uint8).numpy(), want)


def lists(rows, heads, columns, step=2):
    return (torch.arange(columns) * step).to(torch.int32).expand(rows, heads, columns).contiguous()


def test_compact_refuses_lists_that_do_not_ascend(cuda_lib):
    cache, _, table = batch(3, [100, 100, 100])
    good = lists(3, 2, 50)
    for entry, value in ((10, 19), (10, 18), (49, 100), (0, -1), (30, 10**9)):
        kept = good.clone()
        kept[1, 1, entry] = value
        if value == 19:
            kept[1, 1, entry + 1] = 19  # the same token twice
        refused("STATUS_BAD_LIST", cache, table, [100] * 3, kept, [50] * 3, moved=(0, 2))
    refused("STATUS_BAD_LIST", cache, table, [100] * 3, good, [50, 51, 50], moved=(0, 2))  # more than the list holds
    refused("STATUS_BAD_LIST", cache, table, [100] * 3, good, [50] * 3, first=2)  # the second token is not kept


def test_compact_refuses_blocks_of_two_rows(cuda_lib):
    cache, _, table = batch(4, [100, 100, 100, 100])
    kept = lists(4, 2, 50)
    shared = table.clone()
    shared[2, 5] = table[0, 1]
    refused("STATUS_BLOCK_SHARED", cache, shared, [100] * 4, kept, [50] * 4, moved=(1, 3))
    refused("STATUS_BLOCK_SHARED", cache, shared, [100] * 4, kept, [50, 50, 100, 50], moved=(1, 3))  # row 2 keeps everything
    twice = table.clone()
    twice[1, 3] = table[1, 2]
    refused("STATUS_BLOCK_SHARED", cache, twice, [100] * 4, kept, [50] * 4, moved=(0, 2, 3))
    behind = table.clone()
    behind[2, 6] = table[0, 1]  # listed behind the row's 96 tokens
    check_compact(cache, torch.zeros(5, 2, 112), behind, [100, 100, 96, 100], lists(4, 2, 48), torch.tensor([48] * 4, dtype=torch.int32), [0, 1, 2, 3])


def test_compact_leaves_a_shared_prefix_alone(cuda_lib):
    cache, scores, table = batch(5, [100, 90, 80])
    table[1:, :2] = table[0, :2].clone()
    kept = lists(3, 2, 60)
    kept[:, :, :37] = torch.arange(37, dtype=torch.int32)
    kept[:, :, 37:] = 38 + torch.arange(23, dtype=torch.int32)
    check_compact(cache, scores, table, [100, 90, 80], kept, torch.tensor([60, 60, 60], dtype=torch.int32), [0, 1, 2], first=37)
    refused("STATUS_BLOCK_SHARED", cache, table, [100, 90, 80], kept, [60] * 3, first=31)  # block 1 is not protected whole


def test_compact_refuses_blocks_and_slots_outside_their_tables(cuda_lib):
    cache, scores, table = batch(6, [100, 100])
    kept = lists(2, 2, 50)
    for bad in (-1, cache.shape[0], 2**31 - 1):
        broken = table.clone()
        broken[0, 3] = bad
        refused("STATUS_BAD_BLOCK_ID", cache, broken, [100, 100], kept, [50, 50], moved=(1,))
    refused("STATUS_BAD_SLOT", cache, table, [100, 100], kept, [50, 50], scores=scores.cuda(), slots=ints([3, 1]), moved=(1,))
    refused("STATUS_BAD_SLOT", cache, table, [100, 100], kept, [50, 50], scores=scores.cuda(), slots=ints([1, 1]))


def test_tables_with_the_heads_outermost_and_a_strided_cache(cuda_lib):
    from ekv.runtime.eviction import compact_tokens, select_tokens

    lens = [100, 333, 50]
    cache, scores, table = batch(7, lens, heads=3)
    slots = [2, 0, 3]
    outer = scores.permute(1, 0, 2).contiguous().cuda().permute(1, 0, 2)
    kept = torch.empty(3, 3, scores.shape[2] + 5, dtype=torch.int32, device="cuda").permute(1, 0, 2)[..., 2:-3]
    got, new = select_tokens(outer, ints(lens), 40, first_tokens=1, recent_tokens=7, slots=ints(slots), kept=kept)
    want = oat.select(scores.numpy(), np.array(lens), [40] * 3, 1, 7, slots)
    np.testing.assert_array_equal(got.cpu().numpy(), want[0])
    blocks, _, block, heads, dim = cache.shape
    strided = torch.empty(blocks, heads, block, 2, dim + 8, dtype=cache.dtype, device="cuda").permute(0, 3, 2, 1, 4)[..., 8:]
    strided.copy_(cache)
    compact_tokens(strided, table.cuda(), ints(lens), got, new, first_tokens=1, scores=outer, slots=ints(slots))
    moved, moved_scores = oat.compact(cache.view(torch.uint8).numpy(), scores.numpy(), table.numpy(), lens, want[0], want[1], slots)
    np.testing.assert_array_equal(strided.contiguous().cpu().view(torch.uint8).numpy(), moved)
    np.testing.assert_array_equal(outer.cpu().numpy(), moved_scores)


def test_eviction_in_a_replayed_graph_and_on_another_stream(cuda_lib):
    from ekv.runtime.eviction import compact_tokens, select_tokens

    lens = [500, 64, 0, 700]
    cache, scores, table = batch(8, lens)
    dev_cache, dev_scores, dev_lens, tab = cache.cuda(), scores.cuda(), ints(lens), table.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = select_tokens(dev_scores, dev_lens, 100, first_tokens=4, recent_tokens=8)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, new = select_tokens(dev_scores, dev_lens, 100, first_tokens=4, recent_tokens=8)
        compact_tokens(dev_cache, tab, dev_lens, kept, new, first_tokens=4, scores=dev_scores)
    for shift in (0, 37):  # the graph again, on another batch
        now = [max(n - shift, 0) for n in lens]
        dev_cache.copy_(cache)
        dev_scores.copy_(scores)
        dev_lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        want = oat.select(scores.numpy(), np.array(now), [100] * 4, 4, 8, [0, 1, 2, 3])
        np.testing.assert_array_equal(kept.cpu().numpy(), want[0])
        if shift == 0:
            np.testing.assert_array_equal(first[0].cpu().numpy(), want[0])
        moved, moved_scores = oat.compact(cache.view(torch.uint8).numpy(), scores.numpy(), table.numpy(), now, want[0], want[1], [0, 1, 2, 3])
        np.testing.assert_array_equal(dev_cache.cpu().view(torch.uint8).numpy(), moved)
        np.testing.assert_array_equal(dev_scores.cpu().numpy(), moved_scores)


def test_one_long_row(cuda_lib):
    """Clusters of CTAs over one row, keys and values apart, and positions past 2^16."""
    lens = [70001]
    cache, scores, table = batch(9, lens, heads=1, dim=64)
    gen = torch.Generator().manual_seed(1)
    drop = torch.randperm(70001, generator=gen)[:9000]
    keep = torch.ones(70001, dtype=torch.bool)
    keep[drop] = False
    keep[:100] = True
    kept = torch.nonzero(keep)[:, 0].to(torch.int32).view(1, 1, -1)
    check_compact(cache, scores, table, lens, kept, torch.tensor([kept.shape[2]], dtype=torch.int32), [1], first=100)


def test_a_bounded_cache_over_many_steps(cuda_lib):
    """Attend, add the weights up, and at 96 tokens cut the row to 64: the cache as a serving loop uses it, against the
    same loop in float64 over lists of tokens."""
    from ekv.runtime.attention import attend_scored
    from ekv.runtime.eviction import compact_tokens, select_tokens

    rows, heads, q_heads, dim, block, width, scale = 3, 2, 8, 64, 16, 6, 0.2
    gen = torch.Generator().manual_seed(9)
    cache = torch.zeros(rows * width + 1, 2, block, heads, dim, dtype=torch.float16, device="cuda")
    table = torch.randperm(rows * width + 1, generator=gen)[: rows * width].reshape(rows, width).to(torch.int32)
    tab = table.cuda()
    scores = torch.full((rows, heads, width * block), float("nan"), device="cuda")
    lens = [90, 30, 95]
    host = [[(torch.randn(heads, dim, generator=gen).half(), torch.randn(heads, dim, generator=gen).half()) for _ in range(n)]
            for n in lens]
    keys = [[[tok[0][h] for tok in row] for h in range(heads)] for row in host]
    vals = [[[tok[1][h] for tok in row] for h in range(heads)] for row in host]
    for r, n in enumerate(lens):
        for t in range(n):
            for h in range(heads):
                cache[table[r, t // block], 0, t % block, h] = keys[r][h][t].cuda()
                cache[table[r, t // block], 1, t % block, h] = vals[r][h][t].cuda()
    weight = [[np.zeros(0) for _ in range(heads)] for _ in range(rows)]
    fresh = ints(lens)
    evictions = 0
    for step in range(25):
        query = torch.randn(rows, q_heads, dim, generator=gen).half()
        out, _ = attend_scored(query.cuda(), cache, tab, ints(lens), scale, scores, fresh=fresh)
        fresh = None
        for r in range(rows):
            for h in range(heads):
                k = torch.stack(keys[r][h]).double().numpy()
                v = torch.stack(vals[r][h]).double().numpy()
                x = query[r, h * 4:(h + 1) * 4].double().numpy() @ k.T * scale
                p = np.exp(x - x.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                got = out[r, h * 4:(h + 1) * 4].double().cpu().numpy()
                assert np.all(np.abs(got - p @ v) <= 2**-11 * (np.abs(p @ v) + 1.1 * np.abs(v).max()) + 1e-4)
                w = weight[r][h]
                weight[r][h] = np.concatenate([w, np.zeros(len(k) - len(w))]) + p.sum(0)
        counts = [64 if n >= 96 else -1 for n in lens]
        kept, new = select_tokens(scores, ints(lens), ints(counts), first_tokens=2, recent_tokens=8)
        compact_tokens(cache, tab, ints(lens), kept, new, first_tokens=2, scores=scores)
        for r in range(rows):
            if counts[r] < 0:
                continue
            evictions += 1
            for h in range(heads):
                took = kept[r, h, :64].tolist()
                want = weight[r][h]
                inner = np.array([t for t in range(2, lens[r] - 8)])
                chosen = np.array([t for t in took if t in set(inner.tolist())])
                dropped = np.setdiff1d(inner, chosen)
                # float32 sums of 25 weights may order two nearly equal tokens the other way
                assert want[chosen].min() >= want[dropped].max() - 1e-4
                assert took[:2] == [0, 1] and took[-8:] == list(range(lens[r] - 8, lens[r]))
                keys[r][h], vals[r][h], weight[r][h] = ([a[t] for t in took] for a in (keys[r][h], vals[r][h], want))
        lens = new.tolist()
        for r in range(rows):  # the step's own token
            t = lens[r]
            tok = torch.randn(2, heads, dim, generator=gen).half()
            cache[table[r, t // block], :, t % block] = tok.cuda()
            for h in range(heads):
                keys[r][h].append(tok[0, h])
                vals[r][h].append(tok[1, h])
            lens[r] = t + 1
    assert evictions >= 2
    np.testing.assert_allclose(scores[1, 0, : lens[1] - 1].cpu().numpy(), weight[1][0], rtol=1e-5, atol=1e-4)


# ---- protected blocks ---------------------------------------------------------------------------------


def first_then_every_other(rows, heads, first, columns):
    """Lists that keep the first tokens in place and every other one behind them."""
    kept = first + 2 + 2 * torch.arange(columns, dtype=torch.int32)
    kept = torch.cat([torch.arange(first, dtype=torch.int32), kept])[:columns]
    return kept.expand(rows, heads, columns).contiguous()


@pytest.mark.parametrize("lens, new, moved", [([100] * 4, [50] * 4, (0, 2, 3)), ([100, 100, 14, 100], [50, 50, 9, 50], (0, 2, 3)),
                                              ([100] * 4, [100, 50, 50, 50], (2, 3))])
def test_compact_refuses_to_write_another_rows_protected_block(cuda_lib, lens, new, moved):
    """Row 1 lists, where its own tokens go, a block of which other rows keep the first tokens in place; they stay as they
    are, also where those rows are moved, are shorter than what is kept in place, or are not moved at all."""
    cache, _, table = batch(11, lens, width=7)
    table[3, 0] = table[0, 0]  # a prefix of two rows
    broken = table.clone()
    broken[1, 2] = table[0, 0]
    refused("STATUS_BLOCK_SHARED", cache, broken, lens, first_then_every_other(4, 2, 16, 50), new, first=16, moved=moved)


def test_compact_refuses_a_row_that_repeats_its_own_protected_block(cuda_lib):
    cache, _, table = batch(12, [100] * 4)
    kept = first_then_every_other(4, 2, 33, 50)
    for where in (2, 5):  # among the blocks that tokens move to, and among those that they leave
        broken = table.clone()
        broken[2, where] = table[2, 1]
        refused("STATUS_BLOCK_SHARED", cache, broken, [100] * 4, kept, [50] * 4, first=33, moved=(0, 1, 3))


def test_many_rows_with_one_prefix_and_some_that_would_write_it(cuda_lib):
    """Claims and protections of the same blocks from many CTAs at once: the outcome is the same in every run."""
    import ekv._lib as L
    from ekv.runtime.eviction import compact_tokens

    rows = 96
    cache, _, table = batch(13, [100] * rows, heads=1, dim=64)
    table[:, :2] = table[0, :2].clone()
    wrong = [5, 50]  # of different blocks
    for r in wrong:
        table[r, 3 + r % 3] = table[0, r % 2]
    kept = first_then_every_other(rows, 1, 32, 60)
    new = [60] * rows
    want, _ = oat.compact(cache.view(torch.uint8).numpy(), None, table.numpy(), [100] * rows, kept.numpy(),
                          [-1 if r in wrong else 60 for r in range(rows)], list(range(rows)))
    for _ in range(5):
        got, status = cache.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
        compact_tokens(got, table.cuda(), ints([100] * rows), kept.cuda(), ints(new), first_tokens=32, status=status)
        assert int(status) == L.STATUS_BLOCK_SHARED
        np.testing.assert_array_equal(got.cpu().view(torch.uint8).numpy(), want)


def test_a_replayed_graph_over_a_large_table(cuda_lib):
    """More than 512 table entries: the owner table is cleared by every replay, so one batch leaves the next nothing."""
    from ekv.runtime.eviction import compact_tokens

    lens = [500, 640, 30, 700]
    cache, _, table = batch(14, lens, width=200)
    kept = first_then_every_other(4, 2, 16, 200)
    dev, tab, new, status = cache.cuda(), table.cuda(), ints([200, 200, 30, 200]), torch.zeros(1, dtype=torch.int32, device="cuda")
    dev_lens, dev_kept = ints(lens), kept.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        compact_tokens(dev, tab, dev_lens, dev_kept, new, first_tokens=16, status=status)
    shared = table.clone()
    shared[3, 5] = table[1, 0]
    for now, left in ((table, ()), (shared, (3,)), (table.flip(0).contiguous(), ())):
        now_lens = lens if now is not shared else [500, 640, 0, 700]
        dev.copy_(cache)
        tab.copy_(now)
        dev_lens.copy_(torch.tensor(now_lens, dtype=torch.int32))
        status.zero_()
        graph.replay()
        assert (int(status) != 0) == bool(left)
        want, _ = oat.compact(cache.view(torch.uint8).numpy(), None, now.numpy(), now_lens, kept.numpy(),
                              [-1 if r in left else m for r, m in enumerate([200, 200, 30, 200])], list(range(4)))
        np.testing.assert_array_equal(dev.cpu().view(torch.uint8).numpy(), want)


# ---- what became of each row ------------------------------------------------------------------------------


@pytest.mark.parametrize("width", [7, 300])
def test_compact_reports_each_rows_length(cuda_lib, width):
    """Moved, not shrinking, with nothing in its cache, and refused for each reason: with few blocks and with many."""
    import ekv._lib as L
    from ekv.runtime.eviction import compact_tokens

    lens = [100, 100, 0, 100, 100, 100, 100, 100, 100, 1]
    cache, _, table = batch(15, lens, width=width)
    scores = torch.rand(10, 2, width * 16, device="cuda")
    table[4, 3] = table[3, 2]  # rows 3 and 4 share a block, the kept lists of row 5 do not ascend, row 6 has a block outside the pool
    kept = lists(10, 2, 50)
    kept[5, 1, 7] = 3
    table[6, 6] = -1
    slots = [0, 1, 2, 3, 4, 5, 6, 7, 10, 9]  # row 8's is outside the table
    new = [50, 100, 0, 50, 50, 50, 50, 50, 50, 0]
    after, status = ints([-7] * 11), torch.zeros(1, dtype=torch.int32, device="cuda")
    got = cache.cuda()
    compact_tokens(got, table.cuda(), ints(lens), kept.cuda(), ints(new), scores=scores, slots=ints(slots), result_lens=after,
                   status=status)
    assert int(status) == L.STATUS_BLOCK_SHARED | L.STATUS_BAD_LIST | L.STATUS_BAD_BLOCK_ID | L.STATUS_BAD_SLOT
    assert after.tolist() == [50, 100, 0, 100, 100, 100, 100, 50, 100, 0, -7]
    moved = [m if r in (0, 7, 9) else -1 for r, m in enumerate(new)]
    want, _ = oat.compact(cache.view(torch.uint8).numpy(), None, table.numpy(), lens, kept.numpy(), moved, list(range(10)))
    np.testing.assert_array_equal(got.cpu().view(torch.uint8).numpy(), want)


def test_a_refused_row_goes_on_with_all_of_its_tokens(cuda_lib):
    """Select, compact and attend by the reported lengths: the refused row attends as before, the moved one to what it kept."""
    from ekv.runtime.attention import attend
    from ekv.runtime.eviction import compact_tokens, select_tokens

    lens = [100, 100, 100]
    gen = torch.Generator().manual_seed(16)
    table = torch.randperm(21, generator=gen).reshape(3, 7).to(torch.int32)
    table[2, :2] = table[1, :2].clone()  # a shared prefix that no first_tokens covers
    cache = torch.randn(21, 2, 16, 2, 64, generator=gen).half()
    query = torch.randn(3, 4, 64, generator=gen).half()
    scores = torch.rand(3, 2, 112, generator=gen)
    dev, after = cache.cuda(), ints([0] * 3)
    kept, new = select_tokens(scores.cuda(), ints(lens), 40, first_tokens=4, recent_tokens=8)
    compact_tokens(dev, table.cuda(), ints(lens), kept, new, first_tokens=4, scores=scores.cuda(), result_lens=after)
    assert after.tolist() == [40, 100, 100] and new.tolist() == [40, 40, 40]
    out, _ = attend(query.cuda(), dev, table.cuda(), after, 0.1)
    whole, _ = attend(query.cuda(), cache.cuda(), table.cuda(), ints(lens), 0.1)
    assert torch.equal(out[1:], whole[1:])
    for h in range(2):
        at = kept[0, h, :40].cpu().long()
        k, v = (cache[table[0, at // 16].long(), part, at % 16, h].double() for part in (0, 1))
        p = torch.softmax(query[0, 2 * h : 2 * h + 2].double() @ k.T * 0.1, -1)
        # half a step of the output and one of each probability, both relative to 2^-11
        assert torch.all((out[0, 2 * h : 2 * h + 2].double().cpu() - p @ v).abs() <= 2**-11 * ((p @ v).abs() + 1.1 * v.abs().max()) + 1e-4)


def test_counts_of_any_whole_number_type(cuda_lib):
    from ekv.runtime.attention import attend
    from ekv.runtime.eviction import compact_tokens, select_tokens

    scores = torch.rand(2, 1, 90, generator=torch.Generator().manual_seed(17)).cuda()
    want = select_tokens(scores, ints([90, 70]), 40, first_tokens=3, recent_tokens=5)
    for kind in (np.int64, np.uint8, lambda v: torch.tensor(v).numpy(), lambda v: type("Count", (), {"__index__": lambda _: v})()):
        got = select_tokens(scores, ints([90, 70]), kind(40), first_tokens=kind(3), recent_tokens=kind(5))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for keep in (2**40, -(2**40)):
        assert select_tokens(scores, ints([90, 70]), keep, first_tokens=2**40)[1].tolist() == [90, 70]
    cache, _, table = batch(18, [90, 70], heads=1, dim=64)
    compact_tokens(cache.cuda(), table.cuda(), ints([90, 70]), want[0], want[1], first_tokens=np.int32(3))
    query = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(19)).bfloat16().cuda()
    table[1] = table[0].clone()
    dev = torch.randn(cache.shape, generator=torch.Generator().manual_seed(20)).bfloat16().cuda()
    out = [attend(query, dev, table.cuda(), ints([90, 90]), 0.1, prefix_blocks=n)[0] for n in (6, np.int64(6), 2**31, 2**32, 2**40)]
    assert all(torch.equal(out[0], o) for o in out)
