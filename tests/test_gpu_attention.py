"""Attention over the paged cache against the float64 oracle: lengths, masks, layouts, shared prefixes.

Tolerances. ``out`` is rounded to its type (half a step, u = eps / 2 relative) and its probabilities were rounded to
the same type before the products with the values, each off by at most u relative: |error| <= u |out| + u (1 + u)
sum_j p_j |v_j| <= u (|out| + 1.01 max |v|). Float32 work (scores of at most 128 products, sums) adds relative errors
below 128 * 2^-24 * sum |q k| * scale in the exponent; with the inputs here (|x| <= 40) 3e-5 covers it. fp16
probabilities below 2^-14 are off by at most 2^-25 each, 2^-25 * n * max |v| in all: 2^-25 * 1024 < u / 8.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import attention as oat

pytestmark = pytest.mark.gpu


def make(seed, lens, queries=None, q_heads=8, kv_heads=2, dim=128, block=16, dtype=torch.bfloat16, width=None,
         groups=None, spare=3):
    """A batch: rows with their own blocks, except that a group (first row, last row, blocks) shares its prefix."""
    gen = torch.Generator().manual_seed(seed)
    rows = len(lens)
    width = width or max(1, max(-(-n // block) for n in lens))
    pool = rows * width + spare
    table = torch.randperm(pool, generator=gen)[: rows * width].reshape(rows, width).to(torch.int32)
    for a, b, shared in groups or []:
        table[a:b, :shared] = table[a, :shared].clone()
    queries = [1] * rows if queries is None else queries
    start = torch.tensor(np.concatenate([[0], np.cumsum(queries)]), dtype=torch.int32)
    query = torch.randn(int(start[-1]), q_heads, dim, generator=gen).to(dtype)
    cache = torch.randn(pool, 2, block, kv_heads, dim, generator=gen).to(dtype)
    return dict(query=query, cache=cache, table=table, lens=torch.tensor(lens, dtype=torch.int32), start=start)


def widen(x, tokens=1 << 16):
    """The same rows in a table that could hold many more tokens, which is what the kernel for many query rows is picked by."""
    block = x["cache"].shape[2]
    more = torch.full((len(x["table"]), tokens // block - x["table"].shape[1]), -1, dtype=torch.int32)
    return dict(x, table=torch.cat([x["table"], more], 1))


def on_device(x):
    return {k: v.cuda() for k, v in x.items()}


def check(got, x, scale, dtype, pool_ok=None, start=True):
    out, lse, _ = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(),
                             x["lens"].numpy(), scale, x["start"].numpy() if start else None, pool_ok)
    u = torch.finfo(dtype).eps / 2
    biggest = x["cache"][:, 1].float().nan_to_num(0, 0, 0).abs().max().item()
    some = ~np.isnan(lse)
    o, e = got[0].float().cpu().numpy().astype(np.float64)[some], got[1].cpu().numpy().astype(np.float64)[some]
    np.testing.assert_array_equal(np.isinf(e), np.isinf(lse[some]))
    live = np.isfinite(lse[some])
    np.testing.assert_allclose(e[live], lse[some][live], rtol=0, atol=3e-5)
    assert np.all(np.abs(o - out[some]) <= 1.05 * u * (np.abs(out[some]) + 1.01 * biggest) + 3e-5 * biggest)
    assert np.all(o[~live] == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, block", [(128, 16), (64, 16), (128, 8), (64, 32), (128, 64)])
def test_decode_rows_of_every_length(cuda_lib, dtype, dim, block):
    from ekv.runtime.attention import attend

    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 641]
    x = make(1, lens, dim=dim, block=block, dtype=dtype)
    d = on_device(x)
    got = attend(d["query"], d["cache"], d["table"], d["lens"], 1 / math.sqrt(dim))
    check(got, x, 1 / math.sqrt(dim), dtype, start=False)


@pytest.mark.parametrize("wide", [False, True])
def test_short_rows_with_and_without_a_wide_table(cuda_lib, wide):
    """Rows of at most 512 tokens in few items get a CTA each; a table that could hold longer ones has their tiles dealt."""
    from ekv.runtime.attention import attend

    x = make(33, [333, 0, 512, 1, 64], queries=[1, 3, 2, 0, 9], width=33 if wide else 32)
    d = on_device(x)
    out, lse = torch.full_like(d["query"], 7.0), torch.full(tuple(d["query"].shape[:2]), 7.0, device="cuda")
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], out=out, lse=lse), x, 0.1, torch.bfloat16)


@pytest.mark.parametrize("q_heads, kv_heads", [(2, 2), (10, 2), (16, 1), (32, 1), (12, 3), (48, 1)])
def test_head_groups(cuda_lib, q_heads, kv_heads):
    from ekv.runtime.attention import attend

    x = make(2, [70, 333, 5], q_heads=q_heads, kv_heads=kv_heads)
    d = on_device(x)
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.09), x, 0.09, torch.bfloat16, start=False)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("queries", [[1, 4, 2, 1], [0, 7, 0, 3], [33, 1, 20, 64], [5, 5, 5, 5]])
def test_several_query_tokens_a_row(cuda_lib, queries, wide):
    from ekv.runtime.attention import attend

    x = make(3, [100, 64, 33, 200], queries=queries, dtype=torch.float16)
    x = widen(x) if wide else x
    d = on_device(x)
    got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"])
    check(got, x, 0.1, torch.float16)


@pytest.mark.parametrize("scale", [1e-38, 1e-4, 1.0])
def test_scales(cuda_lib, scale):
    from ekv.runtime.attention import attend

    x = make(42, [150, 700, 20], queries=[30, 1, 25], q_heads=16)
    for y in (x, widen(x)):
        d = on_device(y)
        check(attend(d["query"], d["cache"], d["table"], d["lens"], scale, query_start=d["start"]), y, scale, torch.bfloat16)


def test_more_query_tokens_than_cached_ones(cuda_lib):
    from ekv.runtime.attention import attend

    x = make(4, [3, 0, 20], queries=[5, 2, 1])  # the first tokens of row 0 see nothing, nor do row 1's
    d = on_device(x)
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"]), x, 0.1, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries", [1, 3])
@pytest.mark.parametrize("groups", [[(0, 6, 5)], [(0, 2, 9), (2, 3, 1), (3, 6, 4)], [(0, 1, 3), (1, 6, 0)]])
def test_shared_prefixes(cuda_lib, dim, queries, groups):
    from ekv.runtime.attention import attend

    lens = [max(b for a, b_, b in groups if a <= r < b_) * 16 + 1 + 37 * r + queries for r in range(6)]
    x = make(5, lens, queries=[queries] * 6, dim=dim, groups=groups, q_heads=16, kv_heads=2)
    d = on_device(x)
    group_start = torch.tensor([a for a, _, _ in groups] + [6], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([b for _, _, b in groups], dtype=torch.int32, device="cuda")
    got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], prefix_blocks=prefix,
                 group_start=group_start)
    check(got, x, 0.1, torch.bfloat16)
    wide = widen(x)
    d = on_device(wide)
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], prefix_blocks=prefix,
                 group_start=group_start), wide, 0.1, torch.bfloat16)
    d = on_device(x)
    if len(groups) == 1:
        again = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], prefix_blocks=groups[0][2])
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("dtype, dim, block", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32), (torch.float16, 128, 8),
                                               (torch.bfloat16, 64, 64)])
@pytest.mark.parametrize("rows, q_heads, queries", [(20, 8, 1), (40, 16, 1), (9, 32, 4), (70, 8, 1)])
def test_prefixes_of_many_query_rows(cuda_lib, dtype, dim, block, rows, q_heads, queries):
    """80, 320, 576 and 280 query rows a KV head: one subtile, several, and a last one of few rows; prefixes that CTAs
    share, that one covers, that end inside a tile, and one of two."""
    from ekv.runtime.attention import attend

    for blocks in (1, 3, 1000 // block, 5000 // block):
        x = make(20 + blocks, [blocks * block + 1 + r % 37 + queries for r in range(rows)], queries=[queries] * rows, dim=dim,
                 block=block, dtype=dtype, q_heads=q_heads, groups=[(0, rows, blocks)], width=blocks + -(-50 // block))
        prefix = torch.tensor([blocks], dtype=torch.int32, device="cuda")
        for y in (x, widen(x, 1 << 17)):
            d = on_device(y)
            got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], prefix_blocks=prefix)
            check(got, y, 0.1, dtype)


def test_wide_rows_with_gaps_and_growing_scores(cuda_lib):
    """Query windows of 40 tokens on the wide kernel: bad table entries, an unfinished last block whose rest holds NaN,
    and keys that grow along the row, so that the running maximum is raised again and again."""
    import ekv._lib as L
    from ekv.runtime.attention import attend

    x = make(30, [1000, 700, 129, 40], queries=[40] * 4, q_heads=16, dtype=torch.float16)
    x["cache"][:, 0] *= 0.2
    for r, n in enumerate([1000, 700, 129, 40]):
        for b in range(-(-n // 16)):
            x["cache"][x["table"][r, b], 0] += 0.02 * b * torch.sign(x["query"][int(x["start"][r]), :2]).to(torch.float16)
        if n % 16:
            x["cache"][x["table"][r, n // 16], :, n % 16:] = float("nan")
    ok = np.ones(tuple(x["table"].shape), dtype=bool)
    for r, b, bad in [(0, 2, -1), (0, 40, 10**9), (1, 0, x["cache"].shape[0]), (1, 30, -7)]:
        x["table"][r, b], ok[r, b] = bad, False
    for y in (x, widen(x)):
        d = on_device(y)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], status=status)
        more = np.ones((4, y["table"].shape[1] - ok.shape[1]), dtype=bool)
        check(got, y, 0.1, torch.float16, pool_ok=np.concatenate([ok, more], 1))
        assert int(status) == L.STATUS_BAD_BLOCK_ID


# ---- weights accumulated per token -------------------------------------------------------------------


def run_scored(x, d, scale, scores, slots=None, fresh=None, decay=1.0):
    from ekv.runtime.attention import attend_scored

    dev = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    new = None if fresh is None else torch.tensor(fresh, dtype=torch.int32, device="cuda")
    got = scores.cuda()
    out = attend_scored(d["query"], d["cache"], d["table"], d["lens"], scale, got, query_start=d["start"], slots=dev,
                        fresh=new, decay=decay)
    queries = (x["start"][1:] - x["start"][:-1]).tolist()
    _, _, w = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(), x["lens"].numpy(),
                         scale, x["start"].numpy())
    want = oat.accumulate(scores.numpy(), slots or list(range(len(queries))), x["lens"].tolist(), queries, w, fresh, decay)
    # a weight's exponent is off by at most 3e-5 (the log-sum-exp's and the score's error), the sum by float32 steps
    weight = max(1.0, max(float(v.max()) if v.size else 0.0 for v in w))
    np.testing.assert_allclose(got.cpu().numpy(), want, rtol=1e-6, atol=4e-5 * weight)
    return out


@pytest.mark.parametrize("dtype, dim, block", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32), (torch.bfloat16, 64, 8)])
@pytest.mark.parametrize("queries", [[1] * 6, [3, 1, 0, 9, 2, 40]])
def test_scores_gather_the_weights(cuda_lib, dtype, dim, block, queries):
    lens = [1, 64, 0, 130, 65, 333]
    x = make(6, lens, queries=queries, dim=dim, block=block, dtype=dtype, q_heads=10)
    capacity = x["table"].shape[1] * block
    scores = torch.rand(8, 2, capacity, generator=torch.Generator().manual_seed(1))
    got = run_scored(x, on_device(x), 0.1, scores, slots=[7, 0, 3, -1, 5, 1], decay=0.75)
    check(got, x, 0.1, dtype)


@pytest.mark.parametrize("dtype, dim, block", [(torch.float16, 128, 16), (torch.bfloat16, 64, 64), (torch.float16, 64, 8)])
def test_scores_from_windows_of_many_query_rows(cuda_lib, dtype, dim, block):
    """From 8 to 512 query rows a KV head (two rounds of 256), rows that end inside a tile, a row of one tile, a missing block."""
    lens = [1000, 130, 64, 640, 257]
    x = make(31, lens, queries=[64, 33, 32, 1, 40], dim=dim, block=block, dtype=dtype, q_heads=16)
    capacity = x["table"].shape[1] * block
    scores = torch.rand(5, 2, capacity, generator=torch.Generator().manual_seed(2))
    got = run_scored(x, on_device(x), 0.1, scores, fresh=[1000, 100, 70, 1, 0], decay=0.5)
    check(got, x, 0.1, dtype)


@pytest.mark.parametrize("queries", [1, 20])
def test_scores_of_blocks_that_are_not_there(cuda_lib, queries):
    from ekv.runtime.attention import attend_scored

    x = make(32, [100, 300], queries=[queries] * 2)
    ok = np.ones(tuple(x["table"].shape), dtype=bool)
    x["table"][1, 4], ok[1, 4] = -3, False
    d = on_device(x)
    scores = torch.ones(2, 2, x["table"].shape[1] * 16, device="cuda")
    attend_scored(d["query"], d["cache"], d["table"], d["lens"], 0.1, scores, query_start=d["start"], fresh=d["lens"])
    _, _, w = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(), x["lens"].numpy(), 0.1,
                         x["start"].numpy(), ok)
    for r, n in enumerate([100, 300]):
        np.testing.assert_allclose(scores[r, :, :n].cpu().numpy(), w[r], rtol=1e-6, atol=4e-5 * w[r].max())
    assert torch.all(scores[1, :, 64:80] == 0) and torch.all(scores[0, :, 100:] == 1)


def test_a_prompt_with_no_scores_yet_and_scores_that_are_not_numbers(cuda_lib):
    x = make(7, [200, 50, 100], queries=[16, 5, 1])
    scores = torch.full((3, 2, x["table"].shape[1] * 16), float("nan"))
    scores[2] = 0.25  # row 2 has scores but for its newest token
    run_scored(x, on_device(x), 0.1, scores, fresh=[200, 60, 1])
    run_scored(x, on_device(x), 0.1, torch.full_like(scores, float("nan")), decay=0.0)


def test_slots_given_twice_or_past_the_table_are_left(cuda_lib):
    import ekv._lib as L
    from ekv.runtime.attention import attend, attend_scored

    x = make(8, [40, 50, 60, 70])
    d = on_device(x)
    scores = torch.rand(4, 2, x["table"].shape[1] * 16, device="cuda")
    before = scores.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.tensor([1, 1, 4, 2], dtype=torch.int32, device="cuda")
    got = attend_scored(d["query"], d["cache"], d["table"], d["lens"], 0.1, scores, slots=slots, status=status)
    want = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert int(status) == L.STATUS_BAD_SLOT
    assert torch.equal(scores[[0, 1, 3]], before[[0, 1, 3]]) and not torch.equal(scores[2], before[2])


# ---- faults in the tables, strides, streams, graphs ------------------------------------------------------


def test_bad_table_entries_are_skipped(cuda_lib):
    import ekv._lib as L
    from ekv.runtime.attention import attend

    x = make(9, [100, 48, 16, 500])
    ok = np.ones(tuple(x["table"].shape), dtype=bool)
    for r, b, bad in [(0, 2, -1), (1, 0, 10**9), (2, 0, x["cache"].shape[0]), (3, 31, -7)]:
        x["table"][r, b], ok[r, b] = bad, False
    x["table"][1, 3:] = -5  # behind the row: never read
    d = on_device(x)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, status=status)
    check(got, x, 0.1, torch.bfloat16, pool_ok=ok, start=False)
    assert int(status) == L.STATUS_BAD_BLOCK_ID


def test_lengths_past_the_table_and_queries_outside_the_batch(cuda_lib):
    import ekv._lib as L
    from ekv.runtime.attention import attend

    x = make(10, [64, 64, 64])
    d = on_device(x)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([1000, 64, -5], dtype=torch.int32, device="cuda")
    got = attend(d["query"], d["cache"], d["table"], lens, 0.1, status=status)
    x["lens"] = torch.tensor([64, 64, 0], dtype=torch.int32)
    check(got, x, 0.1, torch.bfloat16, start=False)
    assert int(status) == L.STATUS_LEN_OVER_WIDTH
    status.zero_()
    out, lse = torch.full_like(got[0], 7.0), torch.full_like(got[1], 7.0)
    start = torch.tensor([0, 1, 9, 3], dtype=torch.int32, device="cuda")
    attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=start, out=out, lse=lse, status=status)
    assert int(status) == L.STATUS_BAD_QROW
    assert torch.equal(out[0], got[0][0]) and torch.all(out[1:] == 7.0) and torch.all(lse[1:] == 7.0)


def test_values_behind_a_row_may_be_anything(cuda_lib):
    from ekv.runtime.attention import attend

    x = make(11, [70, 5, 16], dtype=torch.float16)
    for r, n in enumerate([70, 5, 16]):
        if n % 16:
            x["cache"][x["table"][r, n // 16], :, n % 16:] = float("nan")
            x["cache"][x["table"][r, n // 16], 1, 15] = float("inf")
    d = on_device(x)
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.1), x, 0.1, torch.float16, start=False)


def test_keys_that_are_not_numbers_reach_the_output(cuda_lib):
    """A NaN key that a query token sees makes its output NaN, wherever in a tile it stands; other rows keep theirs."""
    from ekv.runtime.attention import attend, attend_scored

    for at in (3, 20, 37, 64, 101, 126, 127, 200):
        x = make(43, [400, 130, 300], queries=[40, 30, 20], q_heads=16, dim=64)
        x["cache"][x["table"][0, at // 16], 0, at % 16, 1] = float("nan")
        for y in (x, widen(x)):
            d = on_device(y)
            out, lse = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"])
            assert torch.all(torch.isnan(out[:40, 8:])) and torch.all(torch.isnan(lse[:40, 8:]))
            assert not torch.any(torch.isnan(out[:40, :8])) and not torch.any(torch.isnan(out[40:]))
        scores = torch.zeros(3, 2, y["table"].shape[1] * 16, device="cuda")
        attend_scored(d["query"], d["cache"], d["table"], d["lens"], 0.1, scores, query_start=d["start"])
        assert torch.all(torch.isnan(scores[0, 1, :360])) and not torch.any(torch.isnan(scores[1:])) and not torch.any(torch.isnan(scores[0, 0]))


def test_strided_tensors_and_a_wider_table(cuda_lib):
    from ekv.runtime.attention import attend

    x = make(12, [90, 33], q_heads=4, kv_heads=2)
    d = on_device(x)
    q = torch.zeros(2, 6, 256, dtype=torch.bfloat16, device="cuda")[:, 1:5, 128:]
    q.copy_(d["query"])
    blocks, _, block, heads, dim = d["cache"].shape
    cache = torch.zeros(blocks, block, heads, 2, dim, dtype=torch.bfloat16, device="cuda").permute(0, 3, 1, 2, 4)
    cache.copy_(d["cache"])
    table = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    table[:, : d["table"].shape[1]] = d["table"]
    out = torch.zeros(2, 4, 256, dtype=torch.bfloat16, device="cuda")[:, :, :128]
    got = attend(q, cache, table, d["lens"], 0.1, out=out)
    want = attend(d["query"], d["cache"], table.contiguous(), d["lens"], 0.1)
    check(got, x, 0.1, torch.bfloat16, start=False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_another_stream_and_a_replayed_graph(cuda_lib):
    from ekv.runtime.attention import attend, attend_scored

    x = make(13, [300, 64, 129, 1000], groups=[(0, 4, 4)])
    d = on_device(x)
    want = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, prefix_blocks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, prefix_blocks=4)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    scores = torch.zeros(4, 2, x["table"].shape[1] * 16, device="cuda")
    lens = d["lens"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = attend(d["query"], d["cache"], d["table"], lens, 0.1, prefix_blocks=4)
        b = attend_scored(d["query"], d["cache"], d["table"], lens, 0.1, scores)
    graph.replay()
    assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    lens.copy_(torch.tensor([299, 70, 1, 0], dtype=torch.int32))  # the same graph, another batch
    scores.zero_()
    graph.replay()
    x["lens"] = lens.cpu()
    check(a, x, 0.1, torch.bfloat16, start=False)
    check(b, x, 0.1, torch.bfloat16, start=False)
    assert abs(float(scores[:3].sum()) - 3 * 8) < 1e-3  # each query head's weights sum to one


def test_two_streams_at_once(cuda_lib):
    from ekv.runtime.attention import attend

    x, y = make(14, [4000] * 8, groups=[(0, 8, 100)]), make(15, [3000, 17] * 4)
    dx, dy = on_device(x), on_device(y)
    want = [attend(dx["query"], dx["cache"], dx["table"], dx["lens"], 0.1, prefix_blocks=100),
            attend(dy["query"], dy["cache"], dy["table"], dy["lens"], 0.1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[0]):
            got.append((0, attend(dx["query"], dx["cache"], dx["table"], dx["lens"], 0.1, prefix_blocks=100)))
        with torch.cuda.stream(streams[1]):
            got.append((1, attend(dy["query"], dy["cache"], dy["table"], dy["lens"], 0.1)))
    torch.cuda.synchronize()
    for k, (out, lse) in got:
        assert torch.equal(out, want[k][0]) and torch.equal(lse, want[k][1])


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_hundreds_of_rows_most_of_them_empty(cuda_lib, grouped, wide):
    """More rows than a CTA has threads, long runs of rows with no tokens or no query, groups of every size."""
    from ekv.runtime.attention import attend

    rng = np.random.default_rng(5)
    lens = [int(n) if rng.random() < 0.4 else 0 for n in rng.integers(1, 200, 420)]
    lens[50:190] = [0] * 140
    lens[300] = 1500
    queries = [int(q) for q in rng.integers(0, 6 if wide else 3, 420)]
    queries[200:280] = [0] * 80
    queries[310] = 70 if wide else 1
    edges = sorted({0, 420, 5, 6, 60, 61, 250, 251, 300, 302, *rng.integers(0, 420, 12).tolist()})
    groups = [(a, b, min(3 + a % 7, min([-(-n // 16) for n in lens[a:b] if n] or [0]))) for a, b in zip(edges, edges[1:])]
    x = make(40, lens, queries=queries, q_heads=64 if wide else 4, kv_heads=2, dim=64, groups=groups if grouped else None)
    x = widen(x, 1 << 18) if wide else x
    d = on_device(x)
    more = {}
    if grouped:
        more = dict(group_start=torch.tensor(edges, dtype=torch.int32, device="cuda"),
                    prefix_blocks=torch.tensor([b for _, _, b in groups], dtype=torch.int32, device="cuda"))
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], **more), x, 0.1, torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("grouped", [False, True])
def test_a_batch_with_nothing_in_its_cache(cuda_lib, rows, grouped):
    from ekv.runtime.attention import attend

    x = make(44, [0] * rows, queries=[2] * rows, width=40)
    d = on_device(x)
    out, lse = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], prefix_blocks=3 if grouped else None)
    assert torch.all(out == 0) and torch.all(lse == float("-inf"))


def test_scores_of_hundreds_of_rows(cuda_lib):
    rng = np.random.default_rng(6)
    lens = [int(n) if rng.random() < 0.5 else 0 for n in rng.integers(1, 150, 300)]
    for top in (2, 60):
        x = make(41, lens, queries=[int(q) for q in rng.integers(0, top, 300)], dim=64)
        scores = torch.rand(300, 2, x["table"].shape[1] * 16, generator=torch.Generator().manual_seed(3))
        run_scored(x, on_device(x), 0.1, scores, slots=rng.permutation(300).tolist(), decay=0.5)


def test_a_row_that_is_shorter_than_its_groups_prefix(cuda_lib):
    from ekv.runtime.attention import attend

    x = make(16, [30, 0, 200, 97], groups=[(0, 4, 6)])
    d = on_device(x)
    check(attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, prefix_blocks=6), x, 0.1, torch.bfloat16, start=False)


def test_a_view_of_a_row_attends_to_its_blocks_alone(cuda_lib):
    from ekv.runtime.attention import attend
    from ekv.runtime.block_view import compact_block_table

    x = make(17, [160, 90], block=16)
    keep = torch.tensor(np.random.default_rng(0).random((2, x["table"].shape[1])) < 0.5)
    d = on_device(x)
    view, view_lens = compact_block_table(d["table"], d["lens"], keep.cuda(), 16)
    got = attend(d["query"], d["cache"], view, view_lens, 0.1)
    x["table"], x["lens"] = view.cpu(), view_lens.cpu()
    check(got, x, 0.1, torch.bfloat16, start=False)


# ---- queries and keys that are not numbers ------------------------------------------------------------------


def nan_batch(kind):
    """A batch for each way that parts of a row join: lengths, queries and head counts that pick it, and the call's arguments."""
    shapes = {
        "a CTA an item": dict(lens=[1, 17, 333]),
        "tiles dealt": dict(lens=[1, 17, 333], width=40),
        "split over CTAs": dict(lens=[1, 17, 9001]),
        "24 query rows a head": dict(lens=[1, 17, 333], q_heads=48),
        "48 query rows a head": dict(lens=[1, 17, 9001], q_heads=96),
        "several query tokens": dict(lens=[1, 19, 1025], queries=[3, 3, 3]),
        "many query rows": dict(lens=[1, 41, 3001], queries=[40, 40, 40], q_heads=16),
        "one subtile of many": dict(lens=[1, 17, 3001], queries=[15, 10, 12], q_heads=16),
        "behind a prefix": dict(lens=[65, 81, 700], groups=[(0, 3, 4)]),
        "many behind a prefix": dict(lens=[1985, 2001, 2600], queries=[30, 30, 30], q_heads=16, groups=[(0, 3, 120)]),
    }
    x = make(50, **shapes[kind])
    if "many" in kind:
        x = widen(x, 1 << 17)  # the kernel for many query rows
    prefix = shapes[kind].get("groups", [(0, 0, None)])[0][2]
    return x, {} if prefix is None else dict(prefix_blocks=prefix)


NAN_KINDS = ["a CTA an item", "tiles dealt", "split over CTAs", "24 query rows a head", "48 query rows a head",
             "several query tokens", "many query rows", "one subtile of many", "behind a prefix", "many behind a prefix"]


def put_nan(x, fault):
    start, lens, table, cache = x["start"].tolist(), x["lens"].tolist(), x["table"], x["cache"]
    for r, n in enumerate(lens):
        if fault == "queries":  # a head of each row's newest query token, and in row 2 another's of its oldest
            x["query"][start[r + 1] - 1, 5, 7] = float("nan")
            x["query"][start[2], 0, 0] = float("nan")
        elif fault == "newest keys":
            cache[table[r, (n - 1) // 16], 0, (n - 1) % 16, 1, 3] = float("nan")
        else:  # every key of 128 tokens, or of what the row has before its newest one
            for t in range(max(0, n - 150), max(0, n - 22) if n > 150 else n - 1):
                cache[table[r, t // 16], 0, t % 16, 0, 0] = float("nan")


def same_nan(got, want):
    np.testing.assert_array_equal(np.isnan(got.float().cpu().numpy()), np.isnan(want))


@pytest.mark.parametrize("fault", ["queries", "newest keys", "a run of keys"])
@pytest.mark.parametrize("kind", NAN_KINDS)
def test_nan_reaches_every_output_that_it_is_part_of_and_no_other(cuda_lib, kind, fault):
    from ekv.runtime.attention import attend

    x, more = nan_batch(kind)
    put_nan(x, fault)
    d = on_device(x)
    got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], **more)
    out, lse, _ = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(), x["lens"].numpy(),
                             0.1, x["start"].numpy())
    assert np.isnan(lse).any() and not np.isnan(lse).all()
    same_nan(got[0], out)
    same_nan(got[1], lse)
    check(got, x, 0.1, torch.bfloat16)


@pytest.mark.parametrize("fault", ["queries", "newest keys", "a run of keys"])
@pytest.mark.parametrize("kind", NAN_KINDS[:8])
def test_nan_reaches_every_score_that_it_is_part_of_and_no_other(cuda_lib, kind, fault):
    from ekv.runtime.attention import attend_scored

    x, _ = nan_batch(kind)
    put_nan(x, fault)
    ok = np.ones(tuple(x["table"].shape), dtype=bool)
    if kind != "a CTA an item":
        x["table"][2, 3], ok[2, 3] = -1, False  # a block that is not there gives its tokens no weight
    d = on_device(x)
    used = max(x["lens"].tolist())
    scores = torch.full((3, 2, x["table"].shape[1] * 16), 0.5, device="cuda")
    attend_scored(d["query"], d["cache"], d["table"], d["lens"], 0.1, scores, query_start=d["start"])
    _, lse, w = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(), x["lens"].numpy(), 0.1,
                           x["start"].numpy(), ok)
    queries = (x["start"][1:] - x["start"][:-1]).tolist()
    want = oat.accumulate(np.full((3, 2, used), 0.5), [0, 1, 2], x["lens"].tolist(), queries, w)
    assert np.isnan(want).any() and not np.isnan(want).all()
    # as for weights that are all numbers: 4e-5 of the largest a token can have, one from every query row
    most = max(queries) * x["query"].shape[1] / 2
    np.testing.assert_allclose(scores[..., :used].cpu().numpy(), want, rtol=1e-6, atol=4e-5 * most)
    assert torch.all(scores[..., used:] == 0.5)


def test_scores_in_a_table_too_wide_for_the_logits(cuda_lib):
    """Two rows of one query token in a table of 2^23 and more positions: the weights come from the keys again."""
    x = make(51, [700, 33], q_heads=16, kv_heads=1, dim=64)
    x = widen(x, (1 << 23) + 64)
    scores = torch.full((2, 1, x["table"].shape[1] * 16), 0.25)
    from ekv.runtime.attention import attend_scored

    d, got = on_device(x), scores.cuda()
    check(attend_scored(d["query"], d["cache"], d["table"], d["lens"], 0.1, got), x, 0.1, torch.bfloat16)
    _, _, w = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(), x["lens"].numpy(), 0.1)
    want = oat.accumulate(np.full((2, 1, 700), 0.25), [0, 1], [700, 33], [1, 1], w)
    np.testing.assert_allclose(got[..., :700].cpu().numpy(), want, rtol=1e-6, atol=4e-5 * 16)
    assert torch.all(got[..., 700:] == 0.25)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("queries, lens", [([1] * 5, [60, 0, 200, 97, 1]), ([3, 1, 0, 12, 2], [60, 5, 900, 640, 96]),
                                           ([40] * 5, [90, 20, 700, 130, 96])])
def test_a_row_shorter_than_its_groups_prefix_sees_nothing_of_the_others(cuda_lib, queries, lens, wide):
    """Shared blocks whose keys and values are not numbers behind the shorter rows: the longer rows hold them, the others do not."""
    from ekv.runtime.attention import attend

    x = make(52, lens, queries=queries, q_heads=16, groups=[(0, 5, 6)], width=60)
    for t in range(61, 96):
        x["cache"][x["table"][0, t // 16], 1, t % 16] = float("nan") if t % 2 else float("inf")
        x["cache"][x["table"][0, t // 16], 0, t % 16, 1] = float("nan") if t > 92 else 1.0
    x = widen(x, 1 << 17) if wide else x
    d = on_device(x)
    got = attend(d["query"], d["cache"], d["table"], d["lens"], 0.1, query_start=d["start"], prefix_blocks=6)
    want, lse, _ = oat.attend(x["query"].float().numpy(), x["cache"].float().numpy(), x["table"].numpy(), x["lens"].numpy(), 0.1,
                              x["start"].numpy())
    u = torch.finfo(torch.bfloat16).eps / 2
    start = x["start"].tolist()
    for r in [r for r in range(5) if lens[r] <= 61]:
        a, b = start[r], start[r + 1]
        o, e = got[0][a:b].double().cpu().numpy(), got[1][a:b].double().cpu().numpy()
        biggest = 6.0  # no value of these rows is larger
        np.testing.assert_allclose(e, lse[a:b], rtol=0, atol=3e-5)
        assert np.all(np.abs(o - want[a:b]) <= 1.05 * u * (np.abs(want[a:b]) + 1.01 * biggest) + 3e-5 * biggest)


@pytest.mark.parametrize("kind", NAN_KINDS)
def test_an_output_over_the_query_itself(cuda_lib, kind):
    from ekv.runtime.attention import attend, attend_scored

    x, more = nan_batch(kind)
    d = on_device(x)
    args = (d["cache"], d["table"], d["lens"], 0.1)
    want = attend(d["query"], *args, query_start=d["start"], **more)
    query = d["query"].clone()
    got = attend(query, *args, query_start=d["start"], out=query, **more)
    assert got[0] is query and torch.equal(query, want[0]) and torch.equal(got[1], want[1])
    if more:
        return
    scores = [torch.zeros(3, 2, x["table"].shape[1] * 16, device="cuda") for _ in range(2)]
    attend_scored(d["query"], *args, scores[0], query_start=d["start"])
    query = d["query"].clone()
    if "many" in kind or "query rows a head" in kind:
        with pytest.raises(ValueError, match="share no memory"):
            attend_scored(query, *args, scores[1], query_start=d["start"], out=query)
        assert torch.equal(query, d["query"]) and not scores[1].any()
        # the other half of each token's row is memory of its own
        both = torch.zeros(len(query), 2, *query.shape[1:], dtype=query.dtype, device="cuda")
        both[:, 0] = query
        attend_scored(both[:, 0], *args, scores[1], query_start=d["start"], out=both[:, 1])
        assert torch.equal(both[:, 1], want[0]) and torch.equal(both[:, 0], query)
    else:
        attend_scored(query, *args, scores[1], query_start=d["start"], out=query)
        assert torch.equal(query, want[0])
    assert torch.equal(scores[0], scores[1])


@pytest.mark.parametrize("grouped", [False, True])
def test_rows_that_claim_the_same_query_tokens_over_and_over(cuda_lib, grouped):
    """A query_start that goes up and down gives every second row all 4096 tokens, 2^31 tiles and more in all, which the sizes
    of a call that ascends cannot reach: nothing is attended to, the status says so, and the next call is as ever."""
    import ekv._lib as L
    from ekv.runtime.attention import attend

    rows, tokens, width = 2048, 4096, 4107
    assert rows // 2 * (tokens * 8 // 16) * (65700 // 64) > 2**31
    gen = torch.Generator().manual_seed(53)
    cache = torch.randn(2, 2, 16, 1, 128, generator=gen).bfloat16().cuda()
    query = torch.randn(tokens, 8, 128, generator=gen).bfloat16().cuda()
    table = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
    start = torch.tensor([tokens * (r % 2) for r in range(rows + 1)], dtype=torch.int32, device="cuda")
    more = dict(prefix_blocks=torch.zeros(1, dtype=torch.int32, device="cuda")) if grouped else {}
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lens = torch.full((rows,), 65700, dtype=torch.int32, device="cuda")
    out, lse = attend(query, cache, table, lens, 0.1, query_start=start, status=status, **more)
    assert int(status) == L.STATUS_BAD_QROW
    assert not out.any() and torch.all(lse == float("-inf"))
    ascending = torch.arange(0, 2 * rows + 1, 2, dtype=torch.int32, device="cuda")
    short = torch.full((rows,), 9, dtype=torch.int32, device="cuda")
    status.zero_()
    out, lse = attend(query, cache, table, short, 0.1, query_start=ascending, status=status, **more)
    want = oat.attend(query[:6].float().cpu().numpy(), cache.float().cpu().numpy(), np.zeros((3, 1), dtype=int), np.array([9] * 3), 0.1,
                      np.array([0, 2, 4, 6]))
    assert int(status) == 0
    np.testing.assert_allclose(lse[:6].cpu().numpy(), want[1], rtol=0, atol=3e-5)
    u = torch.finfo(torch.bfloat16).eps / 2
    assert np.all(np.abs(out[:6].double().cpu().numpy() - want[0]) <= 1.05 * u * (np.abs(want[0]) + 1.01 * 6) + 3e-5 * 6)
