"""The refusals of the attention and eviction entry points: bad arguments raise, or return the documented code,
before anything touches a device. CPU only."""

from __future__ import annotations

import ctypes

import pytest
import torch

import ekv._lib as L

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    import ekv.build

    ekv.build.build()
    return L.load()


def attend_args(**over):
    args = dict(q=FAKE, qs0=1024, qs1=128, kv=FAKE, s0=8192, s1=4096, s2=256, s3=128, pool=64, table=FAKE, ts=8, lens=FAKE,
                start=None, tokens=4, rows=4, width=8, bs=16, qh=8, kvh=2, D=128, dtype=L.DTYPE_BF16, scale=0.1, groups=0,
                members=None, prefix=None, common=0, out=FAKE, os0=1024, os1=128, lse=FAKE, ws=FAKE, ws_bytes=1 << 40,
                status=None, stream=None)
    args.update(over)
    return list(args.values())


SHARED = [
    (dict(q=None), L.EINVAL),
    (dict(kv=None), L.EINVAL),
    (dict(out=None), L.EINVAL),
    (dict(rows=0, tokens=0), L.EINVAL),
    (dict(tokens=5), L.EINVAL),  # five tokens for four rows and no query_start
    (dict(qh=7), L.EINVAL),
    (dict(D=96), L.ENOTSUP),
    (dict(bs=12), L.ENOTSUP),
    (dict(bs=128), L.ENOTSUP),
    (dict(dtype=7), L.EINVAL),
    (dict(scale=0.0), L.EINVAL),
    (dict(scale=-0.1), L.EINVAL),
    (dict(scale=float("nan")), L.EINVAL),
    (dict(scale=float("inf")), L.EINVAL),
    (dict(ts=7), L.EINVAL),
    (dict(q=ctypes.c_void_p(0x1002)), L.EINVAL),
    (dict(qs1=100), L.EINVAL),
    (dict(kv=ctypes.c_void_p(0x1008)), L.EINVAL),
    (dict(s2=260), L.EINVAL),
    (dict(s3=0), L.EINVAL),
    (dict(os0=1001), L.EINVAL),
    (dict(pool=1 << 31), L.ENOTSUP),
    (dict(rows=2049, tokens=2049), L.ENOTSUP),
    (dict(width=1 << 28, ts=1 << 28), L.ENOTSUP),
    (dict(ws=None), L.ERANGE),
    (dict(ws_bytes=100), L.ERANGE),
    (dict(ws=ctypes.c_void_p(0x1010)), L.ERANGE),
]


@pytest.mark.parametrize("over, code", SHARED + [
    (dict(groups=5), L.EINVAL),
    (dict(groups=-1), L.EINVAL),
    (dict(groups=2), L.EINVAL),  # two groups and nothing that says which rows
    (dict(groups=1, common=-1), L.EINVAL),
])
def test_attend_refuses(lib, over, code):
    assert lib.ekv_attend(*attend_args(**over)) == code
    assert lib.ekv_last_error_string()


def scored_args(**over):
    # a table that holds any batch, unless the case is about the table
    more = dict(scores=FAKE, ss0=1 << 41, ss1=1 << 40, n_slots=4096, slots=None, fresh=None, decay=1.0)
    more.update({k: v for k, v in over.items() if k in more})
    base = attend_args(**{k: v for k, v in over.items() if k not in more})
    return base[:22] + list(more.values()) + base[26:]


@pytest.mark.parametrize("over, code", SHARED + [
    (dict(scores=None), L.EINVAL),
    (dict(lse=None), L.EINVAL),
    (dict(ss1=127), L.EINVAL),  # a head's scores do not hold width * block_size tokens
    (dict(ss0=100, ss1=128), L.EINVAL),
    (dict(n_slots=0), L.EINVAL),
    (dict(n_slots=3), L.EINVAL),
    (dict(decay=1.5), L.EINVAL),
    (dict(decay=-0.5), L.EINVAL),
    (dict(decay=float("nan")), L.EINVAL),
])
def test_attend_scored_refuses(lib, over, code):
    assert lib.ekv_attend_scored(*scored_args(**over)) == code


@pytest.mark.parametrize("over, code", [
    (dict(scores=None), L.EINVAL),
    (dict(kept=None), L.EINVAL),
    (dict(rows=0), L.EINVAL),
    (dict(capacity=0), L.EINVAL),
    (dict(n_slots=3), L.EINVAL),
    (dict(first=-1), L.EINVAL),
    (dict(recent=-1), L.EINVAL),
    (dict(s1=99), L.EINVAL),
    (dict(k1=99), L.EINVAL),
    (dict(capacity=2**31 - 1, s1=2**31, s0=2**33, k1=2**31, k0=2**33), L.ENOTSUP),
])
def test_select_tokens_refuses(lib, over, code):
    args = dict(scores=FAKE, s0=200, s1=100, n_slots=4, capacity=100, slots=None, lens=FAKE, keep=None, keep_all=10, first=0,
                recent=0, rows=4, heads=2, kept=FAKE, k0=200, k1=100, new=FAKE, status=None, stream=None)
    args.update(over)
    assert lib.ekv_select_tokens(*args.values()) == code


@pytest.mark.parametrize("over, code", [
    (dict(kv=None), L.EINVAL),
    (dict(new=None), L.EINVAL),
    (dict(rows=0), L.EINVAL),
    (dict(columns=0), L.EINVAL),
    (dict(head_bytes=200), L.ENOTSUP),
    (dict(head_bytes=1040), L.ENOTSUP),
    (dict(s2=520), L.EINVAL),
    (dict(kv=ctypes.c_void_p(0x1004)), L.EINVAL),
    (dict(ts=7), L.EINVAL),
    (dict(k1=50), L.EINVAL),
    (dict(first=-1), L.EINVAL),
    (dict(scores=FAKE, ss0=256, ss1=127, n_slots=4), L.EINVAL),
    (dict(scores=FAKE, ss0=256, ss1=128, n_slots=3), L.EINVAL),
    (dict(width=1 << 28, ts=1 << 28), L.ENOTSUP),
    (dict(ws=None), L.ERANGE),
    (dict(ws_bytes=100), L.ERANGE),
])
def test_compact_tokens_refuses(lib, over, code):
    args = dict(kv=FAKE, s0=16384, s1=8192, s2=512, s3=256, pool=64, head_bytes=256, table=FAKE, ts=8, lens=FAKE, rows=4,
                width=8, heads=2, bs=16, kept=FAKE, k0=256, k1=128, columns=128, new=FAKE, first=0, scores=None, ss0=0, ss1=0,
                n_slots=0, slots=None, ws=FAKE, ws_bytes=1 << 30, status=None, stream=None)
    args.update(over)
    assert lib.ekv_compact_tokens(*args.values()) == code


def test_workspace_sizes(lib):
    assert lib.ekv_attend_workspace_bytes(0, 1, 0, 8, 2, 128) == 0
    assert lib.ekv_attend_workspace_bytes(4, 4, 0, 7, 2, 128) == 0
    alone, grouped = (lib.ekv_attend_workspace_bytes(4, 4, g, 8, 2, 128) for g in (0, 2))
    assert 0 < alone < grouped and alone % 256 == 0 and grouped % 256 == 0
    assert lib.ekv_compact_tokens_workspace_bytes(4, 2, 0) == 0
    assert lib.ekv_compact_tokens_workspace_bytes(4, 2, 1000) >= 4 * (1000 + 4 + 8)


def test_the_python_calls_refuse_what_is_not_on_a_device_or_does_not_fit():
    from ekv.runtime.attention import attend, attend_scored
    from ekv.runtime.eviction import compact_tokens, select_tokens

    query, cache = torch.zeros(2, 8, 128, dtype=torch.bfloat16), torch.zeros(9, 2, 16, 2, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        attend(query, cache, table, lens, 0.1)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        attend(query.float(), cache.float(), table, lens, 0.1)
    with pytest.raises(ValueError, match="KV cache"):
        attend(query, cache[:, 0], table, lens, 0.1)
    with pytest.raises(ValueError, match="query"):
        attend(query[..., :64], cache, table, lens, 0.1)
    with pytest.raises(ValueError, match="int32"):
        attend(query, cache, table.long(), lens, 0.1)
    with pytest.raises(ValueError, match="length per row"):
        attend(query, cache, table, lens[:1], 0.1)
    with pytest.raises(ValueError, match="contiguous"):
        attend(query, cache, table.t().contiguous().t(), lens, 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        attend_scored(query, cache, table, lens, 0.1, torch.zeros(2, 2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        select_tokens(torch.zeros(2, 2, 64), lens, 10)
    with pytest.raises(ValueError, match="float32"):
        select_tokens(torch.zeros(2, 2, 64, dtype=torch.float16), lens, 10)
    with pytest.raises(ValueError, match="CUDA"):
        compact_tokens(cache, table, lens, torch.zeros(2, 2, 64, dtype=torch.int32), lens)
    with pytest.raises(ValueError, match="KV cache"):
        compact_tokens(cache[:, 0], table, lens, torch.zeros(2, 2, 64, dtype=torch.int32), lens)


def test_compact_tokens_lens_refuses_what_compact_tokens_refuses_and_shared_memory(lib):
    args = dict(kv=FAKE, s0=16384, s1=8192, s2=512, s3=256, pool=64, head_bytes=256, table=FAKE, ts=8, lens=FAKE, rows=4,
                width=8, heads=2, bs=16, kept=FAKE, k0=256, k1=128, columns=128, new=ctypes.c_void_p(0x2000), first=0, scores=None,
                ss0=0, ss1=0, n_slots=0, slots=None, result=ctypes.c_void_p(0x3000), ws=FAKE, ws_bytes=1 << 30, status=None, stream=None)
    for over, code in [(dict(kv=None), L.EINVAL), (dict(rows=0), L.EINVAL), (dict(ws_bytes=100), L.ERANGE),
                       (dict(result=FAKE), L.EINVAL),                      # the lengths themselves
                       (dict(result=ctypes.c_void_p(0x1000 + 12)), L.EINVAL),  # from their last entry on
                       (dict(result=ctypes.c_void_p(0x2000 - 12)), L.EINVAL),  # up to the new lengths' first
                       (dict(result=ctypes.c_void_p(0x1000 + 16), ws_bytes=0), L.ERANGE)]:  # right behind them: the next check
        assert lib.ekv_compact_tokens_lens(*{**args, **over}.values()) == code


@pytest.mark.parametrize("wrong", [0.5, 512.0, "3", None])
def test_counts_have_to_be_whole_numbers(wrong):
    """A fraction is refused before anything else is looked at: cut to a whole number, a `keep` of one half would keep nothing."""
    from ekv.runtime.attention import attend
    from ekv.runtime.eviction import compact_tokens, select_tokens

    scores, lens = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    cache, table = torch.zeros(9, 2, 16, 2, 128, dtype=torch.bfloat16), torch.zeros(2, 4, dtype=torch.int32)
    kept = torch.zeros(2, 2, 64, dtype=torch.int32)
    calls = [lambda: select_tokens(scores, lens, wrong), lambda: select_tokens(scores, lens, 4, first_tokens=wrong),
             lambda: select_tokens(scores, lens, 4, recent_tokens=wrong),
             lambda: compact_tokens(cache, table, lens, kept, lens, first_tokens=wrong)]
    if wrong is not None:  # which means that no prefix is shared
        calls.append(lambda: attend(torch.zeros(2, 8, 128, dtype=torch.bfloat16), cache, table, lens, 0.1, prefix_blocks=wrong))
    for call in calls:
        with pytest.raises(ValueError, match="whole number"):
            call()


def test_attend_scored_refuses_an_output_over_queries_that_it_reads_again(lib):
    """256 query tokens of four heads' groups: 64 query rows a row and KV head. Apart as a whole or by columns is accepted, as far
    as this machine without a device goes."""
    at = lambda n: ctypes.c_void_p(0x100000 + n)
    size = 256 * 1024 * 2
    shape = dict(tokens=256, rows=4, start=FAKE, q=at(0))
    for over in (dict(out=at(0)), dict(out=at(256)), dict(out=at(size - 2048)), dict(out=at(2048 - size)),
                 dict(out=at(2048), os0=2048), dict(qs0=2048, os0=2048, out=at(1024)), dict(qs0=2048, os0=2048, qs1=256, os1=256, out=at(128)),
                 dict(qs0=0, out=at(512))):
        assert lib.ekv_attend_scored(*scored_args(**{**shape, **over})) == L.EINVAL and b"share" in lib.ekv_last_error_string(), over
    for over in (dict(out=at(size)), dict(out=at(-size)), dict(qs0=2048, os0=2048, out=at(2048)),  # a row's other half
                 dict(qs0=2048, os0=2048, qs1=256, os1=256, out=at(256))):  # a head's other half
        assert lib.ekv_attend_scored(*scored_args(**{**shape, **over})) != L.EINVAL, over
    # with one query token a row its logits are kept
    assert lib.ekv_attend_scored(*scored_args()) != L.EINVAL
    assert lib.ekv_attend(*attend_args(**{**shape, "out": at(0)})) != L.EINVAL
