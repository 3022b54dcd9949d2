"""Eviction from the paged KV cache by accumulated attention weight, on the sm_100a kernels.

A view (``block_view``) leaves blocks unread; eviction frees them. ``attention.attend_scored`` adds up the
attention weight each cached token receives; ``select_tokens`` decides, per row and KV head, which tokens a bounded
cache keeps (the row's first and newest ones, and the best of the others), and ``compact_tokens`` moves them, with
their scores, to the front of the row's blocks, in place and in order. The row's blocks behind its new length are
then the engine's to reuse. Keys carry their rotation when they are cached, so a moved token attends as before.
"""

from __future__ import annotations

import functools

import torch

from .. import _lib
from .attention import _count, _index, _status, check_scores


@functools.lru_cache(maxsize=256)
def _workspace(*sizes: int) -> int:
    return _lib.load().ekv_compact_tokens_workspace_bytes(*sizes)


def select_tokens(
    scores: torch.Tensor,
    lens: torch.Tensor,
    keep: torch.Tensor | int,
    *,
    first_tokens: int = 0,
    recent_tokens: int = 0,
    slots: torch.Tensor | None = None,
    kept: torch.Tensor | None = None,
    new_lens: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The tokens each row and KV head keeps: ``(kept, new_lens)``.

    ``scores`` is the float32 [slots, heads, capacity] table of ``attend_scored`` and ``slots`` its row map, ``lens``
    int32 [rows], ``keep`` how many tokens a row keeps: an int, or int32 [rows], where a negative count keeps the row
    whole, as a quota of -1 does. A row of more tokens keeps its first ``first_tokens`` and newest
    ``recent_tokens`` whatever they score (and so at least that many), and the best of the others; NaN ranks as -inf,
    equal scores go to the older token. ``kept`` int32 [rows, heads, capacity] lists the kept positions in ascending
    order, then -1; ``new_lens`` int32 [rows] counts them.
    """
    first_tokens, recent_tokens = _count("first_tokens", first_tokens), _count("recent_tokens", recent_tokens)
    count = 0 if isinstance(keep, torch.Tensor) else _count("keep", keep)
    device = scores.device
    if scores.dim() != 3:
        raise ValueError(f"scores must be a float32 [slots, heads, tokens] tensor, got {tuple(scores.shape)}")
    n_slots, heads, capacity = scores.shape
    if device.type != "cuda" and scores.dtype is torch.float32:
        raise ValueError("the selection runs on the device: scores must be a CUDA tensor")
    stride = check_scores(scores, heads, 1, device)
    if lens.dim() != 1:
        raise ValueError("lens must be [rows]")
    rows = lens.shape[0]
    length = _index("lens", lens, rows, device)
    places = _index("slots", slots, rows, device)
    if slots is None and n_slots < rows:
        raise ValueError(f"{n_slots} score slots for {rows} rows")
    if first_tokens < 0 or recent_tokens < 0:
        raise ValueError("first_tokens and recent_tokens must not be negative")
    counts = _index("keep", keep, rows, device) if isinstance(keep, torch.Tensor) else None
    if kept is None:
        kept = scores.new_empty((rows, heads, capacity), dtype=torch.int32)
    elif kept.shape != (rows, heads, capacity) or kept.dtype is not torch.int32 or kept.device != device or kept.stride(2) != 1:
        raise ValueError(f"kept must be an int32 [{rows}, {heads}, {capacity}] tensor on {device}")
    if new_lens is None:
        new_lens = lens.new_empty(rows)
    new = _index("new_lens", new_lens, rows, device)
    word = _status(status, device)
    if rows == 0:
        return kept, new_lens
    kept_stride = kept.stride()
    with _lib.on_device(device) as stream:
        rc = _lib.load().ekv_select_tokens(
            scores.data_ptr(), stride[0], stride[1], n_slots, capacity, places, length, counts,
            max(min(count, 0x7FFFFFFF), -1), min(first_tokens, capacity), min(recent_tokens, capacity), rows, heads,
            kept.data_ptr(), kept_stride[0], kept_stride[1], new, word, stream,
        )
    _lib.check(rc, "ekv_select_tokens")
    return kept, new_lens


def compact_tokens(
    kv_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    kept: torch.Tensor,
    new_lens: torch.Tensor,
    *,
    first_tokens: int = 0,
    scores: torch.Tensor | None = None,
    slots: torch.Tensor | None = None,
    result_lens: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> None:
    """Move each row's kept tokens to the front of its blocks, in place.

    ``kv_cache`` is [blocks, 2, block, heads, dim] of any type, ``table`` int32 [rows, width], ``lens`` the rows'
    tokens before and ``new_lens`` after (int32 [rows]; a row that does not shrink is not touched), ``kept`` int32
    [rows, heads, >= tokens] as ``select_tokens`` lists it: ascending, and the identity on the first ``first_tokens``.
    With ``scores`` (``attend_scored``'s table, and its ``slots``) each token's score moves along.

    Blocks wholly among the first ``first_tokens`` tokens may be shared between rows; every other block of a row that
    shrinks must be its own. A row whose lists, blocks or slot break this is left as it was, with the reason in
    ``status`` (EKV_STATUS_BAD_LIST, _BLOCK_SHARED, _BAD_BLOCK_ID, _BAD_SLOT), which speaks for the whole batch.
    ``result_lens`` (int32 [rows], memory of its own) receives the tokens each row holds afterwards: ``new_lens[r]``
    where the row was moved, ``lens[r]`` where it was left. These are the rows' lengths from here on; only the blocks
    behind them are free.
    """
    first_tokens = _count("first_tokens", first_tokens)
    if kv_cache.dim() != 5 or kv_cache.shape[1] != 2 or kv_cache.stride(4) != 1:
        raise ValueError(f"expected a KV cache [blocks, 2, block, heads, dim] with contiguous heads, got {tuple(kv_cache.shape)}")
    device = kv_cache.device
    if device.type != "cuda":
        raise ValueError("the cache is compacted on the device: it must be a CUDA tensor")
    blocks, _, block_size, heads, dim = kv_cache.shape
    if table.dtype is not torch.int32 or table.dim() != 2 or table.device != device or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"the block table must be an int32 [rows, width] tensor on {device} with contiguous rows")
    rows, width = table.shape
    length = _index("lens", lens, rows, device)
    new = _index("new_lens", new_lens, rows, device)
    places = _index("slots", slots, rows, device)
    if kept.dtype is not torch.int32 or kept.dim() != 3 or kept.shape[:2] != (rows, heads) or kept.device != device or kept.stride(2) != 1:
        raise ValueError(f"kept must be an int32 [{rows}, {heads}, tokens] tensor on {device}")
    score_stride = (0, 0)
    if scores is not None:
        score_stride = check_scores(scores, heads, width * block_size, device)
        if slots is None and scores.shape[0] < rows:
            raise ValueError(f"{scores.shape[0]} score slots for {rows} rows")
    elif slots is not None:
        raise ValueError("slots map rows to scores: there are none")
    if first_tokens < 0:
        raise ValueError("first_tokens must not be negative")
    after = _index("result_lens", result_lens, rows, device)
    word = _status(status, device)
    if rows == 0:
        return
    lib = _lib.load()
    size = _workspace(rows, heads, blocks)
    item = kv_cache.element_size()
    s_block, s_part, s_pos, s_head, _ = kv_cache.stride()
    kept_stride = kept.stride()
    with _lib.on_device(device) as stream:
        workspace = kv_cache.new_empty(size, dtype=torch.uint8)
        rc = lib.ekv_compact_tokens_lens(
            kv_cache.data_ptr(), s_block * item, s_part * item, s_pos * item, s_head * item, blocks, dim * item,
            table.data_ptr(), table.stride(0), length, rows, width, heads, block_size, kept.data_ptr(), kept_stride[0],
            kept_stride[1], kept.shape[2], new, min(first_tokens, width * block_size), _lib.ptr(scores),
            score_stride[0], score_stride[1], len(scores) if scores is not None else 0, places, after,
            workspace.data_ptr(), size, word, stream,
        )
    _lib.check(rc, "ekv_compact_tokens")
