"""Attention over the paged KV cache through a block table, on the sm_100a kernels.

The audit kernel (``audit_kernel``) measures what each block of a row draws and the view (``block_view``)
drops blocks from the row; ``attend`` is the attention that reads the row, whole or viewed: ``table`` and
``lens`` are an engine's block table and lengths or the buffers of a ``DecodeView``. The reference leaves this
step to its engine's backend.

Rows that begin with the same blocks (samples of one prompt, requests under one system prompt) are read
once: ``prefix_blocks`` says how many blocks each group of rows shares, and the queries of all the group's
rows meet the shared keys and values together. The kernels take their work from the lengths on the device, so
a call is the same for every batch of its shape and a CUDA graph can capture it.

``attend_scored`` also adds up, per KV head, the attention weight each cached token receives from step to step:
the score by which ``eviction`` decides which tokens of a bounded cache to keep.
"""

from __future__ import annotations

import functools
import operator

import torch

from .. import _lib

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


@functools.lru_cache(maxsize=256)
def _workspace(*sizes: int) -> int:
    return _lib.load().ekv_attend_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=256)
def _scored_workspace(*sizes: int) -> int:
    return _lib.load().ekv_attend_scored_workspace_bytes(*sizes)


def _index(name: str, t: torch.Tensor | None, size: int, device: torch.device) -> int | None:
    """The address of an int32 index array of at least ``size`` entries on the call's device."""
    if t is None:
        return None
    if (t.dtype is not torch.int32 or t.dim() != 1 or len(t) < size or t.get_device() != device.index
            or (size > 1 and t.stride(0) != 1)):
        raise ValueError(f"{name} must be a contiguous int32 tensor of at least {size} entries on {device}")
    return t.data_ptr()


def _count(name: str, value) -> int:
    """A count of any whole-number type; a fraction is refused, not cut to one."""
    try:
        return operator.index(value)
    except TypeError:
        raise ValueError(f"{name} must be a whole number, got {value!r}") from None


def _batch(query: torch.Tensor, kv_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor) -> tuple:
    """What a call passes on of its batch, checked: each tensor's shape and strides are asked for once."""
    q_shape, kv_shape, table_shape = query.shape, kv_cache.shape, table.shape
    if len(kv_shape) != 5 or kv_shape[1] != 2:
        raise ValueError(f"expected a KV cache [blocks, 2, block, heads, dim], got {tuple(kv_shape)}")
    if len(q_shape) != 3 or q_shape[2] != kv_shape[4]:
        raise ValueError(f"expected a query [tokens, heads, {kv_shape[4]}], got {tuple(q_shape)}")
    dtype = _DTYPES.get(query.dtype)
    if dtype is None or kv_cache.dtype is not query.dtype:
        raise ValueError(f"query and cache must both be float16 or bfloat16, got {query.dtype}, {kv_cache.dtype}")
    q_stride, kv_stride = query.stride(), kv_cache.stride()
    if q_stride[2] != 1 or kv_stride[4] != 1:
        raise ValueError("the head dimension of the query and the cache must be contiguous")
    if table.dtype is not torch.int32 or lens.dtype is not torch.int32:
        raise ValueError("the block table and the lengths must be int32")
    if len(table_shape) != 2 or lens.dim() != 1 or len(lens) < table_shape[0]:
        raise ValueError("the block table must be [rows, width] with a length per row")
    table_stride = table.stride()
    if (table_shape[1] > 1 and table_stride[1] != 1) or (table_shape[0] > 1 and lens.stride(0) != 1):
        raise ValueError("the block table's rows and the lengths must be contiguous")
    device = query.device
    if device.type != "cuda":
        raise ValueError("the attention runs on the device: the query must be a CUDA tensor")
    index = device.index
    if kv_cache.get_device() != index or table.get_device() != index or lens.get_device() != index:
        raise ValueError(f"the cache, the block table and the lengths must be on the query's device {device}")
    return device, dtype, q_shape, kv_shape, table_shape, q_stride, kv_stride, table_stride[0]


def _outputs(query: torch.Tensor, out: torch.Tensor | None, lse: torch.Tensor | None):
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != query.shape or out.dtype is not query.dtype or out.device != query.device or out.stride(2) != 1:
        raise ValueError("out must match the query's shape, dtype and device, its head dimension contiguous")
    if lse is None:
        lse = query.new_empty(query.shape[:2], dtype=torch.float32)
    elif lse.shape != query.shape[:2] or lse.dtype is not torch.float32 or lse.device != query.device or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 {tuple(query.shape[:2])} tensor on the query's device")
    return out, lse


def _status(status: torch.Tensor | None, device: torch.device) -> int | None:
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.numel() != 1 or status.device != device:
        raise ValueError(f"status must be one int32 on {device}")
    return status.data_ptr()


def attend(
    query: torch.Tensor,
    kv_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    scale: float,
    *,
    query_start: torch.Tensor | None = None,
    prefix_blocks: torch.Tensor | int | None = None,
    group_start: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``softmax(scale * query keys) values`` of every query token, and the log of its sum of exponentials.

    ``query`` is [tokens, q_heads, dim], ``kv_cache`` [blocks, 2, block, kv_heads, dim] (keys, then values) of
    the same dtype, float16 or bfloat16, ``table`` int32 [rows, width] and ``lens`` int32 [rows] the row's tokens
    in the cache, those of its query included. Row ``r`` has the query tokens ``query_start[r]`` to
    ``query_start[r + 1]`` (int32 [rows + 1]; without it one token each), the last of which sees the whole row,
    each one before it one position less.

    ``prefix_blocks`` int32 [groups]: the rows ``group_start[g]`` to ``group_start[g + 1]`` (int32 [groups + 1];
    without it one group of every row) begin with the same ``prefix_blocks[g]`` blocks, which are read once for
    the group. An int is one group of every row, as an engine's common prefix length gives it. A row that does not hold
    as much of the prefix as the longest of its group reads what it has itself.

    What lies behind a row may hold anything, another row's tokens in a shared prefix too; values at positions that one of a row's query tokens sees and another does
    not must be finite.

    Returns ``(out, lse)``, float32 [tokens, q_heads] for ``lse``; a token that sees nothing, or only scores of -inf,
    gets 0 and -inf, one that is NaN itself or sees a NaN key gets NaN in both, a token of no row keeps what the
    buffers held. ``status`` (one int32) receives the EKV_STATUS_* bits of faults
    in the tables, which the kernels skip. ``out`` may be the query itself. The call runs on the current stream of the
    query's device.
    """
    whole = prefix_blocks is None or isinstance(prefix_blocks, torch.Tensor)
    common = 0 if whole else _count("prefix_blocks", prefix_blocks)
    device, dtype, q_shape, kv_shape, table_shape, q_stride, kv_stride, table_stride = _batch(query, kv_cache, table, lens)
    tokens, q_heads, dim = q_shape
    rows, width = table_shape
    blocks, _, block_size, kv_heads, _ = kv_shape
    groups = 0
    prefix = None
    if isinstance(prefix_blocks, torch.Tensor):
        groups = prefix_blocks.shape[0] if prefix_blocks.dim() == 1 else 0
        if groups == 0 or (group_start is None and groups != 1):
            raise ValueError("prefix_blocks must hold a count per group, and several groups need group_start")
        prefix = _index("prefix_blocks", prefix_blocks, groups, device)
    elif common:
        if common < 0:
            raise ValueError("prefix_blocks must not be negative")
        common, groups = min(common, width), 1
    if group_start is not None and prefix is None:
        raise ValueError("group_start needs the groups' prefix_blocks")
    starts = _index("query_start", query_start, rows + 1, device)
    members = _index("group_start", group_start, groups + 1, device)
    if starts is None and tokens != rows:
        raise ValueError(f"{tokens} query tokens for {rows} rows: without query_start every row has one")
    word = _status(status, device)
    out, lse = _outputs(query, out, lse)
    if tokens == 0 or rows == 0:
        return out, lse
    out_stride = out.stride()
    lib = _lib.load()
    size = _workspace(rows, tokens, groups, q_heads, kv_heads, dim)
    with _lib.on_device(device) as stream:
        workspace = query.new_empty(size, dtype=torch.uint8)
        rc = lib.ekv_attend(
            query.data_ptr(), q_stride[0], q_stride[1], kv_cache.data_ptr(), kv_stride[0], kv_stride[1], kv_stride[2],
            kv_stride[3], blocks, table.data_ptr(), table_stride, lens.data_ptr(), starts, tokens, rows, width, block_size,
            q_heads, kv_heads, dim, dtype,
            float(scale), groups, members, prefix, common, out.data_ptr(), out_stride[0], out_stride[1], lse.data_ptr(),
            workspace.data_ptr(), size, word, stream,
        )
    _lib.check(rc, "ekv_attend")
    return out, lse


def check_scores(scores: torch.Tensor, heads: int, tokens: int, device: torch.device) -> tuple:
    """The strides of a score table [slots, heads, >= tokens] float32 on ``device``, each head's scores contiguous."""
    shape, stride = scores.shape, scores.stride()
    if scores.dtype is not torch.float32 or len(shape) != 3 or scores.get_device() != device.index:
        raise ValueError(f"scores must be a float32 [slots, heads, tokens] tensor on {device}")
    if shape[1] != heads or shape[2] < tokens:
        raise ValueError(f"scores of {heads} heads and at least {tokens} tokens are needed, got {tuple(shape)}")
    if stride[2] != 1:
        raise ValueError("the scores of a head must be contiguous")
    return stride


def attend_scored(
    query: torch.Tensor,
    kv_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    scale: float,
    scores: torch.Tensor,
    *,
    query_start: torch.Tensor | None = None,
    slots: torch.Tensor | None = None,
    fresh: torch.Tensor | None = None,
    decay: float = 1.0,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``attend``, and the weight that every cached token receives added to its score, in place.

    ``scores`` is float32 [slots, kv_heads, >= width * block]; row ``r`` uses slot ``slots[r]`` (int32 [rows];
    without it slot ``r``). Per KV head, the token at position ``t`` receives the sum of ``exp(scale q.k - lse)`` over
    the row's query tokens and the head's query heads. The row's newest ``fresh[r]`` tokens (int32 [rows]; without it
    the row's query tokens) have no score yet and take that sum; the others' scores become ``decay`` times
    themselves plus it. A prompt's last tokens score the whole prompt with ``fresh = lens``. A negative slot attends
    without scoring; slots must otherwise be one row's alone.

    The other arguments, and the ``(out, lse)`` returned, are ``attend``'s; but with more than 16 query rows a KV head
    (on average) the queries are read again for the weights, and an ``out`` that shares memory with them is refused.
    """
    device, dtype, q_shape, kv_shape, table_shape, q_stride, kv_stride, table_stride = _batch(query, kv_cache, table, lens)
    tokens, q_heads, dim = q_shape
    rows, width = table_shape
    blocks, _, block_size, kv_heads, _ = kv_shape
    score_stride = check_scores(scores, kv_heads, width * block_size, device)
    starts = _index("query_start", query_start, rows + 1, device)
    places = _index("slots", slots, rows, device)
    new = _index("fresh", fresh, rows, device)
    if starts is None and tokens != rows:
        raise ValueError(f"{tokens} query tokens for {rows} rows: without query_start every row has one")
    if not 0.0 <= decay <= 1.0:
        raise ValueError("the decay must lie in [0, 1]")
    word = _status(status, device)
    out, lse = _outputs(query, out, lse)
    if tokens == 0 or rows == 0:
        return out, lse
    out_stride = out.stride()
    lib = _lib.load()
    size = _scored_workspace(rows, tokens, width, block_size, q_heads, kv_heads, dim)
    with _lib.on_device(device) as stream:
        workspace = query.new_empty(size, dtype=torch.uint8)
        rc = lib.ekv_attend_scored(
            query.data_ptr(), q_stride[0], q_stride[1], kv_cache.data_ptr(), kv_stride[0], kv_stride[1], kv_stride[2],
            kv_stride[3], blocks, table.data_ptr(), table_stride, lens.data_ptr(), starts, tokens, rows, width, block_size,
            q_heads, kv_heads, dim, dtype,
            float(scale), scores.data_ptr(), score_stride[0], score_stride[1], len(scores), places, new, float(decay),
            out.data_ptr(), out_stride[0], out_stride[1], lse.data_ptr(), workspace.data_ptr(), size, word, stream,
        )
    _lib.check(rc, "ekv_attend_scored")
    return out, lse
