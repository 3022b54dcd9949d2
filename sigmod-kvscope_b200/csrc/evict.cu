// Eviction from the paged cache by accumulated attention weight: which tokens of a row to keep, and the kept tokens
// moved to the front of the row's blocks.
//
// select_kernel. A token's rank is its score (float32; NaN as -inf), equal scores to the older token; a row's first
// and newest tokens are kept whatever they score. One CTA per (row, KV head): the scores as order-preserving 32-bit
// keys, four passes of an 8-bit digit each find the key of the last token kept and how many equal to it are
// (a histogram in shared memory, counted in integers: no order matters), and one ordered pass writes the kept
// positions, ascending, then -1.
//
// compact: position j of a (row, head) takes the key, value and score of position kept[j] >= j, in place, in
// chunks: a chunk's sources are all read before any of it is written, and later chunks only read positions past
// it, so the copy that fills chunk k + 1 may run while chunk k is stored. check_kernel comes first: the list must ascend
// strictly, from the identity on the protected first tokens, and no block the row writes may be another row's, or
// occur twice in the row (each block a row holds is claimed once in an owner table); a row that fails is left as it was.
#include "ekv_common.cuh"

namespace ekv {

namespace {

// ---- select ------------------------------------------------------------------------------------------------

struct SelectParams {
  const float* scores;
  int64_t s0, s1;
  const int32_t* slots;
  int n_slots, capacity;
  const int32_t* lens;
  const int32_t* keep;  // per row, or NULL: keep_all
  int keep_all, first, recent;
  int rows, heads;
  int32_t* kept;
  int64_t k0, k1;
  int32_t* new_lens;
  uint32_t* status;
};

constexpr int kSelectThreads = 512;

__device__ __forceinline__ uint32_t score_key(float x) {  // larger is better; -0 as 0
  if (isnan(x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelectThreads) select_kernel(const __grid_constant__ SelectParams p) {
  __shared__ int s_hist[256];
  __shared__ int s_scan[kSelectThreads / 32 + 1];
  __shared__ int s_pick[2];
  chain_release();
  chain_wait();
  const int row = blockIdx.x / p.heads, head = blockIdx.x - row * p.heads;
  int n = max(p.lens[row], 0);
  int slot = p.slots != nullptr ? p.slots[row] : row;
  if (threadIdx.x == 0 && head == 0) {
    if (n > p.capacity) set_status(p.status, EKV_STATUS_LEN_OVER_WIDTH);
    if (slot >= p.n_slots) set_status(p.status, EKV_STATUS_BAD_SLOT);
  }
  n = min(n, p.capacity);
  if (slot >= p.n_slots) slot = -1;
  const int keep = p.keep != nullptr ? p.keep[row] : p.keep_all;
  const int first = min(p.first, n), recent = min(p.recent, n - first);
  const int m = keep < 0 || keep >= n || slot < 0 ? n : max(keep, first + recent);
  int32_t* out = p.kept + (int64_t)row * p.k0 + (int64_t)head * p.k1;
  if (threadIdx.x == 0 && head == 0) p.new_lens[row] = m;
  if (m == n) {
    for (int i = threadIdx.x; i < p.capacity; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const float* scores = p.scores + (int64_t)slot * p.s0 + (int64_t)head * p.s1;
  const int lo = first, hi = n - recent;  // the tokens to choose from
  int want = m - first - recent;          // >= 0, < hi - lo
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSelectThreads) s_hist[i] = 0;
    __syncthreads();
    for (int i = lo + threadIdx.x; i < hi; i += kSelectThreads) {
      const uint32_t key = score_key(scores[i]);
      if ((key & mask) == prefix) atomicAdd(&s_hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l holds digits [248 - 8 l, 256 - 8 l): from the largest down
      const int top = 255 - 8 * threadIdx.x;
      int sum = 0;
      for (int d = 0; d < 8; ++d) sum += s_hist[top - d];
      int incl = sum;
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(kFullMask, incl, off);
        if ((int)threadIdx.x >= off) incl += v;
      }
      int before = incl - sum;
      // the digit in which the count of larger keys passes `want`: exactly one lane finds it
      if (before <= want && want < incl) {
        int d = 0;
        while (before + s_hist[top - d] <= want) before += s_hist[top - d++];
        s_pick[0] = top - d;
        s_pick[1] = want - before;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_pick[0] << shift;
    mask |= 255u << shift;
    want = s_pick[1];
    __syncthreads();
  }
  // keep every key above `prefix` and the `want` oldest equal to it
  int at = 0, equal = 0;
  for (int base = 0; base < n; base += kSelectThreads) {
    const int i = base + threadIdx.x;
    bool pin = false, above = false, same = false;
    if (i < n) {
      pin = i < lo || i >= hi;
      const uint32_t key = pin ? 0u : score_key(scores[i]);
      above = !pin && key > prefix;
      same = !pin && key == prefix;
    }
    int same_total = 0, kept_total = 0;
    const int rank = equal + block_exclusive_scan<kSelectThreads>(same ? 1 : 0, s_scan, &same_total);
    const bool take = pin || above || (same && rank < want);
    __syncthreads();
    const int place = at + block_exclusive_scan<kSelectThreads>(take ? 1 : 0, s_scan, &kept_total);
    if (take) out[place] = i;
    at += kept_total;
    equal += same_total;
    __syncthreads();
  }
  for (int i = m + threadIdx.x; i < p.capacity; i += kSelectThreads) out[i] = -1;
}

// ---- compact -------------------------------------------------------------------------------------------------

// Why a row is left as it was.
constexpr int kRowShared = 1, kRowList = 2, kRowBlock = 4, kRowSlot = 8;

struct CompactParams {
  uint8_t* kv;
  int64_t c_block, c_part, c_pos, c_head;  // byte strides
  int64_t pool_blocks;
  const int32_t* table;
  int64_t table_s0;
  const int32_t* lens;
  const int32_t* kept;
  int64_t k0, k1;
  int columns;  // of a list
  const int32_t* new_lens;
  float* scores;  // may be NULL
  int64_t s0, s1;
  const int32_t* slots;
  int n_slots;
  int rows, width, heads, block_size, first, row_bytes;
  int32_t* owner;  // [pool_blocks], 0: nobody's
  int32_t* bad;    // [rows] kRow* bits
  int32_t* hole;   // [rows][heads] the first position that takes another's token
  uint32_t* status;
};

constexpr int kCheckThreads = 256;

// The tokens a row goes from and to; none when the row does not shrink.
__device__ __forceinline__ bool row_moves(const CompactParams& p, int row, int& n, int& m) {
  const int64_t most = (int64_t)p.width * p.block_size;
  const int len = p.lens[row];
  n = (int)(len < 0 ? 0 : (len > most ? most : len));
  m = p.new_lens[row];
  return m >= 0 && m < n;
}

__global__ void __launch_bounds__(kCheckThreads) check_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int s_hole;
  chain_release();
  chain_wait();
  const int row = blockIdx.x / p.heads, head = blockIdx.x - row * p.heads;
  int n, m;
  const bool moves = row_moves(p, row, n, m);
  if (head == 0) {
    const int64_t most = (int64_t)p.width * p.block_size;
    if (threadIdx.x == 0 && p.lens[row] > most) set_status(p.status, EKV_STATUS_LEN_OVER_WIDTH);
    const int blocks = (n + p.block_size - 1) / p.block_size;
    for (int b = threadIdx.x; b < blocks; b += kCheckThreads) {
      const int id = p.table[(int64_t)row * p.table_s0 + b];
      if (id < 0 || id >= p.pool_blocks) {
        if (moves) atomicOr(&p.bad[row], kRowBlock);
        continue;
      }
      if (moves && b < p.first / p.block_size) continue;  // protected: read and written by nobody
      const int other = atomicCAS(&p.owner[id], 0, row + 1);
      if (other != 0) {  // claimed before, by another row or by this one
        atomicOr(&p.bad[row], kRowShared);
        atomicOr(&p.bad[other - 1], kRowShared);
      }
    }
    if (moves && p.scores != nullptr) {
      const int slot = p.slots != nullptr ? p.slots[row] : row;
      bool bad = slot >= p.n_slots;
      if (slot >= 0 && p.slots != nullptr)
        for (int i = threadIdx.x; i < p.rows; i += kCheckThreads) bad |= i != row && p.slots[i] == slot;
      if (bad) atomicOr(&p.bad[row], kRowSlot);
    }
  }
  if (!moves) return;
  if (threadIdx.x == 0) s_hole = m;
  __syncthreads();
  const int32_t* list = p.kept + (int64_t)row * p.k0 + (int64_t)head * p.k1;
  bool ok = m <= p.columns;
  if (ok) {
    for (int j = threadIdx.x; j < m; j += kCheckThreads) {
      const int v = list[j];
      ok = ok && v > (j > 0 ? list[j - 1] : -1) && v < n && (j >= p.first || v == j);
      if (v != j) atomicMin(&s_hole, j);
    }
  }
  if (!ok) atomicOr(&p.bad[row], kRowList);
  __syncthreads();
  if (threadIdx.x == 0) p.hole[row * p.heads + head] = s_hole;
}

constexpr int kMoveThreads = 256;
constexpr int kMoveBytes = 32768;  // of a chunk

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ CompactParams p) {
  extern __shared__ __align__(128) uint8_t s_chunk[];  // two chunks, and two of scores behind them
  chain_release();
  chain_wait();
  const int row = blockIdx.x / p.heads, head = blockIdx.x - row * p.heads;
  int n, m;
  if (!row_moves(p, row, n, m)) return;
  const int bad = p.bad[row];
  if (bad) {
    if (threadIdx.x == 0 && head == 0)
      set_status(p.status, (bad & kRowShared ? EKV_STATUS_BLOCK_SHARED : 0u) | (bad & kRowList ? EKV_STATUS_BAD_LIST : 0u) |
                               (bad & kRowBlock ? EKV_STATUS_BAD_BLOCK_ID : 0u) | (bad & kRowSlot ? EKV_STATUS_BAD_SLOT : 0u));
    return;
  }
  const int32_t* list = p.kept + (int64_t)row * p.k0 + (int64_t)head * p.k1;
  const int32_t* ids = p.table + (int64_t)row * p.table_s0;
  const int slot = p.scores == nullptr ? -1 : (p.slots != nullptr ? p.slots[row] : row);
  float* scores = slot < 0 ? nullptr : p.scores + (int64_t)slot * p.s0 + (int64_t)head * p.s1;
  const int pieces = p.row_bytes / 16;          // 16-byte pieces of a key row
  const int per = kMoveBytes / (2 * p.row_bytes);  // tokens of a chunk
  float* s_scores = reinterpret_cast<float*>(s_chunk + 2 * kMoveBytes);
  auto place = [&](int pos, int part, int piece) {
    const int b = pos / p.block_size;
    return p.kv + (int64_t)ids[b] * p.c_block + part * p.c_part + (int64_t)(pos - b * p.block_size) * p.c_pos +
           (int64_t)head * p.c_head + 16 * piece;
  };
  auto load = [&](int j0, int buf) {
    const int count = min(per, m - j0) * 2 * pieces;
    for (int i = threadIdx.x; i < count; i += kMoveThreads) {
      const int j = i / (2 * pieces), rest = i - j * 2 * pieces, part = rest / pieces;
      cp_async16(s_chunk + buf * kMoveBytes + 16 * i, place(list[j0 + j], part, rest - part * pieces));
    }
    if (scores != nullptr)
      for (int j = threadIdx.x; j < min(per, m - j0); j += kMoveThreads)
        cp_async4(s_scores + buf * per + j, scores + list[j0 + j]);
    cp_async_commit();
  };
  const int start = p.hole[row * p.heads + head];
  if (start >= m) return;
  load(start, 0);
  int buf = 0;
  for (int j0 = start; j0 < m; j0 += per, buf ^= 1) {
    if (j0 + per < m) {
      load(j0 + per, buf ^ 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();  // the whole chunk has been read
    const int count = min(per, m - j0) * 2 * pieces;
    for (int i = threadIdx.x; i < count; i += kMoveThreads) {
      const int j = i / (2 * pieces), rest = i - j * 2 * pieces, part = rest / pieces;
      *reinterpret_cast<uint4*>(place(j0 + j, part, rest - part * pieces)) =
          *reinterpret_cast<const uint4*>(s_chunk + buf * kMoveBytes + 16 * i);
    }
    if (scores != nullptr)
      for (int j = threadIdx.x; j < min(per, m - j0); j += kMoveThreads) scores[j0 + j] = s_scores[buf * per + j];
    __syncthreads();  // before the buffer is filled again
  }
}

struct CompactLayout {
  size_t owner, bad, hole, total;
};

CompactLayout compact_layout(int rows, int heads, int64_t pool_blocks) {
  CompactLayout w{};
  w.owner = 0;
  w.bad = (size_t)pool_blocks * 4;
  w.hole = w.bad + (size_t)rows * 4;
  w.total = round_up(w.hole + (size_t)rows * heads * 4, 256);
  return w;
}

}  // namespace

}  // namespace ekv

using namespace ekv;

extern "C" int ekv_select_tokens(const float* scores, int64_t score_stride_slot, int64_t score_stride_head, int n_slots,
                                 int capacity, const int32_t* slots, const int32_t* lens, const int32_t* keep,
                                 int keep_all, int first_tokens, int recent_tokens, int rows, int heads, int32_t* kept,
                                 int64_t kept_stride_row, int64_t kept_stride_head, int32_t* new_lens, uint32_t* status,
                                 void* stream) {
  clear_error();
  if (!scores || !lens || !kept || !new_lens) return fail(EKV_EINVAL, "a required device pointer is NULL");
  if (rows <= 0 || heads <= 0 || capacity <= 0 || n_slots <= 0)
    return fail(EKV_EINVAL, "rows, heads, capacity and slots must be positive");
  if (!slots && n_slots < rows) return fail(EKV_EINVAL, "%d score slots for %d rows", n_slots, rows);
  if (first_tokens < 0 || recent_tokens < 0) return fail(EKV_EINVAL, "first_tokens and recent_tokens must not be negative");
  if (score_stride_head < capacity || score_stride_slot < 0 || (n_slots > 1 && score_stride_slot < score_stride_head))
    return fail(EKV_EINVAL, "a score stride is below the capacity");
  if (kept_stride_head < capacity || kept_stride_row < kept_stride_head)
    return fail(EKV_EINVAL, "a stride of the kept lists is below the capacity");
  if ((int64_t)rows * heads > 0x7fffffffll || capacity > 0x7fffffff - 4096)
    return fail(EKV_ENOTSUP, "more than 2^31 - 1 rows x heads, or tokens of a row");
  const SelectParams p{scores, score_stride_slot, score_stride_head, slots, n_slots, capacity, lens, keep, keep_all,
                       first_tokens, recent_tokens, rows, heads, kept, kept_stride_row, kept_stride_head, new_lens, status};
  launch_chained(select_kernel, dim3(rows * heads), dim3(kSelectThreads), 0, static_cast<cudaStream_t>(stream), p);
  return check_launch("select_kernel");
}

extern "C" size_t ekv_compact_tokens_workspace_bytes(int rows, int heads, int64_t pool_blocks) {
  if (rows <= 0 || heads <= 0 || pool_blocks <= 0) return 0;
  return compact_layout(rows, heads, pool_blocks).total;
}

extern "C" int ekv_compact_tokens(void* kv, int64_t kv_stride_block, int64_t kv_stride_part, int64_t kv_stride_pos,
                                  int64_t kv_stride_head, int64_t pool_blocks, int head_bytes, const int32_t* table,
                                  int64_t table_stride, const int32_t* lens, int rows, int width, int heads, int block_size,
                                  const int32_t* kept, int64_t kept_stride_row, int64_t kept_stride_head, int columns,
                                  const int32_t* new_lens, int first_tokens, float* scores, int64_t score_stride_slot,
                                  int64_t score_stride_head, int n_slots, const int32_t* slots, void* workspace,
                                  size_t workspace_bytes, uint32_t* status, void* stream) {
  clear_error();
  if (!kv || !table || !lens || !kept || !new_lens) return fail(EKV_EINVAL, "a required device pointer is NULL");
  if (rows <= 0 || width <= 0 || heads <= 0 || block_size <= 0 || pool_blocks <= 0 || columns <= 0)
    return fail(EKV_EINVAL, "rows, width, heads, block_size, columns and pool_blocks must be positive");
  if (head_bytes <= 0 || (head_bytes & 15) || head_bytes > 4096)
    return fail(EKV_ENOTSUP, "a head of %d bytes: this build moves 16 to 4096 in whole 16-byte units", head_bytes);
  if (((uintptr_t)kv & 15) || (kv_stride_block & 15) || (kv_stride_part & 15) || (kv_stride_pos & 15) || (kv_stride_head & 15))
    return fail(EKV_EINVAL, "the cache must be 16-byte aligned with strides of whole 16-byte units");
  if (table_stride < width) return fail(EKV_EINVAL, "the table's row stride is below the width");
  if (kept_stride_head < columns || kept_stride_row < 0) return fail(EKV_EINVAL, "a stride of the kept lists is below their length");
  if (first_tokens < 0) return fail(EKV_EINVAL, "first_tokens must not be negative");
  if (pool_blocks > 0x7fffffffll || (int64_t)width * block_size > 0x7fffffffll - 65536 || (int64_t)rows * heads > 0x7fffffffll)
    return fail(EKV_ENOTSUP, "more than 2^31 - 1 blocks, tokens of a row, or rows x heads");
  if (scores) {
    if (n_slots <= 0 || (!slots && n_slots < rows)) return fail(EKV_EINVAL, "%d score slots for %d rows", n_slots, rows);
    if (score_stride_head < (int64_t)width * block_size || score_stride_slot < 0 ||
        (n_slots > 1 && score_stride_slot < score_stride_head))
      return fail(EKV_EINVAL, "scores must hold a slot's heads of at least width * block_size tokens each");
  }
  const CompactLayout w = compact_layout(rows, heads, pool_blocks);
  if (!workspace || workspace_bytes < w.total || ((uintptr_t)workspace & 255))
    return fail(EKV_ERANGE, "the workspace must hold %zu bytes at a 256-byte boundary", w.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(ws, 0, w.hole, s) != cudaSuccess) return check_launch("cudaMemsetAsync(block owners)");
  const CompactParams p{static_cast<uint8_t*>(kv), kv_stride_block, kv_stride_part, kv_stride_pos, kv_stride_head, pool_blocks,
                        table, table_stride, lens, kept, kept_stride_row, kept_stride_head, columns, new_lens, scores,
                        score_stride_slot, score_stride_head, slots, n_slots, rows, width, heads, block_size, first_tokens,
                        head_bytes, reinterpret_cast<int32_t*>(ws + w.owner), reinterpret_cast<int32_t*>(ws + w.bad),
                        reinterpret_cast<int32_t*>(ws + w.hole), status};
  launch_chained(check_kernel, dim3(rows * heads), dim3(kCheckThreads), 0, s, p);
  int rc = check_launch("check_kernel");
  if (rc != EKV_OK) return rc;
  const size_t smem = 2 * kMoveBytes + 2 * (kMoveBytes / (2 * (size_t)head_bytes)) * 4;
  if (cudaFuncSetAttribute(move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(move_kernel)");
  launch_chained(move_kernel, dim3(rows * heads), dim3(kMoveThreads), smem, s, p);
  return check_launch("move_kernel");
}
