// Eviction from the paged cache by accumulated attention weight: which tokens of a row to keep, and the kept tokens
// moved to the front of the row's blocks.
//
// select_kernel. A token's rank is its score (float32; NaN as -inf), equal scores to the older token; a row's first
// and newest tokens are kept whatever they score. A cluster of CTAs per (row, KV head), each with a slice of the row and
// each warp with a run of it: the scores become order-preserving 32-bit keys in registers (up to 32 a lane; longer rows
// are read again for each pass), four passes of an 8-bit digit each find the key of the last token kept and how many
// equal to it are, and the warps write the kept positions of their runs, ascending, then -1. Scores crowd into a few exponents, so every lane counts in its
// own column of bins, which is a bank of its own (with one histogram for all lanes, or eight, the additions of the first
// pass waited for one another: 8 us of 8 x 8 units of 65536 tokens). The CTAs' counts are added through distributed
// shared memory, in integers: no order matters. The passes end early at a digit with which nothing more is kept.
// What bounds it: 8 rows x 8 heads of 65536 tokens take 35 us (floor 5): a CTA's steps one after another -- 15000 cycles until
// its scores are there, 5000 to 7000 a pass with its two cluster exchanges, 5000 for the lists -- at two CTAs an SM.
//
// compact: position j of a (row, head) takes the key, value and score of position kept[j] >= j, in place, in
// chunks: a chunk's sources are all read before any of it is written, and later chunks only read positions past
// it, so the copy that fills chunk k + 1 may run while chunk k is stored. check_kernel comes first: the list must ascend
// strictly, from the identity on the protected first tokens, and no block behind those may be another row's, or occur
// twice in the row, also where its other holder protects it. A block is claimed once in an owner table, or marked as
// protected there, which any number of rows may do; a row that fails is left as it was.
#include <cooperative_groups.h>

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
constexpr int kSelectWarps = kSelectThreads / 32;
static_assert(kSelectWarps == 16, "the last walk's sums over warps and CTAs");

__device__ __forceinline__ uint32_t score_key(float x) {  // larger is better; -0 as 0
  if (isnan(x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// KEYS: keys of a lane that stay in registers; 0: rows too long for that.
template <int KEYS>
__global__ void __launch_bounds__(kSelectThreads, 2) select_kernel(const __grid_constant__ SelectParams p) {
  namespace cg = cooperative_groups;
  // few keys a lane: one histogram will do, and saves the step that adds the lanes' columns
  constexpr bool kColumns = KEYS == 0 || KEYS > 8;
  __shared__ int s_lanes[kColumns ? 256 : 1][32];
  __shared__ int s_sum[256];
  __shared__ __align__(16) int s_hist[2][256];
  __shared__ int s_pick[2];
  __shared__ int s_count[2][kSelectWarps];  // per warp: tokens kept anyway or above, tokens equal to the last kept
  __shared__ int s_total[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  chain_release();
  chain_wait();
  const int unit = blockIdx.x / C;
  const int row = unit / p.heads, head = unit - row * p.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = max(p.lens[row], 0);
  int slot = p.slots != nullptr ? p.slots[row] : row;
  const bool reports = threadIdx.x == 0 && rank == 0 && head == 0;
  if (reports) {
    if (n > p.capacity) set_status(p.status, EKV_STATUS_LEN_OVER_WIDTH);
    if (slot >= p.n_slots) set_status(p.status, EKV_STATUS_BAD_SLOT);
  }
  n = min(n, p.capacity);
  if (slot >= p.n_slots) slot = -1;
  const int keep = p.keep != nullptr ? p.keep[row] : p.keep_all;
  const int first = min(p.first, n), recent = min(p.recent, n - first);
  const int m = keep < 0 || keep >= n || slot < 0 ? n : max(keep, first + recent);
  int32_t* out = p.kept + (int64_t)row * p.k0 + (int64_t)head * p.k1;
  if (reports) p.new_lens[row] = m;
  if (m == n) {  // the same for every CTA of the cluster
    for (int i = rank * kSelectThreads + threadIdx.x; i < p.capacity; i += C * kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const float* scores = p.scores + (int64_t)slot * p.s0 + (int64_t)head * p.s1;
  // a warp's run of tokens [from, to)
  const int run = KEYS > 0 ? 32 * KEYS : (((n + C - 1) / C + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32;
  const int from = min(n, (rank * kSelectWarps + warp) * run), to = min(n, from + run);
  // A token's key: what is kept anyway above every score, what is not the run's below.
  auto key_of = [&](int i, float x) { return i >= to ? 0u : i < first || i >= n - recent ? 0xffffffffu : score_key(x); };
  uint32_t keys[KEYS > 0 ? KEYS : 1];
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
      const int i = from + 32 * k + lane;
      keys[k] = i < to ? __float_as_uint(scores[i]) : 0u;
    }
  }
  for (int i = m + rank * kSelectThreads + threadIdx.x; i < p.capacity; i += C * kSelectThreads) out[i] = -1;
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int k = 0; k < KEYS; ++k) keys[k] = key_of(from + 32 * k + lane, __uint_as_float(keys[k]));
  }
  // visit(i, key) for the run's tokens, 32 at a time with the whole warp; i may lie behind `to`
  auto walk = [&](auto visit) {
    if constexpr (KEYS > 0) {
#pragma unroll
      for (int k = 0; k < KEYS; ++k) visit(from + 32 * k + lane, keys[k]);
    } else {
      for (int base = from; base < to; base += 32) visit(base + lane, key_of(base + lane, base + lane < to ? scores[base + lane] : 0.f));
    }
  };
  int want = m;  // tokens above the one that is being found: fewer than there are
  uint32_t prefix = 0, mask = 0;
  if (kColumns) {
    for (int i = threadIdx.x; i < 256 * 32; i += kSelectThreads) (&s_lanes[0][0])[i] = 0;
  } else {
    for (int i = threadIdx.x; i < 512; i += kSelectThreads) (&s_hist[0][0])[i] = 0;
  }
  __syncthreads();
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    int* hist = s_hist[pass & 1];
    walk([&](int, uint32_t key) {
      const int digit = (key >> shift) & 255;
      if ((key & mask) == prefix && key != 0u) atomicAdd(kColumns ? &s_lanes[digit][lane] : &hist[digit], 1);
    });
    __syncthreads();
#pragma unroll
    for (int d = 0; kColumns && d < 256 / kSelectWarps; ++d) {
      const int bin = warp * (256 / kSelectWarps) + d;
      const int count = __reduce_add_sync(kFullMask, s_lanes[bin][lane]);
      s_lanes[bin][lane] = 0;
      if (lane == 0) hist[bin] = count;
    }
    cluster.sync();  // every CTA's histogram of this pass; the next pass fills the other one
    if (threadIdx.x < 256) {
      int count = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < C) count += cluster.map_shared_rank(hist, c)[threadIdx.x];
      s_sum[threadIdx.x] = count;
    } else if (!kColumns) {
      s_hist[(pass + 1) & 1][threadIdx.x - 256] = 0;  // read by every CTA before the barrier above
    }
    __syncthreads();
    if (warp == 0) {  // lane l holds digits [248 - 8 l, 256 - 8 l): from the largest down
      const int top = 255 - 8 * lane;
      int count[8], sum = 0;
#pragma unroll
      for (int d = 0; d < 8; ++d) sum += count[d] = s_sum[top - d];
      int incl = sum;
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(kFullMask, incl, off);
        if (lane >= off) incl += v;
      }
      int before = incl - sum;
      // the digit in which the count of larger keys passes `want`: exactly one lane finds it
      if (before <= want && want < incl) {
        int digit = 0;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const bool here = before <= want && want < before + count[d];
          if (here) {
            digit = top - d;
            s_pick[1] = want - before;
          }
          before += count[d];
        }
        s_pick[0] = digit;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_pick[0] << shift;
    mask |= 255u << shift;
    want = s_pick[1];
    if (want == 0) break;  // nothing that begins like this is kept: its further digits do not matter
    __syncthreads();       // before s_pick is written again
  }
  if constexpr (KEYS > 0) {
    if (mask != 0xffffffffu) {
#pragma unroll
      for (int k = 0; k < KEYS; ++k) keys[k] &= mask;
    }
  }
  // keep every key above `prefix` (in the digits found) and the `want` oldest equal to it: counted per warp, then placed
  int sure = 0, equal = 0;
  walk([&](int, uint32_t key) {
    if (KEYS == 0) key &= mask;
    sure += key > prefix;
    equal += key == prefix;
  });
  sure = __reduce_add_sync(kFullMask, sure);
  equal = __reduce_add_sync(kFullMask, equal);
  if (lane == 0) {
    s_count[0][warp] = sure;
    s_count[1][warp] = equal;
  }
  __syncthreads();
  if (warp < 2) {
    const int sum = __reduce_add_sync(kFullMask, lane < kSelectWarps ? s_count[warp][lane] : 0);
    if (lane == 0) s_total[warp] = sum;
  }
  cluster.sync();
  // lanes 0 to 15 add the warps before this one, lanes 16 to 23 the CTAs before
  int sure_before = lane < warp ? s_count[0][lane & 15] : 0, equal_before = lane < warp ? s_count[1][lane & 15] : 0;
  if (lane >= 16 && lane - 16 < rank) {
    const int* remote = cluster.map_shared_rank(s_total, lane - 16);
    sure_before = remote[0];
    equal_before = remote[1];
  }
  sure_before = __reduce_add_sync(kFullMask, sure_before);
  equal_before = __reduce_add_sync(kFullMask, equal_before);
  const uint32_t below = lanes_below();
  if (equal == 0) {  // nearly every run: no score equal to the last one kept
    int place = sure_before + min(equal_before, want);
    walk([&](int i, uint32_t key) {
      const bool take = (KEYS == 0 ? key & mask : key) > prefix;
      const uint32_t takes = __ballot_sync(kFullMask, take);
      if (take) out[place + __popc(takes & below)] = i;
      place += __popc(takes);
    });
  } else {
    walk([&](int i, uint32_t key) {
      if (KEYS == 0) key &= mask;
      const bool is_sure = key > prefix, is_equal = key == prefix;  // where some are kept, `prefix` is a score's whole key: not 0
      const uint32_t sures = __ballot_sync(kFullMask, is_sure), equals = __ballot_sync(kFullMask, is_equal);
      const int tied = equal_before + __popc(equals & below);
      const int place = sure_before + __popc(sures & below) + min(tied, want);
      if (is_sure || (is_equal && tied < want)) out[place] = i;
      sure_before += __popc(sures);
      equal_before += __popc(equals);
    });
  }
  cluster.sync();  // no CTA leaves while another reads its totals
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
  uint32_t* owner;  // [pool_blocks] the row that claimed it + 1, and kProtected; NULL: few blocks, compared with one another
  int32_t* bad;    // [rows] kRow* bits that rows find in each other, with an owner table
  int32_t* flags;  // [rows][heads] kRow* bits
  int32_t* hole;   // [rows][heads] the first position that takes another's token
  int32_t* result_lens;  // [rows] the tokens that the rows hold afterwards, or NULL
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

// Tables of up to this many entries have each moving row's blocks compared with every entry instead: no owner table to
// clear, which is a launch less (four rows of 44 blocks: see ekv_compact_tokens).
constexpr int kFewBlocks = 512;

constexpr uint32_t kProtected = 0x80000000u;  // of an owner entry: a moving row keeps the block's tokens in place

__global__ void __launch_bounds__(kCheckThreads) check_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int s_hole, s_flags;
  __shared__ int s_ids[kFewBlocks];
  chain_release();
  chain_wait();
  const int row = blockIdx.x / p.heads, head = blockIdx.x - row * p.heads;
  int n, m;
  const bool moves = row_moves(p, row, n, m);
  if (threadIdx.x == 0) {
    s_hole = m;
    s_flags = 0;
  }
  __syncthreads();
  if (head == 0) {
    const int64_t most = (int64_t)p.width * p.block_size;
    if (threadIdx.x == 0 && p.lens[row] > most) set_status(p.status, EKV_STATUS_LEN_OVER_WIDTH);
    // the blocks that must be the row's own: all that it holds, but for those a moving row's protected tokens fill
    const int blocks = (n + p.block_size - 1) / p.block_size, own = moves ? p.first / p.block_size : 0;
    auto outside = [&](int id) {
      const bool bad = id < 0 || id >= p.pool_blocks;
      if (bad && moves) atomicOr(&s_flags, kRowBlock);
      return bad;
    };
    if (p.owner == nullptr) {
      for (int b = threadIdx.x; b < blocks; b += kCheckThreads) outside(s_ids[b] = p.table[(int64_t)row * p.table_s0 + b]);
    } else {
      // eight blocks of a thread at a time, whose ids, and then whose claims, are under way together (four rows of 2112 blocks,
      // 2048 of them shared: 25.5 us for the call, 27.4 with one block after another)
      for (int b0 = threadIdx.x; b0 < blocks; b0 += 8 * kCheckThreads) {
        int id[8];
        uint32_t other[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int b = b0 + k * kCheckThreads;
          id[k] = b < blocks ? p.table[(int64_t)row * p.table_s0 + b] : 0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int b = b0 + k * kCheckThreads;
          other[k] = b >= blocks || outside(id[k]) ? 0u
                     : b >= own ? atomicCAS(&p.owner[id[k]], 0u, (uint32_t)row + 1) : atomicOr(&p.owner[id[k]], kProtected);
        }
        // whichever of two comes second sees the other: a second claim is bad for both rows, a claim of what some row
        // protects for the one that claims
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t claimed = other[k] & ~kProtected;
          if (b0 + k * kCheckThreads >= own && other[k] != 0) atomicOr(&p.bad[row], kRowShared);
          if (claimed != 0) atomicOr(&p.bad[claimed - 1], kRowShared);
        }
      }
    }
    if (p.owner == nullptr && moves) {
      __syncthreads();
      for (int i = threadIdx.x; i < p.rows * p.width; i += kCheckThreads) {
        const int r = i / p.width, b = i - r * p.width;
        int held, kept;
        row_moves(p, r, held, kept);
        if (b >= (held + p.block_size - 1) / p.block_size) continue;
        const int id = p.table[(int64_t)r * p.table_s0 + b];
        bool shared = false;
        for (int mine = own; mine < blocks; ++mine) shared |= s_ids[mine] == id && (r != row || mine != b);
        if (shared) atomicOr(&s_flags, kRowShared);
      }
    }
    if (moves && p.scores != nullptr) {
      const int slot = p.slots != nullptr ? p.slots[row] : row;
      bool bad = slot >= p.n_slots;
      if (slot >= 0 && p.slots != nullptr)
        for (int i = threadIdx.x; i < p.rows; i += kCheckThreads) bad |= i != row && p.slots[i] == slot;
      if (bad) atomicOr(&s_flags, kRowSlot);
    }
  }
  if (!moves) return;
  const int32_t* list = p.kept + (int64_t)row * p.k0 + (int64_t)head * p.k1;
  bool ok = m <= p.columns;
  if (ok) {
    for (int j = threadIdx.x; j < m; j += kCheckThreads) {
      const int v = list[j];
      ok = ok && v > (j > 0 ? list[j - 1] : -1) && v < n && (j >= p.first || v == j);
      if (v != j) atomicMin(&s_hole, j);
    }
  }
  if (!ok) atomicOr(&s_flags, kRowList);
  __syncthreads();
  if (threadIdx.x == 0) {
    p.hole[row * p.heads + head] = s_hole;
    p.flags[row * p.heads + head] = s_flags;
  }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kMoveLoads = 4;  // 16-byte loads of a lane and chunk: 2 KB a warp, 16 KB a CTA, two chunks in flight

// A cluster of CTAs per (row, KV head) takes C chunks at a time, one each. SPLIT: keys and values are units of their own.
__global__ void __launch_bounds__(kMoveThreads, 4) move_kernel(const __grid_constant__ CompactParams p, int split) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  chain_release();
  chain_wait();
  int unit = blockIdx.x / C;
  const int only = split ? unit & 1 : 0;  // the part this unit moves
  if (split) unit >>= 1;
  const int row = unit / p.heads, head = unit - row * p.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n, m;
  const bool reports = threadIdx.x == 0 && rank == 0 && head == 0 && only == 0, moves = row_moves(p, row, n, m);
  int bad = 0;  // a row is moved whole or not at all
  if (moves) {  // as every CTA of the cluster finds
    for (int h = lane; h < p.heads; h += 32) bad |= p.flags[row * p.heads + h];
    bad = __reduce_or_sync(kFullMask, bad) | (p.owner != nullptr ? p.bad[row] : 0);
  }
  if (reports && p.result_lens != nullptr) p.result_lens[row] = moves && !bad ? m : p.lens[row];
  if (!moves) return;
  if (bad) {
    if (reports)
      set_status(p.status, (bad & kRowShared ? EKV_STATUS_BLOCK_SHARED : 0u) | (bad & kRowList ? EKV_STATUS_BAD_LIST : 0u) |
                               (bad & kRowBlock ? EKV_STATUS_BAD_BLOCK_ID : 0u) | (bad & kRowSlot ? EKV_STATUS_BAD_SLOT : 0u));
    return;
  }
  const int start = p.hole[row * p.heads + head];
  if (start >= m) return;
  const int32_t* list = p.kept + (int64_t)row * p.k0 + (int64_t)head * p.k1;
  const int32_t* ids = p.table + (int64_t)row * p.table_s0;
  const int slot = p.scores == nullptr || only == 1 ? -1 : (p.slots != nullptr ? p.slots[row] : row);
  float* scores = slot < 0 ? nullptr : p.scores + (int64_t)slot * p.s0 + (int64_t)head * p.s1;
  uint8_t* heads_at = p.kv + (int64_t)head * p.c_head + only * p.c_part;
  const int pieces = p.row_bytes / 16, per_token = split ? pieces : 2 * pieces;  // 16-byte pieces
  const int tw = min(32, kMoveLoads * 32 / per_token);                             // tokens of a warp's chunk
  const uint32_t inverse = (65536 + per_token - 1) / per_token;                    // i / per_token for i < 128
  const int step = C * kMoveWarps * tw;

  // A lane's token of the warp's chunk at j0: its destination is position j0 + lane, its source list[j0 + lane]. Chunks
  // run through a pipeline -- positions, then block ids and with them the bytes' places, then the bytes -- so that only the
  // last step's latency is left at each chunk, and that one beside the chunk before.
  struct Place {
    int64_t source, target;
    int from, to;
  };
  auto positions = [&](int j0, Place& a) {
    const int j = j0 + lane;
    const bool real = lane < tw && j < m;
    a.to = real ? j : -1;
    a.from = real ? list[j] : 0;
  };
  auto places = [&](Place& a) {
    if (a.to < 0) return;
    const int sb = a.from / p.block_size, tb = a.to / p.block_size;
    a.source = (int64_t)ids[sb] * p.c_block + (int64_t)(a.from - sb * p.block_size) * p.c_pos;
    a.target = (int64_t)ids[tb] * p.c_block + (int64_t)(a.to - tb * p.block_size) * p.c_pos;
  };
  auto piece = [&](int s, int& token) -> int64_t {  // where piece s * 32 + lane of the chunk lies in its token's rows
    const uint32_t i = s * 32 + lane;
    token = (int)(i * inverse >> 16);
    const int rest = (int)i - token * per_token;
    const int part = rest >= pieces;
    return (int64_t)part * p.c_part + 16 * (rest - part * pieces);
  };
  auto load = [&](const Place& a, uint4 (&v)[kMoveLoads], float& score) {
#pragma unroll
    for (int s = 0; s < kMoveLoads; ++s) {
      int token;
      const int64_t at = piece(s, token);
      const int64_t source = __shfl_sync(kFullMask, a.source, token & 31);
      const int to = __shfl_sync(kFullMask, a.to, token & 31);
      if (token < tw && to >= 0) v[s] = __ldcg(reinterpret_cast<const uint4*>(heads_at + source + at));
    }
    if (scores != nullptr && a.to >= 0) score = scores[a.from];
  };
  auto store = [&](const Place& a, const uint4 (&v)[kMoveLoads], float score) {
#pragma unroll
    for (int s = 0; s < kMoveLoads; ++s) {
      int token;
      const int64_t at = piece(s, token);
      const int64_t target = __shfl_sync(kFullMask, a.target, token & 31);
      const int to = __shfl_sync(kFullMask, a.to, token & 31);
      if (token < tw && to >= 0) __stcg(reinterpret_cast<uint4*>(heads_at + target + at), v[s]);
    }
    if (scores != nullptr && a.to >= 0) scores[a.to] = score;
  };
  const int j0 = start + (rank * kMoveWarps + warp) * tw;
  Place now, next, after;
  uint4 v[2][kMoveLoads];
  float score[2];
  positions(j0, now);
  positions(j0 + step, next);
  places(now);
  load(now, v[0], score[0]);
  places(next);
  int buf = 0;
  // every chunk of the cluster's step is read before any of it is written; the steps after it read only positions past
  // what this one writes
#pragma unroll 2
  for (int base = start; base < m; base += step) {
    const int j = j0 + (base - start);
    positions(j + 2 * step, after);
    load(next, v[buf ^ 1], score[buf ^ 1]);
    if (C > 1) cluster.sync(); else __syncthreads();
    store(now, v[buf], score[buf]);
    places(after);
    now = next;
    next = after;
    buf ^= 1;
  }
}

struct CompactLayout {
  size_t owner, bad, flags, hole, total;
};

// Whether two arrays of `count` int32 share memory.
bool overlap(const int32_t* a, const int32_t* b, int count) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), size = (uintptr_t)count * 4;
  return x < y + size && y < x + size;
}

CompactLayout compact_layout(int rows, int heads, int64_t pool_blocks) {
  CompactLayout w{};
  w.owner = 0;
  w.bad = (size_t)pool_blocks * 4;
  w.flags = w.bad + (size_t)rows * 4;
  w.hole = w.flags + (size_t)rows * heads * 4;
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
  if ((heads > 1 && score_stride_head < capacity) || (n_slots > 1 && score_stride_slot < capacity))
    return fail(EKV_EINVAL, "a score stride is below the capacity");
  if ((heads > 1 && kept_stride_head < capacity) || (rows > 1 && kept_stride_row < capacity))
    return fail(EKV_EINVAL, "a stride of the kept lists is below the capacity");
  if ((int64_t)rows * heads > 0x7fffffffll / 8 || capacity > 0x7fffffff - 4096)
    return fail(EKV_ENOTSUP, "more than 2^31 - 1 rows x heads, or tokens of a row");
  const SelectParams p{scores, score_stride_slot, score_stride_head, slots, n_slots, capacity, lens, keep, keep_all, first_tokens,
                       recent_tokens, rows, heads, kept, kept_stride_row, kept_stride_head, new_lens, status};
  int device = 0, sms = 0, rc;
  if ((rc = current_device(&device)) != EKV_OK || (rc = sm_count(device, &sms)) != EKV_OK) return rc;
  // The fewest CTAs a unit whose registers hold the row, then as many more as leave every CTA resident (two an SM) with a
  // run of at least 4 keys a lane.
  const int64_t units = (int64_t)rows * heads;
  auto lane_keys = [&](int C) { return (int)(((int64_t)capacity + C * kSelectThreads - 1) / (C * kSelectThreads)); };
  int C = 1;
  while (C < 8 && lane_keys(C) > 32) C *= 2;
  while (C < 8 && lane_keys(C) > 4 && units * C * 2 <= 2 * sms) C *= 2;
  const int keys = lane_keys(C);
  auto kernel = keys <= 4 ? select_kernel<4> : keys <= 8 ? select_kernel<8> : keys <= 16 ? select_kernel<16>
                : keys <= 32 ? select_kernel<32> : select_kernel<0>;
  launch_chained_cluster(kernel, dim3((unsigned)(units * C)), dim3(kSelectThreads), 0, static_cast<cudaStream_t>(stream),
                         (unsigned)C, p);
  return check_launch("select_kernel");
}

extern "C" size_t ekv_compact_tokens_workspace_bytes(int rows, int heads, int64_t pool_blocks) {
  if (rows <= 0 || heads <= 0 || pool_blocks <= 0) return 0;
  return compact_layout(rows, heads, pool_blocks).total;
}

extern "C" int ekv_compact_tokens_lens(void* kv, int64_t kv_stride_block, int64_t kv_stride_part, int64_t kv_stride_pos,
                                       int64_t kv_stride_head, int64_t pool_blocks, int head_bytes, const int32_t* table,
                                       int64_t table_stride, const int32_t* lens, int rows, int width, int heads,
                                       int block_size, const int32_t* kept, int64_t kept_stride_row,
                                       int64_t kept_stride_head, int columns, const int32_t* new_lens, int first_tokens,
                                       float* scores, int64_t score_stride_slot, int64_t score_stride_head, int n_slots,
                                       const int32_t* slots, int32_t* result_lens, void* workspace,
                                       size_t workspace_bytes, uint32_t* status, void* stream) {
  clear_error();
  if (!kv || !table || !lens || !kept || !new_lens) return fail(EKV_EINVAL, "a required device pointer is NULL");
  if (rows <= 0 || width <= 0 || heads <= 0 || block_size <= 0 || pool_blocks <= 0 || columns <= 0)
    return fail(EKV_EINVAL, "rows, width, heads, block_size, columns and pool_blocks must be positive");
  if (head_bytes <= 0 || (head_bytes & 15) || head_bytes > 1024)
    return fail(EKV_ENOTSUP, "a head of %d bytes: this build moves 16 to 1024 in whole 16-byte units", head_bytes);
  if (((uintptr_t)kv & 15) || (kv_stride_block & 15) || (kv_stride_part & 15) || (kv_stride_pos & 15) || (kv_stride_head & 15))
    return fail(EKV_EINVAL, "the cache must be 16-byte aligned with strides of whole 16-byte units");
  if (table_stride < width) return fail(EKV_EINVAL, "the table's row stride is below the width");
  if ((heads > 1 && kept_stride_head < columns) || (rows > 1 && kept_stride_row < columns)) return fail(EKV_EINVAL, "a stride of the kept lists is below their length");
  if (first_tokens < 0) return fail(EKV_EINVAL, "first_tokens must not be negative");
  if (pool_blocks > 0x7fffffffll || (int64_t)width * block_size > 0x7fffffffll - 65536 || (int64_t)rows * heads > 0x7fffffffll / 16)
    return fail(EKV_ENOTSUP, "more than 2^31 - 1 blocks, tokens of a row, or rows x heads");
  if (scores) {
    if (n_slots <= 0 || (!slots && n_slots < rows)) return fail(EKV_EINVAL, "%d score slots for %d rows", n_slots, rows);
    const int64_t most = (int64_t)width * block_size;
    if ((heads > 1 && score_stride_head < most) || (n_slots > 1 && score_stride_slot < most))
      return fail(EKV_EINVAL, "scores must hold at least width * block_size tokens for every slot and head");
  }
  if (result_lens && (overlap(result_lens, lens, rows) || overlap(result_lens, new_lens, rows)))
    return fail(EKV_EINVAL, "result_lens must share no memory with lens or new_lens");
  const CompactLayout w = compact_layout(rows, heads, pool_blocks);
  if (!workspace || workspace_bytes < w.total || ((uintptr_t)workspace & 255))
    return fail(EKV_ERANGE, "the workspace must hold %zu bytes at a 256-byte boundary", w.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool few = (int64_t)rows * width <= kFewBlocks;
  if (!few && cudaMemsetAsync(ws, 0, w.flags, s) != cudaSuccess) return check_launch("cudaMemsetAsync(block owners)");
  const CompactParams p{static_cast<uint8_t*>(kv), kv_stride_block, kv_stride_part, kv_stride_pos, kv_stride_head, pool_blocks,
                        table, table_stride, lens, kept, kept_stride_row, kept_stride_head, columns, new_lens, scores,
                        score_stride_slot, score_stride_head, slots, n_slots, rows, width, heads, block_size, first_tokens,
                        head_bytes, few ? nullptr : reinterpret_cast<uint32_t*>(ws + w.owner), reinterpret_cast<int32_t*>(ws + w.bad),
                        reinterpret_cast<int32_t*>(ws + w.flags), reinterpret_cast<int32_t*>(ws + w.hole), result_lens, status};
  launch_chained(check_kernel, dim3(rows * heads), dim3(kCheckThreads), 0, s, p);
  int rc = check_launch("check_kernel");
  if (rc != EKV_OK) return rc;
  int device = 0, sms = 0;
  if ((rc = current_device(&device)) != EKV_OK || (rc = sm_count(device, &sms)) != EKV_OK) return rc;
  // Up to four CTAs an SM: keys and values apart first, whose units wait for nobody, then clusters of up to the portable size.
  // (32 rows x 8 heads of 4096 tokens: 115 us apart, 130 in clusters of two, 157 as they are; 16 rows of 8192: 132 us apart
  // and in twos, 163 apart alone, 198 with two CTAs an SM.)
  const int64_t units = (int64_t)rows * heads;
  const int split = units * 2 <= 4 * sms;
  int C = 1;
  while (C < 8 && units * (split + 1) * C * 2 <= 4 * sms) C *= 2;
  launch_chained_cluster(move_kernel, dim3((unsigned)(units * C * (split ? 2 : 1))), dim3(kMoveThreads), 0, s, (unsigned)C, p, split);
  return check_launch("move_kernel");
}

extern "C" int ekv_compact_tokens(void* kv, int64_t kv_stride_block, int64_t kv_stride_part, int64_t kv_stride_pos,
                                  int64_t kv_stride_head, int64_t pool_blocks, int head_bytes, const int32_t* table,
                                  int64_t table_stride, const int32_t* lens, int rows, int width, int heads, int block_size,
                                  const int32_t* kept, int64_t kept_stride_row, int64_t kept_stride_head, int columns,
                                  const int32_t* new_lens, int first_tokens, float* scores, int64_t score_stride_slot,
                                  int64_t score_stride_head, int n_slots, const int32_t* slots, void* workspace,
                                  size_t workspace_bytes, uint32_t* status, void* stream) {
  return ekv_compact_tokens_lens(kv, kv_stride_block, kv_stride_part, kv_stride_pos, kv_stride_head, pool_blocks, head_bytes,
                                 table, table_stride, lens, rows, width, heads, block_size, kept, kept_stride_row,
                                 kept_stride_head, columns, new_lens, first_tokens, scores, score_stride_slot,
                                 score_stride_head, n_slots, slots, nullptr, workspace, workspace_bytes, status, stream);
}
