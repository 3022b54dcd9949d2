// The attention kernel for units of many query rows, on the tcgen05 tensor cores: the same mathematics as
// attend_kernel (attend.cu), with accumulators in tensor memory.
//
// A CTA an SM. Its M tile is 256 query rows in two subtiles of 128, one for each of two softmax warpgroups (a
// thread a row), and both meet the same 128-token tiles of keys and values in shared memory: at 512 bytes a token
// and head, one such tile feeds 4 x 128^3 multiply-adds. An item of at most 128 query rows gives both
// warpgroups the same rows and alternate tiles, so the tensor cores still have one warpgroup's scores to work on while
// the other takes its exponentials; its two halves join in the combine kernel.
//   copy warp: block ids, then the TMA copies of K0 K1 V0 K2 V1 ... into a ring of 128-token slots (a block that is not
//     there is copied from past the pool, which the TMA engine reads as zeros).
//   mma warp: S = Q K^T into tensor memory, then O += P V with P from tensor memory; one thread issues. S of the next
//     tile follows O of this one, so a score's arrival also says that the output below it is at rest.
//   softmax warpgroups: a row's 128 scores 32 at a time. The running maximum is only raised when it grew by more than 2^8,
//     so most tiles need one pass over their scores, and the output in tensor memory is rescaled a few times a row, by the
//     same threads; probabilities go back to tensor memory over the scores, rounded to the values' type.
//
// What bounds it: 256 query rows on 32768 tokens, 8 KV heads of 128, take 44 us and 1024 query rows 139 us (0.99 PFLOP/s, 59 %
// of the measured bf16 rate; the SM clock falls to 1.5 GHz under it; boxes differ by a tenth). A tile's period was 3650
// cycles, a warpgroup's softmax (2150: 16 exponentials a clock and SM are 1024 of them, twice that when both warpgroups
// overlap; a third of them now run on the FMA pipes) and its two products with their hand-overs (1500) one after the other,
// where the tensor cores need 2048 for both warpgroups; with the softmax left out the kernel takes 121 us. Some 15 us of
// each launch are beginnings and ends: the walk's first loads, the queries, the first tile, 128 KB of sums out of every CTA.
#include <type_traits>

#include "attend.cuh"
#include "mma5.cuh"

namespace ekv {

namespace {

constexpr int kTokens = 128;  // of a tile
constexpr int kSub = 128;     // query rows of a subtile
constexpr int kThreads = 320;
constexpr int kCopyWarp = 8, kMmaWarp = 9;
constexpr int kColumns = 512;  // of tensor memory: S of both subtiles, then O of both

template <int D>
struct Wide {
  static constexpr int kHalves = D / 64;
  static constexpr int kHalf = kTokens * 128;         // bytes of a 64-dim half of 128 rows
  static constexpr int kSlot = kHalves * kHalf;       // of a tile's keys, or values, or a subtile's queries
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kRing = kSlots * kSlot;
};

template <int D>
struct WideTail {
  uint64_t full[Wide<D>::kSlots], empty[Wide<D>::kSlots];
  uint64_t q_full[2], s_full[2], p_ready[2], o_full[2], o_free[2], drained;
  uint32_t tmem;
  int scratch[kThreads / 32 + 1], found[2];
};

// ---- the walk that all warps share ---------------------------------------------------------------------------

// How an item's tiles fall to the two warpgroups: with one subtile of rows the even tiles to the first and the odd ones
// to the second, otherwise all to both.
struct Share {
  bool single;
  int tiles;  // of the item that this CTA covers
  __device__ __forceinline__ int of(int w) const { return single ? (tiles + 1 - w) / 2 : tiles; }
};

__device__ __forceinline__ Share share_of(const AttendParams& p, const Item& it) {
  const int rows = it.un.q.nq * p.G - it.mt * kWideRows;
  return {rows <= kSub, it.last - it.first};
}

// ---- one tile of one query row ----------------------------------------------------------------------------------

__device__ __forceinline__ float max3(float a, float b, float c) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

struct SoftmaxTile {
  uint32_t s_at, o_at;   // this thread's scores and output in tensor memory
  int pos, limit;        // of the tile's first token, and of the first one the row does not see
  uint32_t missing;      // blocks of the tile that are not there
  int block_shift;
  float scale_log2, grow;
  bool later;            // the output holds earlier tiles
};

// Raises m to `top` in the lanes that ask for it and rescales l and the output to it; returns the new l. With the whole warp.
template <int D>
__device__ __forceinline__ float rescale(const SoftmaxTile& a, bool raise, float top, float& m, float l) {
  const float f = raise ? (m == -INFINITY ? 0.f : exp2_fast((m - top) * a.scale_log2)) : 1.f;
  if (raise) m = top;
  if (a.later) {
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      float o[32];
      tmem_ld32(o, a.o_at + c);
      tmem_wait_ld(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] *= f;
      tmem_st32(a.o_at + c, reinterpret_cast<const uint32_t*>(o));
    }
  }
  return l * f;  // the stores are waited for with the probabilities'
}

// A thread's row of 128 scores that the row sees: raises its running maximum m where it grew by more than `grow` (and then
// rescales its sum l and the output), writes the probabilities over the scores and adds them to l. Two scores to an
// instruction where the hardware has one. (One pass over the scores, against the maximum as it stood, with a second one
// only where it had grown, measured slower: its 64 packed probabilities and 64 scores crowd the registers.)
template <typename T, int D>
__device__ __forceinline__ void seen_softmax(const SoftmaxTile& a, float& m, float& l) {
  float s[2][32];
  auto fetch = [&](int c) { tmem_ld32(s[c & 1], a.s_at + 32 * c); };
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  fetch(0);
#pragma unroll
  for (int c = 0; c < 4; ++c) {  // chunk c + 1 is on its way while chunk c is worked on
    tmem_wait_ld(s[c & 1]);
    if (c < 3) fetch(c + 1);
#pragma unroll
    for (int i = 0; i < 16; ++i) mx[i & 3] = max3(mx[i & 3], s[c & 1][2 * i], s[c & 1][2 * i + 1]);
  }
  const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  const bool raise = top > m + a.grow;  // also a row's first scores: m is -inf
  if (__any_sync(kFullMask, raise)) l = rescale<D>(a, raise, top, m, l);
  const float from = m == -INFINITY ? 0.f : m * a.scale_log2;
  const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2), from2 = pair_of(-from, -from);
  uint64_t sum[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
  fetch(0);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tmem_wait_ld(s[c & 1]);
    if (c < 3) fetch(c + 1);
    uint32_t u[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x, y;
      split(fma_pair(pair_of(s[c & 1][2 * i], s[c & 1][2 * i + 1]), scale2, from2), x, y);
      if (i % 3 == 2) {  // 1024 query rows on 32768 tokens: 146 us with none of the pairs here, 139 with a third
        exp2_pair(x, y);
      } else {
        x = exp2_fast(x);
        y = exp2_fast(y);
      }
      sum[i & 1] = add_pair(sum[i & 1], pair_of(x, y));
      u[i] = pack2<T>(x, y);
    }
    tmem_st16(a.s_at + 16 * c, u);
  }
  float x, y;
  split(add_pair(sum[0], sum[1]), x, y);
  l += x + y;
}

// The same where the row does not see the whole tile. Not inlined: its registers would be the common case's too. Returns
// (m, l).
template <typename T, int D>
__device__ __noinline__ float2 full_softmax(const SoftmaxTile& a, float m, float l) {
  const bool masked = a.missing != 0 || a.pos + kTokens > a.limit;
  float s[32];
  auto fetch = [&](int c) {
    tmem_ld32(s, a.s_at + 32 * c);
    tmem_wait_ld(s);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (a.pos + 32 * c + i >= a.limit || (a.missing >> ((32 * c + i) >> a.block_shift) & 1u)) s[i] = -INFINITY;
    }
    __syncwarp();
  };
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    fetch(c);
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, s[i]);
  }
  const bool raise = top > m + a.grow;  // also a row's first scores: m is -inf
  if (__any_sync(kFullMask, raise)) l = rescale<D>(a, raise, top, m, l);
  const float from = m == -INFINITY ? 0.f : m * a.scale_log2;
  float sum[2] = {0.f, 0.f};
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    fetch(c);
    uint32_t u[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = exp2_fast(fmaf(s[2 * i], a.scale_log2, -from)), y = exp2_fast(fmaf(s[2 * i + 1], a.scale_log2, -from));
      sum[0] += x;
      sum[1] += y;
      u[i] = pack2<T>(x, y);
    }
    tmem_st16(a.s_at + 16 * c, u);  // over scores already read
  }
  tmem_wait_st();
  return make_float2(m, l + (sum[0] + sum[1]));
}

template <typename T, int D, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1) wide_kernel(const __grid_constant__ AttendParams p) {
  using R = Wide<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* queries = base;              // [2] subtiles
  uint8_t* ring = base + 2 * R::kSlot;  // [kSlots]
  WideTail<D>& tail = *reinterpret_cast<WideTail<D>*>(ring + R::kRing);
  const int units = PREFIX ? p.groups : p.rows;
  const int warp = __shfl_sync(kFullMask, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < R::kSlots; ++s) {
      mbar_init(&tail.full[s], 1);
      mbar_init(&tail.empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&tail.q_full[w], kSub);
      mbar_init(&tail.s_full[w], 1);
      mbar_init(&tail.p_ready[w], kSub);
      mbar_init(&tail.o_full[w], 1);
      mbar_init(&tail.o_free[w], kSub);
    }
    mbar_init(&tail.drained, 1);
    fence_mbar_init();
  }
  chain_wait();
  const Deal dealt = deal<PREFIX, kThreads, kTokens>(p, units, kWideRows, tail.scratch, tail.found);
  const int begin = dealt.begin, end = dealt.end;
  chain_release();
  if (begin >= end) return;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail.tmem)), "r"(kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tail.tmem;
  const int per_tile = kTokens >> p.block_shift;  // blocks of a tile
  Walk<PREFIX, kTokens> walk(p, dealt, units, kWideRows);
  bool good = true;  // after a wait that gave up a role goes on without waiting, so that every role ends

  if (warp == kCopyWarp) {
    const uint64_t policy = l2_evict_first_policy();
    const uint32_t block_bytes = (uint32_t)p.block_size * 128u;
    int slot = 0, issued = 0;
    uint32_t phase = 0;
    for (int t = begin; t < end && good;) {
      const Item it = walk.at(p, t, end);
      const int32_t* ids = p.table + (int64_t)it.un.row * p.table_s0;
      const int block0 = it.un.from >> p.block_shift, last_block = (it.un.to - 1) >> p.block_shift;
      const int tiles = it.last - it.first;
      auto copy = [&](int tile, bool values) {
        if (issued >= R::kSlots) good = good && mbar_wait_bounded(&tail.empty[slot], phase ^ 1, p.status);
        good = __all_sync(kFullMask, good);
        if (!good) return;
        if (lane == 0) mbar_arrive_expect_tx(&tail.full[slot], R::kSlot);
        __syncwarp();
        if (lane < per_tile) {
          const int b = block0 + (it.first + tile) * per_tile + lane;
          int id = b <= last_block ? ids[b] : -2;
          if (id < 0 || (int64_t)id >= p.pool_blocks) {
            if (b <= last_block) set_status(p.status, EKV_STATUS_BAD_BLOCK_ID);
            id = (int)p.pool_blocks;  // past the tensor: zeros
          }
          const uint32_t at = smem_u32(ring) + slot * R::kSlot + lane * block_bytes;
#pragma unroll
          for (int h = 0; h < R::kHalves; ++h)
            tensor_copy_4d(at + h * R::kHalf, values ? &p.vmap : &p.kmap, 64 * h, it.head, 0, id, &tail.full[slot], policy);
        }
        ++issued;
        if (++slot == R::kSlots) slot = 0, phase ^= 1;
      };
      copy(0, false);
      for (int tile = 0; tile < tiles; ++tile) {
        if (tile + 1 < tiles) copy(tile + 1, false);
        copy(tile, true);
      }
      t += tiles;
    }
    for (int s = 0; s < R::kSlots; ++s) {  // no CTA leaves with copies in flight
      const int uses = issued > s ? (issued - s - 1) / R::kSlots + 1 : 0;
      if (uses > 0) mbar_wait_bounded(&tail.full[s], (uses - 1) & 1, p.status);
    }
  } else if (warp == kMmaWarp) {
    constexpr uint32_t kScores = mma_shape<std::is_same<T, __half>::value>(kTokens, false);
    constexpr uint32_t kOutput = mma_shape<std::is_same<T, __half>::value>(D, true);
    const uint32_t q_at = smem_u32(queries), ring_at = smem_u32(ring);
    const uint32_t tm = __shfl_sync(kFullMask, tmem, 0);
    int slot = 0;
    uint32_t phase = 0;
    uint32_t q_uses[2] = {0, 0}, p_uses[2] = {0, 0}, items[2] = {0, 0};
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (good) good = mbar_wait_bounded(bar, parity, p.status);
      good = __all_sync(kFullMask, good);
      tc_fence_after();
    };
    // the next ring slot, waited for
    auto take = [&]() {
      const int s = slot;
      wait(&tail.full[s], phase);
      if (++slot == R::kSlots) slot = 0, phase ^= 1;
      return s;
    };
    const uint32_t q_low = operand_low(q_at, 16), ring_low = operand_low(ring_at, 16), value_low = operand_low(ring_at, R::kHalf);
    auto scores = [&](int w, int s) {
      if (!good || !elect_one()) return;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t at = ((uint32_t)(k >> 2) * R::kHalf + (uint32_t)(k & 3) * 32) >> 4;
        mma_ss(tm + w * 128, q_low + w * (R::kSlot >> 4) + at, ring_low + s * (R::kSlot >> 4) + at, kScores, k > 0);
      }
    };
    auto output = [&](int w, int s, bool add) {
      if (!good || !elect_one()) return;
#pragma unroll
      for (int k = 0; k < kTokens / 16; ++k)
        mma_ts(tm + 256 + w * 128, tm + w * 128 + 8 * k, value_low + s * (R::kSlot >> 4) + k * (2048 >> 4), kOutput, add || k > 0);
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) tc_commit(bar);
    };
    // rows of a value tile behind the unit's last token hold whatever the block holds: cleared, since a probability
    // of zero times that need not be zero
    auto clear_tail = [&](const Item& it, int tile, int s) {
      const int first = it.un.to - it.un.from - (it.first + tile) * kTokens;
      const int last = min(kTokens, (first + p.block_size - 1) >> p.block_shift << p.block_shift);
      if (first >= last) return;
      for (int i = lane; i < (last - first) * (D / 8); i += 32) {
        const int r = first + i / (D / 8), c = i % (D / 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring_at + s * R::kSlot + (c >> 3) * R::kHalf + r * 128 +
                                                                     (((c & 7) ^ (r & 7)) << 4)),
                     "r"(0)
                     : "memory");
      }
      proxy_fence_smem();
      __syncwarp();
    };
    for (int t = begin; t < end;) {
      const Item it = walk.at(p, t, end);
      const Share sh = share_of(p, it);
      int ks = take();
      if (sh.single) {
        for (int w = 0; w < 2 && w < sh.tiles; ++w) {
          if (w == 1) ks = take();
          wait(&tail.q_full[w], q_uses[w]++ & 1);
          scores(w, ks);
          commit(&tail.s_full[w]);
          commit(&tail.empty[ks]);
          // the tiles of this walk come as K0 K1 V0 K2 V1 ...: V0 stands before K2
        }
        for (int j = 0; j < sh.tiles; ++j) {
          const int w = j & 1;
          if (j > 0 && j + 1 < sh.tiles) {  // K(j + 1), taken before V(j): its scores wait for this warpgroup's turn
            ks = take();
          }
          const int vs = take();
          clear_tail(it, j, vs);
          // K(j + 1) belongs to the other warpgroup, whose P(j - 1) has been used: its scores can go first
          if (j > 0 && j + 1 < sh.tiles) {
            scores(w ^ 1, ks);
            commit(&tail.s_full[w ^ 1]);
            commit(&tail.empty[ks]);
          }
          wait(&tail.p_ready[w], p_uses[w]++ & 1);
          if (j < 2 && items[w] > 0) wait(&tail.o_free[w], (items[w] - 1) & 1);
          output(w, vs, j >= 2);
          commit(&tail.empty[vs]);
          if (j + 2 >= sh.tiles) commit(&tail.o_full[w]);
        }
      } else {
        for (int w = 0; w < 2; ++w) {
          wait(&tail.q_full[w], q_uses[w]++ & 1);
          scores(w, ks);
          commit(&tail.s_full[w]);
        }
        commit(&tail.empty[ks]);
        for (int j = 0; j < sh.tiles; ++j) {
          const bool more = j + 1 < sh.tiles;
          if (more) ks = take();
          const int vs = take();
          clear_tail(it, j, vs);
          for (int w = 0; w < 2; ++w) {
            wait(&tail.p_ready[w], p_uses[w]++ & 1);
            if (j == 0 && items[w] > 0) wait(&tail.o_free[w], (items[w] - 1) & 1);
            output(w, vs, j > 0);
            if (w == 1) commit(&tail.empty[vs]);
            if (more) {
              scores(w, ks);
              commit(&tail.s_full[w]);
            } else {
              commit(&tail.o_full[w]);
            }
          }
          if (more) commit(&tail.empty[ks]);
        }
      }
      for (int w = 0; w < 2; ++w) items[w] += sh.of(w) > 0;
      t += sh.tiles;
    }
    commit(&tail.drained);
    mbar_wait_bounded(&tail.drained, 0, p.status);
  } else {  // ---- the softmax warpgroups ---------------------------------------------------------------------
    const int w = warp >> 2, row = threadIdx.x & (kSub - 1);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
    const uint32_t s_at = tmem + w * 128 + lanes, o_at = tmem + 256 + w * 128 + lanes;
    uint32_t s_uses = 0, o_uses = 0;
    const float grow = fminf(8.f / p.scale_log2, 1e38f);  // finite: a row's first scores have to be above -inf + grow
    for (int t = begin; t < end;) {
      const Item it = walk.at(p, t, end);
      const Share sh = share_of(p, it);
      const QueryRange uq = it.un.q;
      const int mi = sh.single ? row : w * kSub + row, mrow = it.mt * kWideRows + mi;
      const bool real = mrow < uq.nq * p.G;
      const int token = uq.q0 + mrow / p.G, qhead = it.head * p.G + mrow % p.G;
      float m = -INFINITY, l = 0.f;
      if (sh.of(w) > 0) {
        // the warp's 32 query rows into the subtile's swizzled rows, D / 8 lanes a row
        const int64_t mine = real ? (int64_t)token * p.q_s0 + (int64_t)qhead * p.q_s1 : -1;
        uint4 v[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const int64_t source = __shfl_sync(kFullMask, mine, i * (256 / D) + lane / (D / 8));
          v[i] = source >= 0 ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + source + 8 * (lane % (D / 8)))
                             : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const int c = lane % (D / 8), at = (warp & 3) * 32 + i * (256 / D) + lane / (D / 8);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(queries) + w * R::kSlot + (c >> 3) * R::kHalf +
                                                                       at * 128 + (((c & 7) ^ (at & 7)) << 4)),
                       "r"(v[i].x), "r"(v[i].y), "r"(v[i].z), "r"(v[i].w)
                       : "memory");
        }
        proxy_fence_smem();
        mbar_arrive(&tail.q_full[w]);
        int limit = 0x7fffffff;
        if (real) limit = token_limit<PREFIX>(p, it.un, token);
        limit = min(limit, it.un.to);
        const int32_t* ids = p.table + (int64_t)it.un.row * p.table_s0;
        const int block0 = it.un.from >> p.block_shift, last_block = (it.un.to - 1) >> p.block_shift;
        const int step = sh.single ? 2 : 1;
        auto block_id = [&](int tile) {
          const int b = block0 + tile * per_tile + lane;
          return lane < per_tile && b <= last_block && tile < it.last ? ids[b] : 0;
        };
        int id = block_id(it.first + (sh.single ? w : 0));
        for (int tile = it.first + (sh.single ? w : 0); tile < it.last; tile += step) {
          const uint32_t missing = __ballot_sync(kFullMask, id < 0 || (int64_t)id >= p.pool_blocks);
          id = block_id(tile + step);
          if (good) good = mbar_wait_bounded(&tail.s_full[w], s_uses & 1, p.status);
          ++s_uses;
          tc_fence_after();
          __syncwarp();
          const int pos = it.un.from + tile * kTokens;
          const bool masked = missing != 0 || __any_sync(kFullMask, pos + kTokens > limit);
          const SoftmaxTile st{s_at, o_at, pos, limit, missing, p.block_shift, p.scale_log2, grow, tile >= it.first + step};
          if (!masked) {
            seen_softmax<T, D>(st, m, l);
          } else {
            const float2 ml = full_softmax<T, D>(st, m, l);
            m = ml.x;
            l = ml.y;
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&tail.p_ready[w]);
        }
        if (good) good = mbar_wait_bounded(&tail.o_full[w], o_uses & 1, p.status);
        ++o_uses;
        tc_fence_after();
      }
      const bool complete = it.first == 0 && it.last == it.tiles;
      const int64_t all = (int64_t)p.tokens * p.q_heads;
      float *dst, *ml;
      if (complete) {
        const int64_t at = (int64_t)token * p.q_heads + qhead + (sh.single && w == 1 ? all : 0);
        dst = p.whole + at * D;
        ml = p.whole + 2 * all * D + 2 * at;
      } else {
        const int64_t at = (int64_t)(2 * blockIdx.x + (it.first == 0 ? 1 : 0)) * kWideRows + w * kSub + row;
        dst = p.parts + at * D;
        ml = p.parts + (int64_t)2 * p.max_ctas * kWideRows * D + 2 * at;
      }
      if (real) *reinterpret_cast<float2*>(ml) = make_float2(m == -INFINITY ? m : m * p.scale_log2, l);
      if (sh.of(w) > 0) {
        // The output by way of the queries' shared memory, whose products are complete, so that a store covers whole lines
        // and not 16 bytes of each of 32 rows: 32 dims of the warp's rows at a time, a row's 16-byte pieces turned by its number.
        float* stage = reinterpret_cast<float*>(queries + w * R::kSlot + (warp & 3) * 4096);
        const int64_t to = real ? (int64_t)(dst - p.parts) : INT64_MIN;
        __syncwarp();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld32(o, o_at + c);
          tmem_wait_ld(o);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(stage + lane * 32 + 4 * (i ^ (lane & 7))) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3), k = lane & 7;
            const int64_t target = __shfl_sync(kFullMask, to, r);
            if (target != INT64_MIN)
              *reinterpret_cast<float4*>(p.parts + target + c + 4 * k) = *reinterpret_cast<const float4*>(stage + r * 32 + 4 * (k ^ (r & 7)));
          }
          __syncwarp();
        }
        tc_fence_before();
        mbar_arrive(&tail.o_free[w]);
      }
      t += sh.tiles;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
}

template <typename T, int D, bool PREFIX>
int launch(const AttendParams& p, int device, int sms, int* ctas, cudaStream_t s) {
  const size_t smem = 1024 + 2 * Wide<D>::kSlot + Wide<D>::kRing + (sizeof(WideTail<D>) + 15) / 16 * 16;
  auto kernel = wide_kernel<T, D, PREFIX>;
  static LaunchCache cache;
  int resident = 0;
  const int rc = prepare_launch(cache, kernel, "wide_kernel", device, kThreads, smem, &resident);
  if (rc != EKV_OK) return rc;
  *ctas = min(sms, p.max_ctas);
  launch_chained(kernel, dim3(*ctas), dim3(kThreads), smem, s, p);
  return check_launch("wide_kernel");
}

}  // namespace

template <bool PREFIX>
int launch_wide(const AttendParams& p, int dim, int dtype, int device, int sms, int* ctas, cudaStream_t s) {
  if (dtype == EKV_DTYPE_BF16)
    return dim == 128 ? launch<__nv_bfloat16, 128, PREFIX>(p, device, sms, ctas, s) : launch<__nv_bfloat16, 64, PREFIX>(p, device, sms, ctas, s);
  return dim == 128 ? launch<__half, 128, PREFIX>(p, device, sms, ctas, s) : launch<__half, 64, PREFIX>(p, device, sms, ctas, s);
}

template int launch_wide<true>(const AttendParams&, int, int, int, int, int*, cudaStream_t);
template int launch_wide<false>(const AttendParams&, int, int, int, int, int*, cudaStream_t);

}  // namespace ekv
