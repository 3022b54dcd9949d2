// Attention over the paged cache, prefixes that groups of rows share read once: out = softmax(scale q K^T) V
// and the log of each query's sum of exponentials.
//
// Mathematics. One pass over the keys: with x = scale log2(e) q.k, a running maximum m, sum
// l = sum 2^(x - m) and output o = sum 2^(x - m) v; when m grows to m', l and o are multiplied by 2^(m - m').
// Parts of a row (its group's prefix, its own tokens, tiles of different CTAs) join the same way, so a
// shared prefix is one launch whose query rows are those of every row of the group, and the two results meet
// in the combine kernel: out = sum_j 2^(m_j - m) o_j / sum_j 2^(m_j - m) l_j. A part that saw nothing has l = 0. m = -inf
// does not say so: the maxima pass over NaN, so a part whose scores are all NaN ends with it and l = NaN, which has to reach
// the row's sum, and through it the output and the log.
//
// attend_kernel. A CTA of four math warps and one copy warp walks its share of the launch's tiles (attend.cuh), two CTAs an
// SM. The copy warp reads block ids and asks the TMA engine for the tile's key and value rows of one KV head, a block's
// 64-dim half per copy in the 128-byte swizzle, into a ring of three stages, and hands each item with its query rows to
// the math warps behind the item's first copies. These stand WM along the query rows and WN along the tile's tokens:
// scores by mma.sync m16n8k16 with the query fragments in registers for a whole item, probabilities rounded to the cache's
// type (the two operands of a product have to be of one type) and multiplied with the values in the same registers; sums
// stay in float32 from the unrounded probabilities. In bfloat16 the output is then 0.0017 to 0.0019 of its size from the one in
// 64 bits, and 0.0023 behind 32768 shared tokens, where float32 probabilities and one rounding at the end leave 0.0016 to
// 0.0017. The WN warps join through shared memory at an item's end.
//
// What bounds it: HBM, up to 32 query rows a KV head (2 D M operations on 4 D bytes a token: mma.sync, at about half
// of tcgen05's rate, is 16 % busy at M = 4). 64 rows of up to 8192 tokens, 8 KV heads of 128: 259 us, 6.2 TB/s, 96 % of the
// measured copy rate; 256 rows of 512 tokens 100 us, 84 %, where items of eight tiles show their beginning and end (a
// chain of loads, about 2000 cycles of joining). 64 query rows a head: 264 us for 64 rows of 4096 tokens, 260 TFLOP/s.
// With every warp loading its own queries and its own item, and the joining in eight barriers of two rows each, 2048 rows
// of 64 tokens took 406 us; with the items handed over and a row's sums and place found once, 202 us.
#include <algorithm>
#include <type_traits>

#include "attend.cuh"

namespace ekv {

namespace {

constexpr int kMathWarps = 4;
constexpr int kThreads = (kMathWarps + 1) * 32;

template <int D>
struct Ring {
  static constexpr int kHalves = D / 64;
  static constexpr int kPart = kHalves * kTile * 128;  // bytes of a tile's keys, or values
  static constexpr int kStage = 2 * kPart;
  static constexpr int kStages = 3;
  static constexpr int kBytes = kStages * kStage;
};

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// Bytes from a part's start to 16-byte chunk c of token t's row (128-byte swizzle, 64-dim halves).
__device__ __forceinline__ uint32_t chunk_at(int t, int c) {
  return (uint32_t)(c >> 3) * (kTile * 128) + (uint32_t)t * 128 + (uint32_t)((c & 7) ^ (t & 7)) * 16;
}

// The shared memory behind the ring.
template <int D, int WM, int WN>
struct Tail {
  // query rows of each of the WM that join at a time: all where they fit beside two CTAs' rings, else a few
  static constexpr int kRows = WN == 1 ? 1 : D == 64 ? 16 : 4 / WM;
  uint64_t full[Ring<D>::kStages], empty[Ring<D>::kStages];
  uint64_t item_full, item_empty;
  uint32_t blocks[Ring<D>::kStages];  // which of the stage's blocks were copied (bit b: the tile's block b)
  int scratch[kThreads / 32 + 1], found[2];
  Item item;  // what the math warps take next
  float m[2][WN > 1 ? WN : 1][16 * WM], l[2][WN > 1 ? WN : 1][16 * WM];  // of one item and of the next
  float inverse[16 * WM];   // of a row's sum, or 1 where the part is not the row's last
  int64_t target[16 * WM];  // where a row's output goes, or -1
  alignas(16) float o[WN > 1 ? WM * WN * kRows : 1][WN > 1 ? D + 8 : 4];
  alignas(16) uint8_t queries[WN > 1 ? 16 * WM * D * 2 : 16];  // the item's query rows, in 16-byte pieces turned by the row
};

// Where piece c of query row r lies in the shared queries.
template <int D>
__device__ __forceinline__ uint32_t query_at(int r, int c) {
  return (uint32_t)r * (2 * D) + (uint32_t)((c & ~7) | ((c & 7) ^ (r & 7))) * 16;
}

// The output of an item with no tokens: its query rows saw nothing.
template <typename T, int D>
__device__ __noinline__ void empty_item(const AttendParams& p, int unit, int number, int MT) {
  const Unit un = unit_at<false>(p, unit, false);
  const int mts = un.m_tiles(p, MT), head = number / mts, m0 = (number - head * mts) * MT;
  for (int i = threadIdx.x; i < MT * (D / 2); i += kThreads) {
    const int mrow = m0 + i / (D / 2), c = i % (D / 2);
    if (mrow >= un.q.nq * p.G) break;
    const int64_t token = un.q.q0 + mrow / p.G, qhead = head * p.G + mrow % p.G;
    *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + token * p.out_s0 + qhead * p.out_s1 + 2 * c) = 0u;
    if (c == 0 && p.lse != nullptr) p.lse[token * p.q_heads + qhead] = -INFINITY;
  }
}

template <typename T, int D, int WM, int WN, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 2) attend_kernel(const __grid_constant__ AttendParams p) {
  using R = Ring<D>;
  using TailT = Tail<D, WM, WN>;
  constexpr int MT = 16 * WM;
  constexpr int kWarpTokens = kTile / WN;  // tokens of the tile a warp works on
  constexpr int kN = kWarpTokens / 8;      // its score fragments
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  TailT& tail = *reinterpret_cast<TailT*>(ring + R::kBytes);
  const int units = PREFIX ? p.groups : p.rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&tail.full[s], 1);
      mbar_init(&tail.empty[s], kMathWarps);
    }
    mbar_init(&tail.item_full, 64);  // every lane of the copy warp, and its copies of queries
    mbar_init(&tail.item_empty, kMathWarps);
    fence_mbar_init();
  }
  // The lengths, tables and caches may be the work of the launches before. A launch that follows a prefix launch
  // starts after that one has waited for them, reads nothing that it writes, and so runs beside its last CTAs; it
  // waits at its end, so that what follows finds both complete.
  if (!p.follows) chain_wait();
  const Deal dealt = deal<PREFIX, kThreads>(p, units, MT, tail.scratch, tail.found);
  const int begin = dealt.begin, end = dealt.end;
  chain_release();
  if (begin >= end) {
    if (p.follows) chain_wait();
    if (!PREFIX && p.item_each && dealt.unit >= 0) empty_item<T, D>(p, dealt.unit, dealt.base, MT);
    return;
  }
  const int per_tile = kTile >> p.block_shift;  // blocks of a tile

  if (warp == kMathWarps) {  // ---- the copy warp ------------------------------------------------------
    const uint64_t policy = l2_evict_first_policy();
    const uint32_t block_bytes = (uint32_t)p.block_size * 128u;
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool good = true;
    Walk<PREFIX> walk(p, dealt, units, MT);
    for (int t = begin, n_items = 0; t < end && good; ++n_items) {
      const Item it = walk.at(p, t, end);
      const int from = it.un.from, to = it.un.to;
      const int32_t* ids = p.table + (int64_t)it.un.row * p.table_s0;
      const int last_block = (to - 1) >> p.block_shift;
      const int block0 = (from >> p.block_shift) + lane;
      const bool mine = lane < per_tile;
      int id = mine && block0 + it.first * per_tile <= last_block ? ids[block0 + it.first * per_tile] : -2;
      for (int tile = it.first; tile < it.last && good; ++tile, ++t) {
        const int b = block0 + tile * per_tile;
        const int next = tile + 1 < it.last && mine && b + per_tile <= last_block ? ids[b + per_tile] : -2;
        if (issued >= R::kStages) good = mbar_wait_bounded(&tail.empty[stage], phase ^ 1, p.status);
        good = __all_sync(kFullMask, good);
        if (!good) break;
        const bool inside = mine && b <= last_block;
        const bool ok = inside && id >= 0 && (int64_t)id < p.pool_blocks;
        if (inside && !ok) set_status(p.status, EKV_STATUS_BAD_BLOCK_ID);
        const uint32_t which = __ballot_sync(kFullMask, ok);
        if (lane == 0) {
          tail.blocks[stage] = which;
          mbar_arrive_expect_tx(&tail.full[stage], (uint32_t)__popc(which) * block_bytes * 2 * R::kHalves);
        }
        __syncwarp();
        if (ok) {
          const uint32_t at = smem_u32(ring) + stage * R::kStage + lane * block_bytes;
#pragma unroll
          for (int h = 0; h < R::kHalves; ++h) {
            tensor_copy_4d(at + h * (kTile * 128), &p.kmap, 64 * h, it.head, 0, id, &tail.full[stage], policy);
            tensor_copy_4d(at + h * (kTile * 128) + R::kPart, &p.vmap, 64 * h, it.head, 0, id, &tail.full[stage], policy);
          }
        }
        id = next;
        ++issued;
        if (++stage == R::kStages) stage = 0, phase ^= 1;
        if (tile == it.first) {
          // The item for the math warps, behind its first tile's copies and when they have taken the one before: they find
          // it, and its queries, without a chain of loads of their own.
          if (n_items > 0) good = mbar_wait_bounded(&tail.item_empty, (n_items - 1) & 1, p.status);
          good = __all_sync(kFullMask, good);
          if (!good) break;
          if (lane == 0) tail.item = it;
          if constexpr (WN > 1) {
            constexpr int kStep = 256 / D;  // rows that the warp's 32 pieces cover
            const int piece = lane % (D / 8);
            int r = lane / (D / 8), i = (it.mt * MT + r) / p.G, g = it.mt * MT + r - i * p.G;
#pragma unroll 4
            for (; r < MT; r += kStep) {
              uint8_t* dst = tail.queries + query_at<D>(r, piece);
              if (i < it.un.q.nq)
                cp_async16(dst, static_cast<const T*>(p.q) + (int64_t)(it.un.q.q0 + i) * p.q_s0 +
                                    (int64_t)(it.head * p.G + g) * p.q_s1 + 8 * piece);
              else
                *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
              for (g += kStep; g >= p.G; g -= p.G) ++i;
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&tail.item_full)) : "memory");
          mbar_arrive(&tail.item_full);
        }
      }
    }
    // copies of queries that the math warps did not wait for have to land too
    asm volatile("cp.async.wait_all;" ::: "memory");
    // no CTA leaves with copies in flight: the last phase of every stage that was used has to be complete
    for (int s = 0; s < R::kStages; ++s) {
      const int uses = issued > s ? (issued - s - 1) / R::kStages + 1 : 0;
      if (uses > 0) mbar_wait_bounded(&tail.full[s], (uses - 1) & 1, p.status);
    }
    if (p.follows) chain_wait();
    return;
  }

  // ---- the math warps ------------------------------------------------------------------------------------
  const int wm = warp % WM, wn = warp / WM;
  const int quad = lane >> 2, pair = lane & 3;
  int stage = 0;
  uint32_t phase = 0;
  bool good = true;
  for (int t = begin, n_items = 0; t < end; ++n_items) {
    // after a wait that gave up the warps go on to the item's end without waiting, where their barriers are, and leave together
    if (good) good = mbar_wait_bounded(&tail.item_full, n_items & 1, p.status);
    good = named_barrier_and(2, kMathWarps * 32, good);
    if (!good) break;
    const Item it = tail.item;
    const QueryRange uq = it.un.q;
    const int from = it.un.from, to = it.un.to;
    // this lane's two query rows: the tokens they see, and their fragments
    uint32_t qf[D / 16][4];
    int limit[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int mrow = it.mt * MT + wm * 16 + quad + 8 * j;
      const int token = uq.q0 + mrow / p.G;
      const bool real = mrow < uq.nq * p.G;
      limit[j] = 0x7fffffff;
      if (real) limit[j] = token_limit<PREFIX>(p, it.un, token);
      if constexpr (WN == 1) {
        const T* src = static_cast<const T*>(p.q) + (int64_t)token * p.q_s0 +
                       (int64_t)(it.head * p.G + mrow % p.G) * p.q_s1 + 2 * pair;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[k][j] = real ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
          qf[k][j + 2] = real ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
        }
      }
    }
    if constexpr (WN > 1) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        ldmatrix_x4(qf[k], smem_u32(tail.queries) + query_at<D>(wm * 16 + (lane & 15), 2 * k + (lane >> 4)));
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&tail.item_empty);
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[d][j] = 0.f;

    for (int tile = it.first; tile < it.last; ++tile, ++t) {
      if (good) good = mbar_wait_bounded(&tail.full[stage], phase, p.status);
      const uint32_t keys = smem_u32(ring) + stage * R::kStage, values = keys + R::kPart;
      const uint32_t blocks = tail.blocks[stage];
      const int pos0 = from + tile * kTile + wn * kWarpTokens;  // position of this warp's first token
      float s[kN][4];
#pragma unroll
      for (int j = 0; j < kN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int j = 0; j < kN; j += 2) {
          uint32_t b[4];
          ldmatrix_x4(b, keys + chunk_at(wn * kWarpTokens + 8 * j + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
          const uint32_t b0[2] = {b[0], b[1]}, b1[2] = {b[2], b[3]};
          Mma<T>::run(s[j], qf[k], b0);
          Mma<T>::run(s[j + 1], qf[k], b1);
        }
      }
      const uint32_t all = per_tile == 32 ? ~0u : (1u << per_tile) - 1u;
      const bool whole = blocks == all && pos0 + kWarpTokens <= to;
      const bool seen = pos0 + kWarpTokens <= limit[0] && pos0 + kWarpTokens <= limit[1];
      if (!whole) {
        // rows of the stage that hold no token of the unit: their keys are masked below, their values cleared
        // (a probability of zero times what lies there need not be zero)
        for (int i = lane; i < kWarpTokens * (D / 8); i += 32) {
          const int tk = wn * kWarpTokens + i / (D / 8);
          if (from + tile * kTile + tk >= to || !((blocks >> (tk >> p.block_shift)) & 1u))
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + chunk_at(tk, i % (D / 8))), "r"(0)
                         : "memory");
        }
        __syncwarp();
      }
      if (!__all_sync(kFullMask, whole && seen)) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tk = wn * kWarpTokens + 8 * j + 2 * pair + (e & 1);
            const int pos = from + tile * kTile + tk;
            if (pos >= to || pos >= limit[e >> 1] || !((blocks >> (tk >> p.block_shift)) & 1u)) s[j][e] = -INFINITY;
          }
      }
      if constexpr (WM == 1 && !PREFIX) {
        if (p.logits != nullptr) {  // for the pass that adds up the tokens' weights
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int mrow = it.mt * MT + quad + 8 * j;
            if (mrow >= uq.nq * p.G) continue;
            float* dst = p.logits + ((int64_t)(uq.q0 + mrow / p.G) * p.q_heads + it.head * p.G + mrow % p.G) * p.logits_s0 + pos0 + 2 * pair;
#pragma unroll
            for (int i = 0; i < kN; ++i)
              *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(s[i][2 * j] * p.scale_log2, s[i][2 * j + 1] * p.scale_log2);
          }
        }
      }
      // the running maximum of each query row over this warp's tokens
      float mx[2] = {s[0][0], s[0][2]};
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        mx[0] = fmaxf(mx[0], fmaxf(s[j][0], s[j][1]));
        mx[1] = fmaxf(mx[1], fmaxf(s[j][2], s[j][3]));
      }
      float base[2];
      bool grew = false;
      float mn[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(kFullMask, mx[j], 1));
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(kFullMask, mx[j], 2));
        mn[j] = fmaxf(m[j], mx[j] * p.scale_log2);
        grew |= mn[j] > m[j];
      }
      if (__any_sync(kFullMask, grew)) {
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f[j] = mn[j] > m[j] ? exp2_fast(m[j] - mn[j]) : 1.f;  // 0 for a row's first keys
          l[j] *= f[j];
          m[j] = mn[j];
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][0] *= f[0];
          o[d][1] *= f[0];
          o[d][2] *= f[1];
          o[d][3] *= f[1];
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) base[j] = m[j] == -INFINITY ? 0.f : m[j];
      uint32_t pf[kN / 2][4];
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float a0 = exp2_fast(fmaf(s[j][0], p.scale_log2, -base[0]));
        const float a1 = exp2_fast(fmaf(s[j][1], p.scale_log2, -base[0]));
        const float a2 = exp2_fast(fmaf(s[j][2], p.scale_log2, -base[1]));
        const float a3 = exp2_fast(fmaf(s[j][3], p.scale_log2, -base[1]));
        l[0] += a0 + a1;
        l[1] += a2 + a3;
        pf[j / 2][(j & 1) * 2] = pack2<T>(a0, a1);
        pf[j / 2][(j & 1) * 2 + 1] = pack2<T>(a2, a3);
      }
#pragma unroll
      for (int k = 0; k < kN / 2; ++k) {
#pragma unroll
        for (int d = 0; d < D / 8; d += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, values + chunk_at(wn * kWarpTokens + 16 * k + (lane & 15), d + (lane >> 4)));
          const uint32_t b0[2] = {b[0], b[1]}, b1[2] = {b[2], b[3]};
          Mma<T>::run(o[d], pf[k], b0);
          Mma<T>::run(o[d + 1], pf[k], b1);
        }
      }
      if (!whole) proxy_fence_smem();  // the cleared rows before the copy that refills the stage
      __syncwarp();
      if (lane == 0) mbar_arrive(&tail.empty[stage]);
      if (++stage == R::kStages) stage = 0, phase ^= 1;
    }

    // ---- the item's end: the sums over the quad's lanes, then over the WN warps -----------------------------
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[j] += __shfl_xor_sync(kFullMask, l[j], 1);
      l[j] += __shfl_xor_sync(kFullMask, l[j], 2);
    }
    const bool complete = it.first == 0 && it.last == it.tiles;
    const bool final = complete && p.groups == 0;  // nothing else joins: the output itself
    // where row mrow's part goes: its dims, and its maximum and sum
    auto part_at = [&](int mrow, int token, int head, float*& dst, float*& ml) {
      if (complete) {
        const int64_t at = (int64_t)token * p.q_heads + head;
        dst = p.whole + at * D;
        ml = p.whole + (int64_t)p.tokens * p.q_heads * D + 2 * at;
      } else {
        const int64_t at = (int64_t)(2 * blockIdx.x + (it.first == 0 ? 1 : 0)) * MT + (mrow - it.mt * MT);
        dst = p.parts + at * D;
        ml = p.parts + (int64_t)2 * p.max_ctas * MT * D + 2 * at;
      }
    };
    if constexpr (WN > 1) {
      // The WN warps of a row join through shared memory in the warps' order: a thread a row finds the row's maximum, its sum
      // and its place; each warp scales its part to the maximum; then every thread adds four dims of a row and writes them, a
      // row's lanes side by side.
      constexpr int kRows = TailT::kRows;
      float(&ms)[WN][16 * WM] = tail.m[n_items & 1], (&ls)[WN][16 * WM] = tail.l[n_items & 1];
      if (pair == 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ms[wn][wm * 16 + quad + 8 * j] = m[j];
          ls[wn][wm * 16 + quad + 8 * j] = l[j];
        }
      }
      named_barrier(1, kMathWarps * 32);
      if (threadIdx.x < MT) {
        const int mrow = it.mt * MT + threadIdx.x;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < WN; ++w) top = fmaxf(top, ms[w][threadIdx.x]);
#pragma unroll
        for (int w = 0; w < WN; ++w)
          total += ls[w][threadIdx.x] == 0.f ? 0.f : ls[w][threadIdx.x] * exp2_fast(ms[w][threadIdx.x] - top);
        int64_t target = -1;
        if (mrow < uq.nq * p.G) {
          const int i = mrow / p.G, token = uq.q0 + i, head = it.head * p.G + mrow - i * p.G;
          if (final) {
            target = (int64_t)token * p.out_s0 + (int64_t)head * p.out_s1;
            if (p.lse != nullptr)
              p.lse[(int64_t)token * p.q_heads + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
          } else {
            float *dst, *ml;
            part_at(mrow, token, head, dst, ml);
            target = dst - p.parts;
            *reinterpret_cast<float2*>(ml) = make_float2(top, total);
          }
        }
        tail.target[threadIdx.x] = target;
        tail.inverse[threadIdx.x] = final ? (total == 0.f ? 0.f : 1.f / total) : 1.f;
      }
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WN; ++w) top = fmaxf(top, ms[w][wm * 16 + quad + 8 * j]);
        f[j] = l[j] == 0.f ? 0.f : exp2_fast(m[j] - top);
      }
      const int rows = min(16, uq.nq * p.G - it.mt * MT);  // of the first of the WM: the others have no more
#pragma unroll
      for (int round = 0; round < 16 / kRows; ++round) {
        if (round * kRows >= rows) break;
        if (round > 0) named_barrier(1, kMathWarps * 32);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if ((quad + 8 * j) / kRows != round) continue;
          float* dst = tail.o[(wm * WN + wn) * kRows + (quad + 8 * j) % kRows] + 2 * pair;
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            *reinterpret_cast<float2*>(dst + 8 * d) =
                f[j] == 0.f ? make_float2(0.f, 0.f) : make_float2(o[d][2 * j] * f[j], o[d][2 * j + 1] * f[j]);
        }
        named_barrier(1, kMathWarps * 32);
#pragma unroll
        for (int at = 0; at < kRows * D / 4; at += WN * 32) {
          const int i = at + wn * 32 + lane, r = i / (D / 4), c = i % (D / 4);  // a row of the round and four of its dims
          const int tile_row = wm * 16 + round * kRows + r;
          const int64_t target = r < kRows ? tail.target[tile_row] : -1;
          if (target < 0) continue;
          const float inv = tail.inverse[tile_row];
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WN; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(tail.o[(wm * WN + w) * kRows + r] + 4 * c);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
          }
          if (final) {  // a row that saw nothing has an inverse of 0
            uint2 v;
            v.x = inv == 0.f ? 0u : pack2<T>(sum.x * inv, sum.y * inv);
            v.y = inv == 0.f ? 0u : pack2<T>(sum.z * inv, sum.w * inv);
            *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + target + 4 * c) = v;
          } else {
            *reinterpret_cast<float4*>(p.parts + target + 4 * c) = sum;
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int mrow = it.mt * MT + wm * 16 + quad + 8 * j;
        if (mrow >= uq.nq * p.G) continue;
        const int token = uq.q0 + mrow / p.G, head = it.head * p.G + mrow % p.G;
        if (final) {
          const float inv = 1.f / l[j];
          T* dst = static_cast<T*>(p.out) + (int64_t)token * p.out_s0 + (int64_t)head * p.out_s1 + 2 * pair;
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            *reinterpret_cast<uint32_t*>(dst + 8 * d) = l[j] == 0.f ? 0u : pack2<T>(o[d][2 * j] * inv, o[d][2 * j + 1] * inv);
          if (p.lse != nullptr && pair == 0)
            p.lse[(int64_t)token * p.q_heads + head] = l[j] == 0.f ? -INFINITY : (m[j] + log2f(l[j])) * kLn2;
        } else {
          float *dst, *ml;
          part_at(mrow, token, head, dst, ml);
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            *reinterpret_cast<float2*>(dst + 8 * d + 2 * pair) = make_float2(o[d][2 * j], o[d][2 * j + 1]);
          if (pair == 0) *reinterpret_cast<float2*>(ml) = make_float2(m[j], l[j]);
        }
      }
    }
  }
  if (p.follows) chain_wait();
}

// ---- joining the parts ------------------------------------------------------------------------------------------

// A phase's plan and parts, as its launch left them.
struct PhaseOut {
  const int32_t* cum;
  const float* parts;
  const float* whole;
  int units, MT, max_ctas, ctas;
};

struct CombineParams {
  AttendParams p;
  PhaseOut own, prefix;
};

constexpr int kCombineThreads = 128;

// The parts of an M tile's query rows in one phase: those of a run of CTAs, or the one finished item. A wide launch leaves an
// item of at most kWideRows / 2 query rows in two halves, over alternate tiles.
struct PartList {
  const float *o, *ml;
  int count, halves;
  bool whole;
  int64_t first, rest, step, half;  // where the first CTA's part begins, the second's, one more, and the other half
};

__device__ __forceinline__ PartList list_parts(const AttendParams& p, const PhaseOut& ph, int unit, int nq, int mt, int head, int D) {
  PartList out{nullptr, nullptr, 0, 1, false, 0, 0, 0, 0};
  const int W = ph.cum[ph.units], start = ph.cum[unit], span = ph.cum[unit + 1] - start;
  const int mts = (nq * p.G + ph.MT - 1) / ph.MT;
  if (span == 0 || mts == 0) return out;
  const int n = sharing_ctas(W, ph.ctas);
  const int tiles = span / (mts * p.heads);
  const int a = start + (head * mts + mt) * tiles, b = a + tiles;
  const int c0 = cta_of(a, W, n), c1 = cta_of(b - 1, W, n);
  const int64_t all = (int64_t)p.tokens * p.q_heads;
  if (ph.MT == kWideRows && nq * p.G - mt * ph.MT <= kWideRows / 2) out.halves = 2;
  out.whole = c0 == c1;
  if (out.whole) {
    out.o = ph.whole;
    out.ml = ph.whole + all * (ph.MT == kWideRows ? 2 : 1) * D;
    out.count = 1;
    out.half = all;
  } else {
    out.o = ph.parts;
    out.ml = ph.parts + (int64_t)2 * ph.max_ctas * ph.MT * D;
    out.count = c1 - c0 + 1;
    out.first = (int64_t)(2 * c0 + 1) * ph.MT;
    out.rest = (int64_t)(2 * c0 + 2) * ph.MT;
    out.step = 2 * ph.MT;
    out.half = kWideRows / 2;
  }
  out.count *= out.halves;
  return out;
}

// Part i's row; `at`: the query row's place in an M tile's part, or among all query rows where the list is whole.
__device__ __forceinline__ int64_t part_row(const PartList& l, int i, int64_t at) {
  const int c = l.halves == 2 ? i >> 1 : i;
  return at + (c == 0 ? l.first : l.rest + (c - 1) * l.step) + (l.halves == 2 && (i & 1) ? l.half : 0);
}

// CTAs per (row, KV head), a warp for each `run` query rows in turn; every lane holds D / 32 dims. The parts are added in order.
template <typename T, int D>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const __grid_constant__ CombineParams c, int run) {
  const AttendParams& p = c.p;
  chain_release();
  chain_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x / p.heads, head = blockIdx.x - row * p.heads;
  const Unit un = unit_at<false>(p, row, false);
  const int group = p.groups > 0 ? p.row_group[row] : -1;
  const int4 gi = group >= 0 ? p.group_info[group] : make_int4(0, 0, 0, 0);
  const int M = un.q.nq * p.G, lead = (un.q.q0 - gi.x) * p.G;  // the group's query rows before this row's
  const int warps = gridDim.y * (kCombineThreads / 32), warp = blockIdx.y * (kCombineThreads / 32) + (threadIdx.x >> 5);
  PartList lists[2];
  lists[0].count = lists[1].count = 0;
  int have[2] = {-1, -1};
  int i = -1, g = 0;
  for (int m0 = warp * run, in_run = 0; m0 < M; in_run + 1 < run ? (++in_run, ++m0) : (in_run = 0, m0 += (warps - 1) * run + 1)) {
    if (in_run == 0) {
      i = m0 / p.G;
      g = m0 - i * p.G;
    } else if (++g == p.G) {
      g = 0;
      ++i;
    }
    const int token = un.q.q0 + i, qhead = head * p.G + g;
    const int64_t all = (int64_t)token * p.q_heads + qhead;
    const int own_mt = m0 / c.own.MT;
    if (own_mt != have[0]) lists[0] = list_parts(p, c.own, row, un.q.nq, have[0] = own_mt, head, D);
    if (group >= 0 && lead + m0 >= 0 && lead + m0 < gi.y * p.G) {
      const int prefix_mt = (lead + m0) / c.prefix.MT;
      if (prefix_mt != have[1]) lists[1] = list_parts(p, c.prefix, group, gi.y, have[1] = prefix_mt, head, D);
    } else {
      lists[1].count = 0;
      have[1] = -1;
      if (p.groups == 0 && lists[0].count == 1 && c.own.MT != kWideRows) continue;  // the attention kernel wrote it
    }
    const int64_t place[2] = {lists[0].whole ? all : m0 - own_mt * c.own.MT,
                              lists[1].whole ? all : lead + m0 - have[1] * c.prefix.MT};
    // Parts 32 at a time, a lane each for its maximum and sum; their outputs are asked for before those arrive (a part that
    // holds nothing has a factor of 0 and its loads are not used), eight at a time and the next eight beside them.
    const int total = lists[0].count + lists[1].count;
    float m = -INFINITY, l = 0.f, acc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) acc[d] = 0.f;
    for (int base = 0; base < total; base += 32) {
      const int j = base + lane, k = j < lists[0].count ? 0 : 1;
      const float* src = nullptr;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (j < total) {
        const int64_t at = part_row(lists[k], k == 0 ? j : j - lists[0].count, place[k]);
        src = lists[k].o + at * D;
        ml = *reinterpret_cast<const float2*>(lists[k].ml + 2 * at);
      }
      const int count = min(32, total - base);
      float o[2][8][D / 32];
      auto ask = [&](int i0, float(&to)[8][D / 32]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* from = reinterpret_cast<const float*>(__shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(src), i0 + i));
          if (i0 + i < count) {
            if constexpr (D == 128)
              *reinterpret_cast<float4*>(to[i]) = *reinterpret_cast<const float4*>(from + lane * 4);
            else
              *reinterpret_cast<float2*>(to[i]) = *reinterpret_cast<const float2*>(from + lane * 2);
          }
        }
      };
      ask(0, o[0]);
      float top = ml.x;
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
      top = fmaxf(top, m);
      const float f = ml.y == 0.f ? 0.f : exp2_fast(ml.x - top);
      const float keep = m == -INFINITY ? 0.f : exp2_fast(m - top);
      m = top;
      l = l * keep + f * ml.y;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) acc[d] *= keep;
      auto add = [&](int i0, const float(&from)[8][D / 32]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float fi = __shfl_sync(kFullMask, f, i0 + i);
          if (fi != 0.f) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d) acc[d] = fmaf(from[i][d], fi, acc[d]);
          }
        }
      };
#pragma unroll
      for (int i0 = 0; i0 < 32; i0 += 16) {
        if (i0 >= count) break;
        if (i0 + 8 < count) ask(i0 + 8, o[1]);
        add(i0, o[0]);
        if (i0 + 16 < count) ask(i0 + 16, o[0]);
        if (i0 + 8 < count) add(i0 + 8, o[1]);
      }
    }
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(kFullMask, l, off);
    const float inv = 1.f / l;
    T* dst = static_cast<T*>(p.out) + (int64_t)token * p.out_s0 + (int64_t)qhead * p.out_s1 + lane * (D / 32);
#pragma unroll
    for (int d = 0; d < D / 32; d += 2)
      *reinterpret_cast<uint32_t*>(dst + d) = l == 0.f ? 0u : pack2<T>(acc[d] * inv, acc[d + 1] * inv);
    if (p.lse != nullptr && lane == 0)
      p.lse[(int64_t)token * p.q_heads + qhead] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

// ---- the plan of a batch with groups ------------------------------------------------------------------------------

constexpr int kPlanThreads = 512;

struct PlanParams {
  AttendParams p;
  int32_t *cum_own, *cum_prefix;
  int mt_own, mt_prefix;
};

// Running sums of n over [0, units) into cum, with every thread; count(u) is unit u's tiles. Too many to be dealt are none.
template <typename Count>
__device__ __forceinline__ void running_sum(const AttendParams& p, int32_t* cum, int units, int* scratch, Count count) {
  int carry = 0;
  for (int base = 0; base < units; base += kPlanThreads) {
    const int u = base + threadIdx.x;
    int total = 0;
    const int n = u < units ? count(u) : 0;
    const int before = tiles_before<kPlanThreads>(n, scratch, &total);
    if (u < units) cum[u] = add_tiles(carry, before);
    carry = add_tiles(carry, total);
    __syncthreads();
  }
  if (carry == kTooMany) {
    for (int u = threadIdx.x; u < units; u += kPlanThreads) cum[u] = 0;
    if (threadIdx.x == 0) set_status(p.status, EKV_STATUS_BAD_QROW);
    carry = 0;
  }
  if (threadIdx.x == 0) cum[units] = carry;
}

// One CTA: what every row leaves to its group (whole blocks that it has, so that the prefix launch reads no position
// that no row of the group holds), each group's longest such part and the row it is read from, and both phases' counts.
// A row that has less than its group's longest part leaves it nothing and reads all of its tokens itself: to the prefix launch
// the values behind it would have a probability of zero, and zero times another row's NaN is not zero.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanParams pp) {
  const AttendParams& p = pp.p;
  extern __shared__ uint8_t s_plan[];
  unsigned long long* lead = reinterpret_cast<unsigned long long*>(s_plan);  // [groups] shared tokens << 32 | ~row
  int* starts = reinterpret_cast<int*>(lead + p.groups);                     // [groups + 1]
  int* blocks = starts + p.groups + 1;                                       // [groups]
  __shared__ int scratch[kPlanThreads / 32 + 1];
  const int lane = threadIdx.x & 31;
  chain_release();
  chain_wait();
  for (int g = threadIdx.x; g <= p.groups; g += kPlanThreads) {
    starts[g] = p.group_start == nullptr ? (g == 0 ? 0 : p.rows) : min(max(p.group_start[g], 0), p.rows);
    if (g < p.groups) {
      lead[g] = 0;
      blocks[g] = min(max(p.prefix_blocks != nullptr ? p.prefix_blocks[g] : p.prefix_common, 0), p.width);
    }
  }
  __syncthreads();
  bool more = false;
  for (int r = threadIdx.x; r < p.rows; r += kPlanThreads) {
    const QueryRange q = row_queries(p, r, true);
    const int to = row_tokens(p, r, true);
    int lo = 0, hi = p.groups;  // the last group that starts at or before r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= r) lo = mid; else hi = mid;
    }
    const bool in = r >= starts[lo] && r < starts[lo + 1];
    const int from = in ? min(blocks[lo] << p.block_shift, to >> p.block_shift << p.block_shift) : 0;
    if (in && q.nq > 0) atomicMax(lead + lo, (unsigned long long)(uint32_t)from << 32 | (uint32_t)~(uint32_t)r);
    p.row_info[r] = make_int4(q.q0, q.nq, from, to);
    p.row_group[r] = in ? lo : -1;
    more |= q.nq > 8;
  }
  more = __syncthreads_or(more);
  const int own_tokens = pp.mt_own == kWideRows ? 2 * kTile : kTile;
  running_sum(p, pp.cum_own, p.rows, scratch, [&](int r) {
    int4 v = p.row_info[r];  // this thread's own entries
    const int g = p.row_group[r], nq = v.y, to = v.w;
    if (g >= 0 && v.z < (int)(lead[g] >> 32)) {
      v.z = 0;
      p.row_info[r] = v;
      p.row_group[r] = -1;
    }
    for (int i = 0; i < min(nq, 8); ++i) p.limits[v.x + i] = min(to - nq + i + 1, v.z);
    return to > v.z && nq > 0 ? (to - v.z + own_tokens - 1) / own_tokens * p.heads * ((nq * p.G + pp.mt_own - 1) / pp.mt_own) : 0;
  });
  // rows of many query tokens: their limits by a warp
  for (int r = threadIdx.x >> 5; r < p.rows && more; r += kPlanThreads / 32) {
    const int4 v = p.row_info[r];
    for (int i = 8 + lane; i < v.y; i += 32) p.limits[v.x + i] = min(v.w - v.y + i + 1, v.z);
  }
  const int prefix_tokens = pp.mt_prefix == kWideRows ? 2 * kTile : kTile;
  running_sum(p, pp.cum_prefix, p.groups, scratch, [&](int g) {
    const int a = starts[g], b = starts[g + 1];
    const int to = b > a ? (int)(lead[g] >> 32) : 0, row = to > 0 ? (int)~(uint32_t)lead[g] : 0;
    // the query tokens of the rows [a, b), which follow one another
    int q0 = 0, nq = 0;
    if (b > a) {
      q0 = p.query_start == nullptr ? a : p.query_start[a];
      nq = (p.query_start == nullptr ? min(b, p.tokens) : p.query_start[b]) - q0;
      if (q0 < 0 || nq < 0 || nq > p.tokens - q0) q0 = nq = 0;
    }
    p.group_info[g] = make_int4(q0, nq, row, to);
    return to > 0 && nq > 0 ? (to + prefix_tokens - 1) / prefix_tokens * p.heads * ((nq * p.G + pp.mt_prefix - 1) / pp.mt_prefix) : 0;
  });
}

// ---- host ----------------------------------------------------------------------------------------------------------

struct Workspace {
  size_t cum[2], parts[2], whole[2], row_info, group_info, row_group, limits, logits, total;
};

int max_ctas(int mt) { return mt == kWideRows ? kWideMaxCtas : kAttendMaxCtas; }

// Phase 0: the rows' own tokens; phase 1: the shared prefixes.
Workspace workspace_layout(int rows, int tokens, int groups, int q_heads, int dim, const int (&mt)[2], int64_t logits) {
  Workspace w{};
  size_t at = 0;
  if (groups > 0) {
    w.row_info = at;
    at += round_up((size_t)rows * 16, 256);
    w.group_info = at;
    at += round_up((size_t)groups * 16, 256);
    w.row_group = at;
    at += round_up((size_t)rows * 4, 256);
    w.limits = at;
    at += round_up((size_t)tokens * 4, 256);
  }
  for (int k = 0; k < (groups > 0 ? 2 : 1); ++k) {
    w.cum[k] = at;
    at += round_up(((size_t)(k == 0 ? rows : groups) + 1) * 4, 256);
    w.parts[k] = at;
    at += round_up((size_t)2 * max_ctas(mt[k]) * mt[k] * (dim + 2) * 4, 256);
    w.whole[k] = at;
    if (groups > 0 || mt[k] == kWideRows)
      at += round_up((size_t)tokens * q_heads * (dim + 2) * 4 * (mt[k] == kWideRows ? 2 : 1), 256);
  }
  w.logits = at;
  w.total = at + round_up((size_t)logits * 4, 256);
  return w;
}

// Query rows of an M tile: the smallest variant that holds a unit's average in one tile. Above 64 the tcgen05 kernel, whose
// tensor cores are twice as fast and whose items cost some 10 us each to begin and end (queries in, 128 KB of sums out):
// from 12 of its 128-token tiles an item, as far as `span`, the most tokens that a unit's table row can hold, tells, and 500 tiles
// of 256 query rows and 128 dims in all. The lengths are on the device: behind a table far wider than its rows they are taken
// for long. (128 query rows, 8 heads, one prefix of 8000, 16000 and 32000 tokens: 52, 47 and 58 us there, 45, 58 and 86 us
// here; 64 rows of 1000 tokens, 256 query rows a head: 372 there, 297 here; of 4096: 502 there, 769 here.)
int pick_mt(int64_t tokens, int units, int G, int heads, int dim, int64_t span) {
  const int64_t m = (tokens + units - 1) / units * G;
  if (m <= 64) return m <= 16 ? 16 : m <= 32 ? 32 : 64;
  const int64_t tiles = (span + 2 * kTile - 1) / (2 * kTile), items = (int64_t)units * heads * ((m + kWideRows - 1) / kWideRows);
  return tiles >= 12 && items * tiles * std::min<int64_t>(m, kWideRows) * dim >= 500ll * kWideRows * 128 ? kWideRows : 64;
}

// The bytes for any `span`: where both variants may be picked, of the larger one.
size_t workspace_bytes(int rows, int tokens, int groups, int q_heads, int kv_heads, int dim, int64_t logits) {
  const int G = q_heads / kv_heads;
  size_t most = 0;
  for (int pick = 0; pick < 4; ++pick) {
    const int mt[2] = {pick_mt(tokens, rows, G, kv_heads, dim, pick & 1 ? 0x7fffffff : 0),
                       groups > 0 ? pick_mt(tokens, groups, G, kv_heads, dim, pick & 2 ? 0x7fffffff : 0) : 0};
    most = std::max(most, workspace_layout(rows, tokens, groups, q_heads, dim, mt, logits).total);
  }
  return most;
}

template <typename T, int D, int WM, int WN, bool PREFIX>
int launch_attend(const AttendParams& p, int device, int sms, int* ctas, cudaStream_t s) {
  const size_t smem = 1024 + Ring<D>::kBytes + (sizeof(Tail<D, WM, WN>) + 15) / 16 * 16;
  auto kernel = attend_kernel<T, D, WM, WN, PREFIX>;
  static LaunchCache cache;
  int resident = 0;
  const int rc = prepare_launch(cache, kernel, "attend_kernel", device, kThreads, smem, &resident);
  if (rc != EKV_OK) return rc;
  *ctas = p.item_each ? p.item_each : min(sms * resident, p.max_ctas);
  launch_chained(kernel, dim3(*ctas), dim3(kThreads), smem, s, p);
  return check_launch("attend_kernel");
}

template <typename T, int D, bool PREFIX>
int launch_phase(const AttendParams& p, int device, int sms, int* ctas, cudaStream_t s) {
  switch (p.mt_rows) {
    case 16: return launch_attend<T, D, 1, 4, PREFIX>(p, device, sms, ctas, s);
    case 32: return launch_attend<T, D, 2, 2, PREFIX>(p, device, sms, ctas, s);
    default: return launch_attend<T, D, 4, 1, PREFIX>(p, device, sms, ctas, s);
  }
}

// The CTAs of a launch that gives each item one, or 0 where the tiles are dealt evenly. Rows of at most 512 tokens in at
// most one item an SM: splitting their tiles over CTAs saves as much of the kernel as the launch that joins them takes (one
// row of 333 tokens: 10.4 us whole, 10.0 us split), and that launch costs the host 2.5 us more.
int whole_items(const AttendParams& p, int mt, int sms) {
  const int64_t items = ((int64_t)p.rows + (int64_t)p.tokens * p.G / mt) * p.heads;  // at most
  return p.groups == 0 && mt != kWideRows && (int64_t)p.width * p.block_size <= 8 * kTile && p.rows <= kThreads && items <= sms
             ? (int)items : 0;
}

template <typename T, int D>
int attend(AttendParams p, const Workspace& w, const int (&mt)[2], uint8_t* ws, int device, int sms, cudaStream_t s) {
  CombineParams c{};
  const int phases = p.groups > 0 ? 2 : 1;
  p.item_each = whole_items(p, mt[0], sms);
  const int type = std::is_same<T, __half>::value ? EKV_DTYPE_F16 : EKV_DTYPE_BF16;
  if (p.groups > 0) {
    p.row_info = reinterpret_cast<int4*>(ws + w.row_info);
    p.group_info = reinterpret_cast<int4*>(ws + w.group_info);
    p.row_group = reinterpret_cast<int32_t*>(ws + w.row_group);
    p.limits = reinterpret_cast<int32_t*>(ws + w.limits);
    const PlanParams plan{p, reinterpret_cast<int32_t*>(ws + w.cum[0]), reinterpret_cast<int32_t*>(ws + w.cum[1]), mt[0], mt[1]};
    launch_chained(plan_kernel, dim3(1), dim3(kPlanThreads), (size_t)p.groups * 16 + 16, s, plan);
    const int rc = check_launch("plan_kernel");
    if (rc != EKV_OK) return rc;
  }
  for (int k = phases - 1; k >= 0; --k) {  // the prefixes first
    p.mt_rows = mt[k];
    p.cum = reinterpret_cast<int32_t*>(ws + w.cum[k]);
    p.parts = reinterpret_cast<float*>(ws + w.parts[k]);
    p.whole = reinterpret_cast<float*>(ws + w.whole[k]);
    p.max_ctas = max_ctas(mt[k]);
    p.follows = k == 0 && phases == 2 && mt[0] != kWideRows;
    PhaseOut& out = k == 0 ? c.own : c.prefix;
    out = PhaseOut{p.cum, p.parts, p.whole, k == 0 ? p.rows : p.groups, mt[k], p.max_ctas, 0};
    int* ctas = &out.ctas;
    const int rc = mt[k] == kWideRows ? (k == 1 ? launch_wide<true>(p, D, type, device, sms, ctas, s)
                                                : launch_wide<false>(p, D, type, device, sms, ctas, s))
                   : k == 1 ? launch_phase<T, D, true>(p, device, sms, ctas, s)
                            : launch_phase<T, D, false>(p, device, sms, ctas, s);
    if (rc != EKV_OK) return rc;
  }
  if (p.item_each) return EKV_OK;
  c.p = p;
  // warps for a row's average of query rows, several rows each where there are many: an M tile's list is made once for them
  const int64_t average = std::max<int64_t>(1, (int64_t)p.tokens * p.G / p.rows);
  const int per = kCombineThreads / 32, run = average >= 128 ? 4 : average >= 32 ? 2 : 1;
  const int spread = (int)std::min<int64_t>(64, (average + per * run - 1) / (per * run));
  launch_chained(combine_kernel<T, D>, dim3(p.rows * p.heads, spread), dim3(kCombineThreads), 0, s, c, run);
  return check_launch("combine_kernel");
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return static_cast<PFN_cuTensorMapEncodeTiled_v12000>(nullptr);
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

}  // namespace

int encode_cache_maps(AttendParams& p, const void* kv, int64_t s_block, int64_t s_part, int64_t s_pos, int64_t s_head,
                      int dim, int dtype) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = map_encoder();
  if (encode == nullptr) return fail(EKV_ECUDA, "the driver does not provide cuTensorMapEncodeTiled");
  const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)p.heads, (cuuint64_t)p.block_size, (cuuint64_t)p.pool_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)s_head * 2, (cuuint64_t)s_pos * 2, (cuuint64_t)s_block * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)p.block_size, 1};
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  for (int part = 0; part < 2; ++part) {
    const CUresult r = encode(part == 0 ? &p.kmap : &p.vmap,
                              dtype == EKV_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                              const_cast<uint8_t*>(static_cast<const uint8_t*>(kv)) + part * s_part * 2, dims, strides, box,
                              unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
      return fail(EKV_ENOTSUP, "the cache (strides %lld, %lld, %lld elements) has no tensor map (CUresult %d)",
                  (long long)s_block, (long long)s_pos, (long long)s_head, (int)r);
  }
  return EKV_OK;
}

}  // namespace ekv

using namespace ekv;

namespace {

// The scores' row length where the attention keeps its logits for the pass over the weights, and how many floats that
// takes: for at most 16 query rows a KV head, whose logits (8 bytes of traffic a token and query row) cost less than
// the keys again (256); not beyond 1 GiB, which is a table far wider than its rows.
int64_t logits_row(int width, int block_size) { return ((int64_t)width * block_size + kTile - 1) / kTile * kTile; }
int64_t kept_logits(int tokens, int rows, int width, int block_size, int q_heads, int kv_heads) {
  const int64_t n = (int64_t)tokens * q_heads * logits_row(width, block_size);
  return pick_mt(tokens, rows, q_heads / kv_heads, kv_heads, 128, 0) == 16 && n <= (1ll << 28) ? n : 0;
}

// Whether [tokens][heads][dim] arrays of 2-byte elements share memory, as far as their first bytes and strides tell: apart as a
// whole, or by columns of a common row or of a common head.
bool share_memory(const void* a, int64_t a0, int64_t a1, const void* b, int64_t b0, int64_t b1, int tokens, int heads, int dim) {
  const int64_t from_a = (int64_t)(uintptr_t)a / 2, from_b = (int64_t)(uintptr_t)b / 2;
  const int64_t row_a = (heads - 1) * a1 + dim, row_b = (heads - 1) * b1 + dim;
  if (from_a + (tokens - 1) * a0 + row_a <= from_b || from_b + (tokens - 1) * b0 + row_b <= from_a) return false;
  auto apart = [&](int64_t period, int64_t size_a, int64_t size_b) {
    const int64_t d = ((from_b - from_a) % period + period) % period;
    return d >= size_a && period - d >= size_b;
  };
  if (a0 == b0 && a0 > 0 && apart(a0, row_a, row_b)) return false;
  return !(a0 == b0 && a1 == b1 && a1 > 0 && a0 % a1 == 0 && apart(a1, dim, dim));
}

struct AttendCall {
  AttendParams p;
  Workspace w;
  int mt[2];
  uint8_t* ws;
  int device, sms;
};

// The checks of ekv_attend and ekv_attend_scored; fills the call.
int prepare(AttendCall& c, const void* q, int64_t q_stride_token, int64_t q_stride_head, const void* kv,
            int64_t kv_stride_block, int64_t kv_stride_part, int64_t kv_stride_pos, int64_t kv_stride_head,
            int64_t pool_blocks, const int32_t* table, int64_t table_stride, const int32_t* lens,
            const int32_t* query_start, int tokens, int rows, int width, int block_size, int q_heads, int kv_heads,
            int head_dim, int dtype, float scale, int groups, const int32_t* group_start, const int32_t* prefix_blocks,
            int prefix_common, void* out, int64_t out_stride_token, int64_t out_stride_head, float* lse, void* workspace,
            size_t workspace_bytes, uint32_t* status, bool scored) {
  if (!q || !kv || !table || !lens || !out) return fail(EKV_EINVAL, "a required device pointer is NULL");
  if (rows <= 0 || tokens <= 0 || width <= 0 || pool_blocks <= 0)
    return fail(EKV_EINVAL, "rows, tokens, width and pool_blocks must be positive");
  if (rows > kAttendMaxRows) return fail(EKV_ENOTSUP, "%d rows: this build handles up to %d", rows, kAttendMaxRows);
  if (!query_start && tokens != rows)
    return fail(EKV_EINVAL, "%d query tokens for %d rows: without query_start every row has one", tokens, rows);
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
    return fail(EKV_EINVAL, "%d query heads do not divide over %d KV heads", q_heads, kv_heads);
  if (head_dim != 64 && head_dim != 128) return fail(EKV_ENOTSUP, "head_dim %d: this build has kernels for 64 and 128", head_dim);
  if (block_size != 8 && block_size != 16 && block_size != 32 && block_size != 64)
    return fail(EKV_ENOTSUP, "block_size %d: this build has kernels for 8, 16, 32 and 64", block_size);
  if (dtype != EKV_DTYPE_F16 && dtype != EKV_DTYPE_BF16) return fail(EKV_EINVAL, "unknown dtype %d", dtype);
  if (!(scale > 0.f) || scale > 3.4e38f) return fail(EKV_EINVAL, "the scale must be positive and finite");
  if (pool_blocks > 0x7fffffffll) return fail(EKV_ENOTSUP, "%lld blocks in the pool exceed 2^31 - 1", (long long)pool_blocks);
  if (table_stride < width) return fail(EKV_EINVAL, "the table's row stride is below the width");
  if (((uintptr_t)kv & 15) || (kv_stride_block & 7) || (kv_stride_part & 7) || (kv_stride_pos & 7) || (kv_stride_head & 7))
    return fail(EKV_EINVAL, "the cache must be 16-byte aligned with strides of whole 16-byte units");
  if (kv_stride_block <= 0 || kv_stride_pos <= 0 || kv_stride_head <= 0 || kv_stride_part < 0)
    return fail(EKV_EINVAL, "the cache's strides must be positive");
  if (((uintptr_t)q & 15) || (q_stride_token & 7) || (q_stride_head & 7))
    return fail(EKV_EINVAL, "the query must be 16-byte aligned with strides of whole 16-byte units");
  if (((uintptr_t)out & 15) || (out_stride_token & 7) || (out_stride_head & 7))
    return fail(EKV_EINVAL, "the output must be 16-byte aligned with strides of whole 16-byte units");
  if (groups < 0 || groups > rows) return fail(EKV_EINVAL, "%d groups of %d rows", groups, rows);
  if (groups > 1 && (!group_start || !prefix_blocks))
    return fail(EKV_EINVAL, "%d groups need group_start and prefix_blocks", groups);
  if (prefix_common < 0) return fail(EKV_EINVAL, "a prefix of %d blocks", prefix_common);
  const int64_t tiles = (int64_t)width * block_size / kTile + 1;
  const int G = q_heads / kv_heads;
  if ((int64_t)width * block_size > 0x7fffffffll - 4096 ||
      ((int64_t)rows + (int64_t)tokens * G / 16) * kv_heads * tiles > 0x7fffffffll)
    return fail(EKV_ENOTSUP, "a launch of more than 2^31 - 1 tiles (rows x heads x tokens)");
  if ((int64_t)tokens * q_heads > 0x7fffffffll / 4) return fail(EKV_ENOTSUP, "more than 2^29 query rows");
  const int64_t span = (int64_t)width * block_size;
  c.mt[0] = pick_mt(tokens, rows, G, kv_heads, head_dim, span);
  c.mt[1] = groups > 0 ? pick_mt(tokens, groups, G, kv_heads, head_dim, prefix_blocks ? span : std::min(span, (int64_t)prefix_common * block_size)) : 0;
  const int64_t logits = scored ? kept_logits(tokens, rows, width, block_size, q_heads, kv_heads) : 0;
  const Workspace& w = c.w = workspace_layout(rows, tokens, groups, q_heads, head_dim, c.mt, logits);
  if (!workspace || workspace_bytes < w.total || ((uintptr_t)workspace & 255))
    return fail(EKV_ERANGE, "the workspace must hold %zu bytes at a 256-byte boundary", w.total);
  if (scored && logits == 0 && share_memory(q, q_stride_token, q_stride_head, out, out_stride_token, out_stride_head, tokens, q_heads, head_dim))
    return fail(EKV_EINVAL, "the output must share no memory with the query, which is read again for the weights");
  int rc = current_device(&c.device);
  if (rc != EKV_OK) return rc;
  if ((rc = sm_count(c.device, &c.sms)) != EKV_OK) return rc;
  c.ws = static_cast<uint8_t*>(workspace);
  AttendParams& p = c.p;
  p.q = q; p.q_s0 = q_stride_token; p.q_s1 = q_stride_head;
  p.table = table; p.table_s0 = table_stride; p.lens = lens; p.query_start = query_start;
  p.out = out; p.out_s0 = out_stride_token; p.out_s1 = out_stride_head; p.lse = lse;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.rows = rows; p.width = width; p.block_size = block_size;
  p.block_shift = block_size == 8 ? 3 : block_size == 16 ? 4 : block_size == 32 ? 5 : 6;
  p.heads = kv_heads; p.G = G; p.q_heads = q_heads; p.pool_blocks = pool_blocks; p.tokens = tokens;
  p.groups = groups; p.group_start = group_start; p.prefix_blocks = prefix_blocks; p.prefix_common = prefix_common;
  p.status = status;
  if (logits > 0) {
    p.logits = reinterpret_cast<float*>(c.ws + w.logits);
    p.logits_s0 = logits_row(width, block_size);
  }
  return encode_cache_maps(p, kv, kv_stride_block, kv_stride_part, kv_stride_pos, kv_stride_head, head_dim, dtype);
}

int run(const AttendCall& c, int head_dim, int dtype, cudaStream_t s) {
  if (dtype == EKV_DTYPE_BF16)
    return head_dim == 128 ? attend<__nv_bfloat16, 128>(c.p, c.w, c.mt, c.ws, c.device, c.sms, s)
                           : attend<__nv_bfloat16, 64>(c.p, c.w, c.mt, c.ws, c.device, c.sms, s);
  return head_dim == 128 ? attend<__half, 128>(c.p, c.w, c.mt, c.ws, c.device, c.sms, s)
                         : attend<__half, 64>(c.p, c.w, c.mt, c.ws, c.device, c.sms, s);
}

}  // namespace

extern "C" size_t ekv_attend_workspace_bytes(int rows, int tokens, int groups, int q_heads, int kv_heads, int head_dim) {
  if (rows <= 0 || tokens <= 0 || groups < 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_heads % kv_heads) return 0;
  return workspace_bytes(rows, tokens, groups, q_heads, kv_heads, head_dim, 0);
}

extern "C" size_t ekv_attend_scored_workspace_bytes(int rows, int tokens, int width, int block_size, int q_heads, int kv_heads,
                                                    int head_dim) {
  if (rows <= 0 || tokens <= 0 || width <= 0 || block_size <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_heads % kv_heads)
    return 0;
  return workspace_bytes(rows, tokens, 0, q_heads, kv_heads, head_dim, kept_logits(tokens, rows, width, block_size, q_heads, kv_heads));
}

extern "C" int ekv_attend(const void* q, int64_t q_stride_token, int64_t q_stride_head, const void* kv,
                          int64_t kv_stride_block, int64_t kv_stride_part, int64_t kv_stride_pos, int64_t kv_stride_head,
                          int64_t pool_blocks, const int32_t* table, int64_t table_stride, const int32_t* lens,
                          const int32_t* query_start, int tokens, int rows, int width, int block_size, int q_heads,
                          int kv_heads, int head_dim, int dtype, float scale, int groups, const int32_t* group_start,
                          const int32_t* prefix_blocks, int prefix_common, void* out, int64_t out_stride_token,
                          int64_t out_stride_head, float* lse, void* workspace, size_t workspace_bytes, uint32_t* status,
                          void* stream) {
  clear_error();
  AttendCall c{};
  const int rc = prepare(c, q, q_stride_token, q_stride_head, kv, kv_stride_block, kv_stride_part, kv_stride_pos,
                         kv_stride_head, pool_blocks, table, table_stride, lens, query_start, tokens, rows, width, block_size,
                         q_heads, kv_heads, head_dim, dtype, scale, groups, group_start, prefix_blocks, prefix_common, out,
                         out_stride_token, out_stride_head, lse, workspace, workspace_bytes, status, false);
  return rc != EKV_OK ? rc : run(c, head_dim, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int ekv_attend_scored(const void* q, int64_t q_stride_token, int64_t q_stride_head, const void* kv,
                                 int64_t kv_stride_block, int64_t kv_stride_part, int64_t kv_stride_pos,
                                 int64_t kv_stride_head, int64_t pool_blocks, const int32_t* table, int64_t table_stride,
                                 const int32_t* lens, const int32_t* query_start, int tokens, int rows, int width,
                                 int block_size, int q_heads, int kv_heads, int head_dim, int dtype, float scale,
                                 float* scores, int64_t score_stride_slot, int64_t score_stride_head, int n_slots,
                                 const int32_t* slots, const int32_t* fresh, float decay, void* out,
                                 int64_t out_stride_token, int64_t out_stride_head, float* lse, void* workspace,
                                 size_t workspace_bytes, uint32_t* status, void* stream) {
  clear_error();
  if (!scores || !lse) return fail(EKV_EINVAL, "a required device pointer is NULL");
  const int64_t most = (int64_t)width * block_size;
  if (n_slots <= 0 || (kv_heads > 1 && score_stride_head < most) || (n_slots > 1 && score_stride_slot < most))
    return fail(EKV_EINVAL, "scores must hold at least width * block_size tokens for every slot and head");
  if (!slots && n_slots < rows) return fail(EKV_EINVAL, "%d score slots for %d rows", n_slots, rows);
  if (!(decay >= 0.f && decay <= 1.f)) return fail(EKV_EINVAL, "the decay must lie in [0, 1]");
  AttendCall c{};
  int rc = prepare(c, q, q_stride_token, q_stride_head, kv, kv_stride_block, kv_stride_part, kv_stride_pos, kv_stride_head,
                   pool_blocks, table, table_stride, lens, query_start, tokens, rows, width, block_size, q_heads, kv_heads,
                   head_dim, dtype, scale, 0, nullptr, nullptr, 0, out, out_stride_token, out_stride_head, lse, workspace,
                   workspace_bytes, status, true);
  if (rc != EKV_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = run(c, head_dim, dtype, s);
  if (rc != EKV_OK) return rc;
  return launch_score_kernel(c.p, head_dim, dtype, scores, score_stride_slot, score_stride_head, slots, fresh, n_slots,
                             decay, c.device, c.sms, s);
}
