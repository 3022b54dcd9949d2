// The attention weight that cached tokens receive, accumulated per (row, KV head, token).
//
// Mathematics. Once the attention has left each query row's log-sum-exp, the weight of query row i on token t
// is p = exp(scale q_i.k_t - lse_i), so a token's weight w_t = sum_i p needs no second softmax: scores_t becomes w_t for
// a token with no score yet and decay * scores_t + w_t for the others. Every token's sum is one thread's, in a fixed
// order; nothing is added atomically.
//
// Few query rows (decode): the attention kernel has left its logits, and add_kernel reads them back, 4 bytes a token
// and query row, mostly from L2. 64 rows of up to 4096 tokens, four query rows a KV head: the pass adds 20 us to the
// attention's 133; multiplying the keys again, as for windows, added 140.
//
// Many query rows (a window that scores a prompt): weigh_kernel multiplies the keys again, on the tcgen05 tensor cores with
// the roles turned: 128 tokens are the rows of the product and up to 256 query rows its columns, so a token is a lane of
// tensor memory, its thread reads the columns 32 at a time, takes their exponentials and adds them up in a register. Two
// warpgroups take alternate tiles. The exponentials bound it: 16 a clock and SM, 2048 clocks for 128 x 256 against 1024
// of the products. Four prompts of up to 16001 tokens, 256 query rows a KV head: 55 us, of which the exponentials are 29
// (992 us with mma.sync and the queries read from L1 for every tile).
#include <algorithm>
#include <type_traits>

#include "attend.cuh"
#include "mma5.cuh"

namespace ekv {

namespace {

struct ScoreParams {
  AttendParams a;
  float* scores;
  int64_t s0, s1;        // element strides between slots and between heads
  const int32_t* slots;  // or NULL: row r's slot is r
  const int32_t* fresh;  // or NULL: a row's query tokens
  int n_slots;
  float decay;
};

constexpr float kLog2e = 1.4426950408889634f;

// The score row of batch row r, or -1: none is wanted, or the slot is not one row's alone. With the whole warp.
__device__ __forceinline__ int slot_of(const ScoreParams& p, int r, int lane) {
  if (p.slots == nullptr) return r < p.n_slots ? r : -1;
  const int slot = p.slots[r];
  if (slot < 0) return -1;
  bool bad = slot >= p.n_slots;
  for (int i = lane; i < p.a.rows; i += 32) bad |= i != r && p.slots[i] == slot;
  bad = __any_sync(kFullMask, bad);
  if (bad) set_status(p.a.status, EKV_STATUS_BAD_SLOT);
  return bad ? -1 : slot;
}

// ---- from the attention's logits ---------------------------------------------------------------------------

constexpr int kAddThreads = 256;

// CTAs of a (row, KV head) take its tokens 4 a thread; a warp's 128 tokens are read from every query row in turn.
__global__ void __launch_bounds__(kAddThreads) add_kernel(const __grid_constant__ ScoreParams sp) {
  const AttendParams& p = sp.a;
  chain_release();
  chain_wait();  // the logits and the log-sum-exps
  const int row = blockIdx.x / p.heads, head = blockIdx.x - row * p.heads;
  const Unit un = unit_at<false>(p, row, false);
  const int M = un.q.nq * p.G;
  if (M == 0) return;
  const int slot = slot_of(sp, row, threadIdx.x & 31);
  if (slot < 0) return;
  const int fresh = sp.fresh != nullptr ? sp.fresh[row] : un.q.nq;
  const int old_end = un.to - max(fresh, 0);  // tokens from here on have no score yet
  float* dst = sp.scores + (int64_t)slot * sp.s0 + (int64_t)head * sp.s1;
  const float* first = p.logits + ((int64_t)un.q.q0 * p.q_heads + head * p.G) * p.logits_s0;
  const float* lses = p.lse + (int64_t)un.q.q0 * p.q_heads + head * p.G;
  const int32_t* ids = p.table + (int64_t)row * p.table_s0;
  for (int pos = 4 * (blockIdx.y * kAddThreads + threadIdx.x); pos < un.to; pos += 4 * gridDim.y * kAddThreads) {
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    int seen = 0;  // by query tokens whose log-sum-exp is no number
    for (int i = 0; i < un.q.nq; ++i) {
#pragma unroll 4
      for (int g = 0; g < p.G; ++g) {
        const float lse = lses[(int64_t)i * p.q_heads + g] * kLog2e;
        if (!(lse > -INFINITY)) {  // it saw nothing, or something that is no number
          if (lse != -INFINITY) seen = un.to - un.q.nq + i + 1;
          continue;
        }
        const float4 x = *reinterpret_cast<const float4*>(first + ((int64_t)i * p.q_heads + g) * p.logits_s0 + pos);
        w[0] += exp2_fast(x.x - lse);
        w[1] += exp2_fast(x.y - lse);
        w[2] += exp2_fast(x.z - lse);
        w[3] += exp2_fast(x.w - lse);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (pos + e >= seen) break;
      const int id = ids[(pos + e) >> p.block_shift];
      if (id >= 0 && (int64_t)id < p.pool_blocks) w[e] = NAN;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (pos + e < un.to)
        dst[pos + e] = pos + e >= old_end || sp.decay == 0.f ? w[e] : fmaf(sp.decay, dst[pos + e], w[e]);
  }
}

// ---- from the keys --------------------------------------------------------------------------------------------

constexpr int kOneTile = 1 << 30;  // query rows of an M tile of the plan: a unit's rows are all in one
constexpr int kTokens = 128;
constexpr int kColumns = 256;  // query rows at a time
constexpr int kThreads = 320;
constexpr int kCopyWarp = 8, kMmaWarp = 9;

template <int D>
struct Ring {
  static constexpr int kHalves = D / 64;
  static constexpr int kHalf = kTokens * 128;
  static constexpr int kSlot = kHalves * kHalf;
  static constexpr int kSlots = 4;
  static constexpr int kBytes = kSlots * kSlot;
  static constexpr int kQueryHalf = kColumns * 128;
  static constexpr int kQueries = kHalves * kQueryHalf;
};

template <int D>
struct Tail {
  uint64_t full[Ring<D>::kSlots], empty[Ring<D>::kSlots], q_full, s_full[2], s_free[2], drained;
  uint32_t tmem;
  int scratch[kThreads / 32 + 1], found[2];
  alignas(16) float lse[kColumns];  // minus it, in powers of two
  alignas(16) int limit[kColumns];
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) weigh_kernel(const __grid_constant__ ScoreParams sp) {
  using R = Ring<D>;
  const AttendParams& p = sp.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* queries = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = queries + R::kQueries;
  Tail<D>& tail = *reinterpret_cast<Tail<D>*>(ring + R::kBytes);
  const int units = p.rows;
  const int warp = __shfl_sync(kFullMask, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < R::kSlots; ++s) {
      mbar_init(&tail.full[s], 1);
      mbar_init(&tail.empty[s], 1);
    }
    mbar_init(&tail.q_full, 256);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&tail.s_full[w], 1);
      mbar_init(&tail.s_free[w], 128);
    }
    mbar_init(&tail.drained, 1);
    fence_mbar_init();
  }
  chain_wait();  // the attention's log-sum-exps
  const Deal dealt = deal<false, kThreads, kTokens>(p, units, kOneTile, tail.scratch, tail.found);
  const int begin = dealt.begin, end = dealt.end;
  chain_release();
  if (begin >= end) return;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tail.tmem;
  const int per_tile = kTokens >> p.block_shift;
  Walk<false, kTokens> walk(p, dealt, units, kOneTile);
  bool good = true;  // after a wait that gave up a role goes on without waiting, so that every role ends

  if (warp == kCopyWarp) {
    const uint64_t policy = l2_evict_first_policy();
    const uint32_t block_bytes = (uint32_t)p.block_size * 128u;
    int slot = 0, issued = 0;
    uint32_t phase = 0;
    for (int t = begin; t < end && good;) {
      const Item it = walk.at(p, t, end);
      const int32_t* ids = p.table + (int64_t)it.un.row * p.table_s0;
      const int last_block = (it.un.to - 1) >> p.block_shift;
      for (int m0 = 0; m0 < it.un.q.nq * p.G && good; m0 += kColumns) {
        for (int tile = it.first; tile < it.last; ++tile) {
          if (issued >= R::kSlots) good = mbar_wait_bounded(&tail.empty[slot], phase ^ 1, p.status);
          good = __all_sync(kFullMask, good);
          if (!good) break;
          if (lane == 0) mbar_arrive_expect_tx(&tail.full[slot], R::kSlot);
          __syncwarp();
          if (lane < per_tile) {
            const int b = tile * per_tile + lane;
            int id = b <= last_block ? ids[b] : -2;
            if (id < 0 || (int64_t)id >= p.pool_blocks) id = (int)p.pool_blocks;  // past the tensor: zeros
            const uint32_t at = smem_u32(ring) + slot * R::kSlot + lane * block_bytes;
#pragma unroll
            for (int h = 0; h < R::kHalves; ++h)
              tensor_copy_4d(at + h * R::kHalf, &p.kmap, 64 * h, it.head, 0, id, &tail.full[slot], policy);
          }
          ++issued;
          if (++slot == R::kSlots) slot = 0, phase ^= 1;
        }
      }
      t += it.last - it.first;
    }
    for (int s = 0; s < R::kSlots; ++s) {  // no CTA leaves with copies in flight
      const int uses = issued > s ? (issued - s - 1) / R::kSlots + 1 : 0;
      if (uses > 0) mbar_wait_bounded(&tail.full[s], (uses - 1) & 1, p.status);
    }
  } else if (warp == kMmaWarp) {
    const uint32_t tm = __shfl_sync(kFullMask, tmem, 0);
    const uint32_t q_low = operand_low(smem_u32(queries), 16), ring_low = operand_low(smem_u32(ring), 16);
    int slot = 0;
    uint32_t phase = 0, q_uses = 0, uses[2] = {0, 0};
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (good) good = mbar_wait_bounded(bar, parity, p.status);
      good = __all_sync(kFullMask, good);
      tc_fence_after();
    };
    for (int t = begin; t < end;) {
      const Item it = walk.at(p, t, end);
      const int M = it.un.q.nq * p.G;
      for (int m0 = 0; m0 < M; m0 += kColumns) {
        const uint32_t shape = mma_shape<std::is_same<T, __half>::value>((min(M - m0, kColumns) + 15) / 16 * 16, false);
        wait(&tail.q_full, q_uses++ & 1);
        for (int j = 0; j < it.last - it.first; ++j) {
          const int w = j & 1;
          wait(&tail.full[slot], phase);
          if (uses[w] > 0) wait(&tail.s_free[w], (uses[w] - 1) & 1);
          ++uses[w];
          if (good && elect_one()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_ss(tm + w * kColumns, ring_low + slot * (R::kSlot >> 4) + (((uint32_t)(k >> 2) * R::kHalf + (k & 3) * 32) >> 4),
                     q_low + (((uint32_t)(k >> 2) * R::kQueryHalf + (k & 3) * 32) >> 4), shape, k > 0);
          }
          if (elect_one()) tc_commit(&tail.s_full[w]);
          if (elect_one()) tc_commit(&tail.empty[slot]);
          if (++slot == R::kSlots) slot = 0, phase ^= 1;
        }
      }
      t += it.last - it.first;
    }
    if (elect_one()) tc_commit(&tail.drained);
    mbar_wait_bounded(&tail.drained, 0, p.status);
  } else {  // ---- the warpgroups that add ----------------------------------------------------------------------
    const int w = warp >> 2, token_lane = threadIdx.x & 127, column = threadIdx.x;  // column: the query row this thread loads
    const uint32_t s_at = tmem + w * kColumns + ((uint32_t)(warp & 3) << 21);
    const uint64_t scale2 = pair_of(p.scale_log2, p.scale_log2);
    uint32_t s_uses = 0;
    for (int t = begin; t < end;) {
      const Item it = walk.at(p, t, end);
      const QueryRange uq = it.un.q;
      const int to = it.un.to, M = uq.nq * p.G;
      const int slot = slot_of(sp, it.unit, lane);
      const int fresh = sp.fresh != nullptr ? sp.fresh[it.unit] : uq.nq;
      const int old_end = to - max(fresh, 0);  // tokens from here on have no score yet
      float* dst = sp.scores + (int64_t)max(slot, 0) * sp.s0 + (int64_t)it.head * sp.s1;
      const int32_t* ids = p.table + (int64_t)it.un.row * p.table_s0;
      const int last_block = (to - 1) >> p.block_shift;
      for (int m0 = 0; m0 < M; m0 += kColumns) {
        const int count = min(M - m0, kColumns), padded = (count + 15) / 16 * 16;
        named_barrier(1, 256);  // every product with the queries before is complete, and every read of their sums
        const int m = m0 + column, i = m / p.G, qhead = it.head * p.G + m - i * p.G;
        const bool real = column < count;
        const int64_t mine = real ? (int64_t)(uq.q0 + i) * p.q_s0 + (int64_t)qhead * p.q_s1 : -1;
        uint4 v[D / 8];
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {  // the warp's 32 query rows, D / 8 lanes a row
          const int64_t source = __shfl_sync(kFullMask, mine, k * (256 / D) + lane / (D / 8));
          v[k] = source >= 0 ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + source + 8 * (lane % (D / 8)))
                             : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          const int c = lane % (D / 8), at = warp * 32 + k * (256 / D) + lane / (D / 8);
          if (at < padded)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(queries) + (c >> 3) * R::kQueryHalf + at * 128 +
                                                                         (((c & 7) ^ (at & 7)) << 4)),
                         "r"(v[k].x), "r"(v[k].y), "r"(v[k].z), "r"(v[k].w)
                         : "memory");
        }
        if (column < padded) {
          const float lse = real ? p.lse[(int64_t)(uq.q0 + i) * p.q_heads + qhead] : -INFINITY;
          tail.lse[column] = lse == -INFINITY ? -INFINITY : -lse * kLog2e;  // no weight from a query that saw nothing
          tail.limit[column] = real ? to - uq.nq + i + 1 : 0;
        }
        proxy_fence_smem();
        mbar_arrive(&tail.q_full);
        named_barrier(1, 256);
        for (int tile = it.first + w; tile < it.last; tile += 2) {
          const int b = tile * per_tile + lane;
          const int id = lane < per_tile && b <= last_block ? ids[b] : 0;
          const uint32_t missing = __ballot_sync(kFullMask, id < 0 || (int64_t)id >= p.pool_blocks);
          if (good) good = mbar_wait_bounded(&tail.s_full[w], s_uses & 1, p.status);
          ++s_uses;
          tc_fence_after();
          __syncwarp();
          const int pos = tile * kTokens + token_lane;
          const bool inner = (tile + 1) * kTokens <= to - uq.nq + 1;  // every query token sees the whole tile
          uint64_t sums[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
          float sum = 0.f;
          float s[2][32];
          tmem_ld32(s[0], s_at);
          // 64 columns in turn through the two buffers: one chunk is on its way while the other is worked on
          for (int c0 = 0; c0 < count; c0 += 64) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int c = c0 + 32 * half;
              if (c >= count) break;
              tmem_wait_ld(s[half]);
              if (c + 32 < count) tmem_ld32(s[half ^ 1], s_at + c + 32);
              if (inner && c + 32 <= count) {
                const float4* lse = reinterpret_cast<const float4*>(tail.lse + c);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float4 v = lse[k];  // minus the log-sum-exps
                  float a, b, d, e;
                  split(fma_pair(pair_of(s[half][4 * k], s[half][4 * k + 1]), scale2, pair_of(v.x, v.y)), a, b);
                  split(fma_pair(pair_of(s[half][4 * k + 2], s[half][4 * k + 3]), scale2, pair_of(v.z, v.w)), d, e);
                  sums[0] = add_pair(sums[0], pair_of(exp2_fast(a), exp2_fast(b)));
                  sums[1] = add_pair(sums[1], pair_of(exp2_fast(d), exp2_fast(e)));
                }
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const int at = min(c + k, kColumns - 1);
                  const float v = exp2_fast(fmaf(s[half][k], p.scale_log2, tail.lse[at]));
                  if (c + k < count && pos < tail.limit[at]) sum += v;
                }
              }
            }
          }
          tc_fence_before();
          mbar_arrive(&tail.s_free[w]);
          float x, y;
          split(add_pair(sums[0], sums[1]), x, y);
          float weight = (x + y) + sum;
          if (missing >> (token_lane >> p.block_shift) & 1u) weight = 0.f;  // keys that were not read
          if (slot >= 0 && pos < to) {  // this thread's token in every round of query rows
            const float old = m0 > 0 ? dst[pos] : (pos >= old_end || sp.decay == 0.f ? 0.f : sp.decay * dst[pos]);
            dst[pos] = old + weight;
          }
        }
      }
      t += it.last - it.first;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename T, int D>
int launch_weigh(const ScoreParams& p, int device, int sms, cudaStream_t s) {
  const size_t smem = 1024 + Ring<D>::kQueries + Ring<D>::kBytes + (sizeof(Tail<D>) + 15) / 16 * 16;
  auto kernel = weigh_kernel<T, D>;
  static LaunchCache cache;
  int resident = 0;
  const int rc = prepare_launch(cache, kernel, "weigh_kernel", device, kThreads, std::max(smem, (size_t)120 * 1024), &resident);
  if (rc != EKV_OK) return rc;
  // more than half of an SM's shared memory: one CTA an SM, which takes all of its tensor memory
  launch_chained(kernel, dim3(sms), dim3(kThreads), std::max(smem, (size_t)120 * 1024), s, p);
  return check_launch("weigh_kernel");
}

}  // namespace

int launch_score_kernel(const AttendParams& a, int dim, int dtype, float* scores, int64_t s0, int64_t s1,
                        const int32_t* slots, const int32_t* fresh, int n_slots, float decay, int device, int sms, cudaStream_t s) {
  const ScoreParams p{a, scores, s0, s1, slots, fresh, n_slots, decay};
  if (a.logits != nullptr) {
    // about eight CTAs an SM, or one for every 4 KB of a row's logits
    const int64_t units = (int64_t)a.rows * a.heads, chunks = (a.logits_s0 + 4 * kAddThreads - 1) / (4 * kAddThreads);
    const int64_t spread = std::min(chunks, std::max<int64_t>(1, 8ll * sms / units));
    launch_chained(add_kernel, dim3((unsigned)units, (unsigned)std::min<int64_t>(spread, 65535)), dim3(kAddThreads), 0, s, p);
    return check_launch("add_kernel");
  }
  if (dtype == EKV_DTYPE_BF16)
    return dim == 128 ? launch_weigh<__nv_bfloat16, 128>(p, device, sms, s) : launch_weigh<__nv_bfloat16, 64>(p, device, sms, s);
  return dim == 128 ? launch_weigh<__half, 128>(p, device, sms, s) : launch_weigh<__half, 64>(p, device, sms, s);
}

}  // namespace ekv
