// The attention weight that cached tokens receive, accumulated per (row, KV head, token).
//
// Mathematics. Once the attention has left each query row's log-sum-exp, the weight of query row i on token t
// is p = exp(scale q_i.k_t - lse_i), so a token's weight w_t = sum_i p needs the keys alone and no second softmax:
// scores_t becomes w_t for a token with no score yet and decay * scores_t + w_t for the others.
//
// score_kernel walks tiles of 64 tokens as attend_kernel does (attend.cuh), keys only. A math warp takes 16 of the
// tile's tokens as the rows of mma.sync m16n8k16 and eight query rows as its columns, so a token's sum is two
// registers and two shuffles, in a fixed order; every token belongs to one CTA and nothing is added atomically.
#include "attend.cuh"

namespace ekv {

namespace {

constexpr int kMathWarps = 4;
constexpr int kThreads = (kMathWarps + 1) * 32;
constexpr int kOneTile = 1 << 30;  // query rows of an M tile: a unit's rows are all in one

struct ScoreParams {
  AttendParams a;
  float* scores;
  int64_t s0, s1;        // element strides between slots and between heads
  const int32_t* slots;  // or NULL: row r's slot is r
  const int32_t* fresh;  // or NULL: a row's query tokens
  int n_slots;
  float decay;
};

template <int D>
struct Ring {
  static constexpr int kHalves = D / 64;
  static constexpr int kStage = kHalves * kTile * 128;
  static constexpr int kStages = 5;
  static constexpr int kBytes = kStages * kStage;
};

template <int D>
struct Tail {
  uint64_t full[Ring<D>::kStages], empty[Ring<D>::kStages];
  uint32_t blocks[Ring<D>::kStages];
  int scratch[kThreads / 32 + 1];
};

__device__ __forceinline__ uint32_t chunk_at(int t, int c) {
  return (uint32_t)(c >> 3) * (kTile * 128) + (uint32_t)t * 128 + (uint32_t)((c & 7) ^ (t & 7)) * 16;
}

// The score row of batch row r, or -1: none is wanted, or the slot is not one row's alone.
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

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) score_kernel(const __grid_constant__ ScoreParams sp) {
  using R = Ring<D>;
  const AttendParams& p = sp.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Tail<D>& tail = *reinterpret_cast<Tail<D>*>(ring + R::kBytes);
  const Plan plan{reinterpret_cast<int*>(ring + R::kBytes + (sizeof(Tail<D>) + 15) / 16 * 16), p.rows};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&tail.full[s], 1);
      mbar_init(&tail.empty[s], kMathWarps);
    }
    fence_mbar_init();
  }
  chain_wait();  // the attention's log-sum-exps
  make_plan<false, kThreads>(p, plan, kOneTile, tail.scratch);
  chain_release();
  const int W = plan.cum[plan.units];
  const int n = sharing_ctas(W, gridDim.x);
  if ((int)blockIdx.x >= n || W == 0) return;
  const int begin = first_tile(blockIdx.x, W, n), end = first_tile(blockIdx.x + 1, W, n);
  const int per_tile = kTile >> p.block_shift;

  if (warp == kMathWarps) {  // ---- the copy warp --------------------------------------------------------
    const uint64_t policy = l2_evict_first_policy();
    const uint32_t block_bytes = (uint32_t)p.block_size * 128u;
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool good = true;
    for (int t = begin; t < end && good;) {
      const Item it = item_at<false>(p, plan, kOneTile, t, end);
      const int32_t* ids = p.table + (int64_t)it.un.row * p.table_s0;
      const int last_block = (it.un.to - 1) >> p.block_shift;
      const bool mine = lane < per_tile;
      int id = mine && lane + it.first * per_tile <= last_block ? ids[lane + it.first * per_tile] : -2;
      for (int tile = it.first; tile < it.last && good; ++tile, ++t) {
        const int b = lane + tile * per_tile;
        const int next = tile + 1 < it.last && mine && b + per_tile <= last_block ? ids[b + per_tile] : -2;
        if (issued >= R::kStages) good = mbar_wait_bounded(&tail.empty[stage], phase ^ 1, p.status);
        good = __all_sync(kFullMask, good);
        if (!good) break;
        const bool ok = mine && b <= last_block && id >= 0 && (int64_t)id < p.pool_blocks;
        const uint32_t which = __ballot_sync(kFullMask, ok);
        if (lane == 0) {
          tail.blocks[stage] = which;
          mbar_arrive_expect_tx(&tail.full[stage], (uint32_t)__popc(which) * block_bytes * R::kHalves);
        }
        __syncwarp();
        if (ok) {
          const uint32_t at = smem_u32(ring) + stage * R::kStage + lane * block_bytes;
#pragma unroll
          for (int h = 0; h < R::kHalves; ++h)
            tensor_copy_4d(at + h * (kTile * 128), &p.kmap, 64 * h, it.head, 0, id, &tail.full[stage], policy);
        }
        id = next;
        ++issued;
        if (++stage == R::kStages) stage = 0, phase ^= 1;
      }
    }
    for (int s = 0; s < R::kStages; ++s) {  // no CTA leaves with copies in flight
      const int uses = issued > s ? (issued - s - 1) / R::kStages + 1 : 0;
      if (uses > 0) mbar_wait_bounded(&tail.full[s], (uses - 1) & 1, p.status);
    }
    return;
  }

  // ---- the math warps ---------------------------------------------------------------------------------------
  const int quad = lane >> 2, pair = lane & 3;
  int stage = 0;
  uint32_t phase = 0;
  bool good = true;
  for (int t = begin; t < end;) {
    const Item it = item_at<false>(p, plan, kOneTile, t, end);
    const QueryRange uq = it.un.q;
    const int to = it.un.to, M = uq.nq * p.G;
    const int slot = slot_of(sp, it.unit, lane);
    const int fresh = sp.fresh != nullptr ? sp.fresh[it.unit] : uq.nq;
    const int old_end = to - max(fresh, 0);  // tokens from here on have no score yet
    float* dst = sp.scores + (int64_t)max(slot, 0) * sp.s0 + (int64_t)it.head * sp.s1;
    for (int tile = it.first; tile < it.last; ++tile, ++t) {
      if (good) good = mbar_wait_bounded(&tail.full[stage], phase, p.status);
      const uint32_t keys = smem_u32(ring) + stage * R::kStage;
      const uint32_t blocks = tail.blocks[stage];
      uint32_t kf[D / 16][4];
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        ldmatrix_x4(kf[k], keys + chunk_at(warp * 16 + (lane & 15), 2 * k + (lane >> 4)));
      __syncwarp();
      if (lane == 0) mbar_arrive(&tail.empty[stage]);  // the keys are in registers
      if (++stage == R::kStages) stage = 0, phase ^= 1;
      const int pos[2] = {tile * kTile + warp * 16 + quad, tile * kTile + warp * 16 + quad + 8};
      float w[2] = {0.f, 0.f};
      for (int m0 = 0; m0 < M; m0 += 8) {
        const int mq = m0 + quad;  // the query row of this lane's operand
        const bool real = mq < M;
        const T* src = static_cast<const T*>(p.q) + (int64_t)(uq.q0 + mq / p.G) * p.q_s0 +
                       (int64_t)(it.head * p.G + mq % p.G) * p.q_s1 + 2 * pair;
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t b[2] = {real ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u,
                                 real ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u};
          Mma<T>::run(c, kf[k], b);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // this lane's two result columns
          const int m = m0 + 2 * pair + e;
          if (m >= M) continue;
          const int i = m / p.G;
          const float lse = p.lse[(int64_t)(uq.q0 + i) * p.q_heads + it.head * p.G + (m - i * p.G)];
          if (lse == -INFINITY) continue;
          const float base = lse * 1.4426950408889634f;
          const int limit = to - uq.nq + i + 1;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (pos[j] < limit) w[j] += exp2_fast(fmaf(c[2 * j + e], p.scale_log2, -base));
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        w[j] += __shfl_xor_sync(kFullMask, w[j], 1);
        w[j] += __shfl_xor_sync(kFullMask, w[j], 2);
        const int tk = warp * 16 + quad + 8 * j;
        if (!((blocks >> (tk >> p.block_shift)) & 1u)) w[j] = 0.f;  // keys that were not read
        if (pair == 0 && slot >= 0 && pos[j] < to)
          dst[pos[j]] = pos[j] >= old_end || sp.decay == 0.f ? w[j] : fmaf(sp.decay, dst[pos[j]], w[j]);
      }
    }
  }
}

template <typename T, int D>
int launch_scores(const ScoreParams& p, int device, int sms, cudaStream_t s) {
  const size_t smem = 1024 + Ring<D>::kBytes + (sizeof(Tail<D>) + 15) / 16 * 16 + plan_bytes(p.a.rows);
  auto kernel = score_kernel<T, D>;
  static LaunchCache cache;
  int resident = 0;
  const int rc = prepare_launch(cache, kernel, "score_kernel", device, kThreads, smem, &resident);
  if (rc != EKV_OK) return rc;
  launch_chained(kernel, dim3(min(resident * sms, kAttendMaxCtas)), dim3(kThreads), smem, s, p);
  return check_launch("score_kernel");
}

}  // namespace

int launch_score_kernel(const AttendParams& a, int dim, int dtype, float* scores, int64_t s0, int64_t s1,
                        const int32_t* slots, const int32_t* fresh, int n_slots, float decay, int device, int sms, cudaStream_t s) {
  const ScoreParams p{a, scores, s0, s1, slots, fresh, n_slots, decay};
  if (dtype == EKV_DTYPE_BF16)
    return dim == 128 ? launch_scores<__nv_bfloat16, 128>(p, device, sms, s) : launch_scores<__nv_bfloat16, 64>(p, device, sms, s);
  return dim == 128 ? launch_scores<__half, 128>(p, device, sms, s) : launch_scores<__half, 64>(p, device, sms, s);
}

}  // namespace ekv
