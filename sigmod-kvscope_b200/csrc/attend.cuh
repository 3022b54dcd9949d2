// Shared parts of the attention kernels over the paged cache (attend.cu, attend_mma5.cu, attend_scores.cu): the launch
// parameters, what a unit of work is, and how the tiles of a launch are dealt out to its CTAs.
//
// Work. A unit is one row of the batch (its own tokens, behind its group's shared prefix), or, in a prefix
// launch, one group of rows (the tokens they share). A unit's M = query tokens x query heads per KV head
// query rows are cut into M tiles, its tokens into tiles of kTile; the launch's tiles, numbered unit by
// unit, KV head, M tile, token tile, are dealt evenly: CTA c of n takes tiles [c W / n, (c + 1) W / n). The units'
// running tile counts come from the lengths on the device, so no plan travels through the host: without
// groups every CTA adds them up itself (one level of loads), with groups a one-CTA kernel goes ahead, since what a
// row shares takes a chain of dependent loads that would otherwise stand at the start of every CTA of every launch.
//
// Parts. A CTA that covers a whole (unit, KV head, M tile) finishes it; one that covers some of its tiles
// leaves the part's running maximum, sum and unnormalised output in the workspace. A CTA has at most two
// such parts: one that starts where the item started earlier (slot 2c), one that ends before it (2c + 1).
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "ekv_common.cuh"

namespace ekv {

constexpr int kTile = 64;          // tokens of a tile
constexpr int kAttendMaxRows = 2048;
constexpr int kAttendMaxCtas = 512;

// Two values rounded to the cache's type, in one register.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

struct AttendParams {
  CUtensorMap kmap, vmap;  // the caches as (head dim, KV head, token of the block, block)
  const void* q;
  int64_t q_s0, q_s1;
  const int32_t* table;
  int64_t table_s0;
  const int32_t* lens;
  const int32_t* query_start;  // [rows + 1], or NULL: row r's one query token is token r
  void* out;
  int64_t out_s0, out_s1;
  float* lse;  // [tokens][q_heads], may be NULL
  float scale_log2;  // scale * log2(e): the kernels work in powers of two
  int rows, width, block_size, block_shift, heads, G, q_heads;
  int64_t pool_blocks;
  int tokens;
  int groups;                    // 0: nothing is shared
  const int32_t* group_start;    // [groups + 1], or NULL: one group of every row
  const int32_t* prefix_blocks;  // [groups], or NULL: prefix_common
  int prefix_common;
  uint32_t* status;
  float* logits;      // [tokens][q_heads][logits_s0] scores in powers of two, or NULL
  int64_t logits_s0;
  // the workspace. With groups, what plan_kernel leaves:
  int4* row_info;    // [rows] q0, nq, from, to
  int4* group_info;  // [groups] q0, nq, table row, to
  int32_t* row_group;  // [rows] or -1
  int32_t* limits;     // [tokens] the positions of its group's prefix that a query token sees
  // of the launch's phase:
  int32_t* cum;   // [units + 1] running tile counts
  float* parts;   // [2 CTAs][MT][D], and behind them their [2 CTAs][MT][2] maxima and sums
  float* whole;   // [tokens * q_heads][D] and [tokens * q_heads][2]: finished items when another phase joins (twice that
                  // in a wide launch, whose items of few query rows end in two halves)
  int follows;    // the launch before this one is the same call's prefix launch
  int item_each;  // a CTA an item, however long: nothing is left in parts, and no launch joins them
  int mt_rows;    // query rows of an M tile
  int max_ctas;
};

// ---- units -----------------------------------------------------------------------------------------

struct QueryRange {
  int q0, nq;
};

// Row r's query tokens; none when query_start does not describe tokens of the batch.
__device__ __forceinline__ QueryRange row_queries(const AttendParams& p, int r, bool report) {
  if (p.query_start == nullptr) return {r, r < p.tokens ? 1 : 0};
  const int a = p.query_start[r], b = p.query_start[r + 1];
  if (a < 0 || b < a || b > p.tokens) {
    if (report) set_status(p.status, EKV_STATUS_BAD_QROW);
    return {0, 0};
  }
  return {a, b - a};
}

// Row r's cached tokens, at most what its table holds.
__device__ __forceinline__ int row_tokens(const AttendParams& p, int r, bool report) {
  const int len = p.lens[r];
  const int most = p.width << p.block_shift;
  if (len > most) {
    if (report) set_status(p.status, EKV_STATUS_LEN_OVER_WIDTH);
    return most;
  }
  return len > 0 ? len : 0;
}

// ---- the plan ----------------------------------------------------------------------------------------

// A unit: its query tokens, the table row its blocks are in, and its positions [from, to).
struct Unit {
  QueryRange q;
  int row, from, to;
  __device__ __forceinline__ int m_tiles(const AttendParams& p, int MT) const { return (q.nq * p.G + MT - 1) / MT; }
  template <int TOKENS>
  __device__ __forceinline__ int tiles() const {
    return to > from && q.nq > 0 ? (to - from + TOKENS - 1) / TOKENS : 0;
  }
};

template <bool PREFIX>
__device__ __forceinline__ Unit unit_at(const AttendParams& p, int u, bool report) {
  if (PREFIX) {
    const int4 v = __ldcg(p.group_info + u);
    return {{v.x, v.y}, v.z, 0, v.w};
  }
  if (p.groups > 0) {
    const int4 v = __ldcg(p.row_info + u);  // from L2: a launch that follows another has not waited itself
    return {{v.x, v.y}, u, v.z, v.w};
  }
  return {row_queries(p, u, report), u, 0, row_tokens(p, u, report)};
}

// The positions that query token t of a unit sees end here.
template <bool PREFIX>
__device__ __forceinline__ int token_limit(const AttendParams& p, const Unit& un, int t) {
  return PREFIX ? p.limits[t] : un.to - un.q.nq + (t - un.q.q0) + 1;
}

// The tiles of CTA c when n CTAs share W, and the CTA that holds tile t.
__device__ __forceinline__ int first_tile(int c, int W, int n) { return (int)((int64_t)c * W / n); }
__device__ __forceinline__ int cta_of(int t, int W, int n) {  // floor(((t + 1) n - 1) / W), by an estimate put right
  const int64_t x = ((int64_t)t + 1) * n - 1;
  int c = (int)((float)x / (float)W);
  while ((int64_t)(c + 1) * W <= x) ++c;
  while ((int64_t)c * W > x) --c;
  return c;
}
__device__ __forceinline__ int sharing_ctas(int W, int ctas) { return W < ctas ? (W > 0 ? W : 1) : ctas; }

// A unit's tiles over all KV heads and M tiles.
template <int TOKENS>
__device__ __forceinline__ int unit_tiles(const AttendParams& p, const Unit& un, int MT) {
  return un.template tiles<TOKENS>() * p.heads * un.m_tiles(p, MT);
}

// Sums of tile counts. The host bounds a launch's tiles below 2^31 by its query tokens, which a query_start or group_start
// that descends gives to several units at once: such sums stop at kTooMany, and a launch that reaches it has no tiles.
constexpr int kTooMany = 0x7fffffff;
__device__ __forceinline__ int add_tiles(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kTooMany); }

// The units' tiles before this thread's, and of all of them.
template <int THREADS>
__device__ __forceinline__ int tiles_before(int mine, int* scratch, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto before = [&](int v) {  // of the lanes below
    int incl = v;
    for (int off = 1; off < 32; off <<= 1) {
      const int n = __shfl_up_sync(kFullMask, incl, off);
      if (lane >= off) incl = add_tiles(incl, n);
    }
    const int below = __shfl_up_sync(kFullMask, incl, 1);
    return make_int2(lane > 0 ? below : 0, incl);
  };
  const int2 in_warp = before(mine);
  __syncthreads();
  if (lane == 31) scratch[warp] = in_warp.y;
  __syncthreads();
  if (warp == 0) {
    const int2 warps = before(lane < THREADS / 32 ? scratch[lane] : 0);
    if (lane < THREADS / 32) scratch[lane] = warps.x;
    if (lane == THREADS / 32 - 1) scratch[THREADS / 32] = warps.y;
  }
  __syncthreads();
  *total = scratch[THREADS / 32];
  return add_tiles(scratch[warp], in_warp.x);
}

// What a CTA is dealt: tiles [begin, end) of W, the first of them in unit `unit`, whose tiles start at `base`.
struct Deal {
  int begin, end, W, unit, base;
};

// With every thread of the CTA (THREADS of them); scratch holds THREADS / 32 + 1 ints, found 2. Without groups CTA 0 also
// leaves the running counts for the combine kernel. With item_each, CTA c's tiles are all of item c's, and base is 0; an
// item without a tile has begin == end and its number in unit and base.
template <bool PREFIX, int THREADS, int TOKENS = kTile>
__device__ __forceinline__ Deal deal(const AttendParams& p, int units, int MT, int* scratch, int* found) {
  Deal d;
  const bool report = blockIdx.x == 0;
  if (!PREFIX && p.item_each) {  // at most THREADS units
    const int u = threadIdx.x;
    int items = 0, tiles = 0, total = 0;
    if (u < units) {
      const Unit un = unit_at<false>(p, u, report);
      items = p.heads * un.m_tiles(p, MT);
      tiles = un.template tiles<TOKENS>();
    }
    const int first = block_exclusive_scan<THREADS>(items, scratch, &total), c = blockIdx.x;
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    if (first <= c && c < first + items) {
      found[0] = u;
      found[1] = c - first;
      scratch[0] = tiles;
    }
    __syncthreads();
    d.unit = found[0];
    const int span = d.unit < 0 ? 0 : scratch[0];
    d.base = span > 0 ? 0 : found[1];
    d.begin = span > 0 ? found[1] * span : 0;
    d.end = d.begin + span;
    d.W = total;
    return d;
  }
  int mine = 0, before = 0;  // of the last THREADS units looked at
  if (PREFIX || p.groups > 0) {
    d.W = __ldcg(p.cum + units);
  } else {
    d.W = 0;
    for (int base = 0; base < units; base += THREADS) {
      const int u = base + threadIdx.x;
      mine = u < units ? unit_tiles<TOKENS>(p, unit_at<PREFIX>(p, u, report), MT) : 0;
      int total = 0;
      before = add_tiles(d.W, tiles_before<THREADS>(mine, scratch, &total));
      d.W = add_tiles(d.W, total);
    }
  }
  const bool too_many = d.W == kTooMany;
  if (too_many) {
    d.W = before = 0;
    if (report && threadIdx.x == 0) set_status(p.status, EKV_STATUS_BAD_QROW);
  }
  const int n = sharing_ctas(d.W, gridDim.x);
  if (threadIdx.x == 0) found[0] = found[1] = 0;
  __syncthreads();
  d.begin = (int)blockIdx.x < n ? first_tile(blockIdx.x, d.W, n) : d.W;
  d.end = (int)blockIdx.x < n ? first_tile(blockIdx.x + 1, d.W, n) : d.W;
  int carry = 0;
  for (int base = 0; base < units; base += THREADS) {
    const int u = base + threadIdx.x;
    if (PREFIX || p.groups > 0) {
      before = u < units ? __ldcg(p.cum + u) : d.W;
      mine = u < units ? __ldcg(p.cum + u + 1) - before : 0;
    } else if (units > THREADS) {
      mine = u < units ? unit_tiles<TOKENS>(p, unit_at<PREFIX>(p, u, false), MT) : 0;
      int total = 0;
      before = too_many ? 0 : carry + tiles_before<THREADS>(mine, scratch, &total);
      carry += total;
    }
    if (u < units && before <= d.begin && d.begin < before + mine) {  // one thread at most
      found[0] = u;
      found[1] = before;
    }
    if (!PREFIX && p.groups == 0 && report && p.cum != nullptr && u < units) p.cum[u] = before;
  }
  if (!PREFIX && p.groups == 0 && report && p.cum != nullptr && threadIdx.x == 0) p.cum[units] = d.W;
  __syncthreads();
  d.unit = found[0];
  d.base = found[1];
  return d;
}

// One item of a CTA's tiles: (unit, KV head, M tile) and its tiles [first, last) that the CTA covers.
struct Item {
  Unit un;
  int unit, head, mt, first, last, tiles;
};

// A warp's walk through the units from the one its CTA starts in, 32 of them in its lanes at a time, so that the next item
// costs a vote and some shuffles and not a chain of loads.
template <bool PREFIX, int TOKENS = kTile>
struct Walk {
  Unit un;           // this lane's unit
  int unit, start, count;
  int MT, units;
  __device__ __forceinline__ void load(const AttendParams& p, int first, int base) {
    unit = first + (int)(threadIdx.x & 31);
    un = Unit{{0, 0}, 0, 0, 0};
    if (unit < units) un = unit_at<PREFIX>(p, unit, false);
    count = unit_tiles<TOKENS>(p, un, MT);
    int incl = count;
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(kFullMask, incl, off);
      if ((int)(threadIdx.x & 31) >= off) incl += v;
    }
    start = base + incl - count;
  }
  __device__ __forceinline__ Walk(const AttendParams& p, const Deal& d, int units_, int MT_) : MT(MT_), units(units_) { load(p, d.unit, d.base); }
  // The item that tile t (at or past the one before's) starts or continues; with the whole warp.
  __device__ __forceinline__ Item at(const AttendParams& p, int t, int end) {
    uint32_t here;
    while ((here = __ballot_sync(kFullMask, start <= t && t < start + count)) == 0) {
      const int next = __shfl_sync(kFullMask, unit, 31) + 1, base = __shfl_sync(kFullMask, start + count, 31);
      if (next >= units) break;  // no tile is past the last unit
      load(p, next, base);
    }
    const int l = here ? __ffs(here) - 1 : 0;
    Item it;
    it.un.q.q0 = __shfl_sync(kFullMask, un.q.q0, l);
    it.un.q.nq = __shfl_sync(kFullMask, un.q.nq, l);
    it.un.row = __shfl_sync(kFullMask, un.row, l);
    it.un.from = __shfl_sync(kFullMask, un.from, l);
    it.un.to = __shfl_sync(kFullMask, un.to, l);
    it.unit = __shfl_sync(kFullMask, unit, l);
    it.tiles = max(it.un.template tiles<TOKENS>(), 1);
    const int mts = max(it.un.m_tiles(p, MT), 1);
    const int rem = t - __shfl_sync(kFullMask, start, l), hm = rem / it.tiles;
    it.head = hm / mts;
    it.mt = hm - it.head * mts;
    it.first = rem - hm * it.tiles;
    it.last = min(it.tiles, it.first + end - t);
    return it;
  }
};

// ---- copies ------------------------------------------------------------------------------------------------

__device__ __forceinline__ void tensor_copy_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                               uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void proxy_fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Whether `ok` holds for all `threads` that meet at the barrier.
__device__ __forceinline__ bool named_barrier_and(int id, int threads, bool ok) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(all)
               : "r"(id), "r"(threads), "r"((uint32_t)ok)
               : "memory");
  return all != 0;
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLn2 = 0.69314718055994531f;

// ---- host ---------------------------------------------------------------------------------------------------

// The CTAs of a kernel of one instantiation that an SM holds, by device; 0 until its shared memory, the same for every launch,
// has been asked for there (the attribute and occupancy calls cost microseconds).
struct LaunchCache {
  std::mutex lock;
  int resident[kMaxDevices] = {};
};

template <typename Kernel>
int prepare_launch(LaunchCache& cache, Kernel kernel, const char* name, int device, int threads, size_t smem, int* resident) {
  std::lock_guard<std::mutex> hold(cache.lock);
  if (cache.resident[device] == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return check_launch(name);
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) return check_launch(name);
    if (n < 1) return fail(EKV_ENOTSUP, "%s does not fit this device", name);
    cache.resident[device] = n;
  }
  *resident = cache.resident[device];
  return EKV_OK;
}

// Encodes p.kmap and p.vmap for a cache at `kv` ([blocks][2][block_size][heads][D], element strides).
int encode_cache_maps(AttendParams& p, const void* kv, int64_t s_block, int64_t s_part, int64_t s_pos, int64_t s_head,
                      int dim, int dtype);

// An attention launch on the tcgen05 tensor cores (attend_mma5.cu): M tiles of kWideRows query rows, one CTA an SM.
constexpr int kWideRows = 256;
constexpr int kWideMaxCtas = 160;
template <bool PREFIX>
int launch_wide(const AttendParams& p, int dim, int dtype, int device, int sms, int* ctas, cudaStream_t s);

// Adds each token's weight to its score after an attention launch that left a.lse (attend_scores.cu).
int launch_score_kernel(const AttendParams& a, int dim, int dtype, float* scores, int64_t s0, int64_t s1,
                        const int32_t* slots, const int32_t* fresh, int n_slots, float decay, int device, int sms, cudaStream_t s);

}  // namespace ekv
