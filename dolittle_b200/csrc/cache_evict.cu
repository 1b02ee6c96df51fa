// Eviction from KV caches by accumulated attention weight (see
// dl_cache_evict in the public header for the definition).
//
// Two launches.  evict_select_kernel: one cluster of 1-8 CTAs per (cache, KV
// head) orders the slots by a 32-bit key (protected highest, then the weight's
// order-preserving bits, NaN lowest), finds the budget-th largest key by radix
// selection over 11-, 11- and 10-bit digits, and ranks ties, vacated slots
// ("holes", below the kept count) and kept slots beyond it ("movers") with
// prefix sums in slot order; hole i receives mover i.  evict_move_kernel
// copies the rows of the resulting (destination, source) list.  Sources lie
// at or above the kept count and destinations below it, so moving in place
// needs no order between rows.  Counts and integer prefix sums only: results
// do not depend on scheduling.
#include <algorithm>
#include <climits>

#include "cache_evict.h"
#include "tcgen05.cuh"

namespace dl {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;
constexpr int kMaxCached = 40 * 1024;  // keys held in shared memory per CTA

// dst, src and mover lists of one unit, then the entry count of every unit.
__host__ __device__ __forceinline__ int* list_of(int* ws, int unit, int budget) { return ws + size_t(unit) * 3 * budget; }

// Exclusive prefix sum over the CTA; *total receives the sum.  `warp_sums`
// is shared memory of 33 values.  All threads call.
template <class T>
__device__ __forceinline__ T block_scan(T v, T* warp_sums, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    T s = warp_sums[lane], e = s;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const T y = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) e += y;
    }
    warp_sums[lane] = e - s;
    if (lane == 31) warp_sums[32] = e;
  }
  __syncthreads();
  const T r = warp_sums[warp] + x - v;
  *total = warp_sums[32];
  __syncthreads();
  return r;
}

__device__ __forceinline__ unsigned remote_u32(const unsigned* p, unsigned rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(tc::mapa_shared(smem_addr(p), rank)) : "memory");
  return v;
}

// Sum of *p over the cluster's CTAs before this one; *total over all.
__device__ __forceinline__ unsigned cluster_offset(const unsigned* p, unsigned rank, unsigned ctas, unsigned* total) {
  unsigned before = 0, all = 0;
  for (unsigned r = 0; r < ctas; ++r) {
    const unsigned v = remote_u32(p, r);
    before += r < rank ? v : 0;
    all += v;
  }
  *total = all;
  return before;
}

// Larger = kept first.  -0 counts as +0, NaN below -infinity.
__device__ __forceinline__ unsigned slot_key(float w, int position, int first, long long recent_from) {
  if (position < first || position > recent_from) return 0xffffffffu;
  if (w != w) return 0u;
  const unsigned b = __float_as_uint(w + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs a, int* ws, int cached_max) {
  extern __shared__ unsigned cached[];
  __shared__ unsigned hist[3][kBins];
  __shared__ unsigned scan_u[33], found[2], tie_total, hole_total, mover_total, newest_s;
  __shared__ unsigned long long scan_l[33];
  const unsigned ctas = gridDim.x / (a.caches * a.kv_heads), rank = tc::cluster_ctarank();
  const int unit = blockIdx.x / ctas, cache = unit / a.kv_heads, t = threadIdx.x;
  allow_next();
  wait_prior();
  const long long len = a.lengths[cache];
  const int n = int(len < 0 ? 0 : len > a.capacity ? a.capacity : len);
  const int keep = min(n, a.budget);
  const int chunk = (n + ctas - 1) / ctas;
  const int s0 = min(n, int(rank) * chunk), s1 = min(n, s0 + chunk);
  const float* weights = a.weights + size_t(unit) * a.capacity;
  const int* positions = a.positions + size_t(unit) * a.capacity;
  const bool all = n <= a.budget;  // nothing is evicted
  const bool use_cache = chunk <= cached_max;
  auto sync = [&] {
    if (ctas > 1) tc::cluster_sync();
    else __syncthreads();
  };

  long long recent_from = 0;
  unsigned threshold = 0, need = 0;
  if (!all) {
    for (int i = t; i < 3 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
    int newest = INT_MIN;
    for (int s = s0 + t; s < s1; s += kThreads) newest = max(newest, positions[s]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (t == 0) newest_s = unsigned(INT_MIN);
    __syncthreads();
    if ((t & 31) == 0) atomicMax(reinterpret_cast<int*>(&newest_s), newest);
    sync();
    for (unsigned r = 0; r < ctas; ++r) newest = max(newest, int(remote_u32(&newest_s, r)));
    recent_from = (long long)newest - a.recent;
  }
  auto key_at = [&](int s) {
    return use_cache ? cached[s - s0] : slot_key(weights[s], positions[s], a.first, recent_from);
  };
  if (!all) {
    if (use_cache)
      for (int s = s0 + t; s < s1; s += kThreads)
        cached[s - s0] = slot_key(weights[s], positions[s], a.first, recent_from);
    unsigned mask = 0;
    need = keep;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const unsigned bins = pass == 2 ? 1024 : 2048;
      for (int s = s0 + t; s < s1; s += kThreads) {  // its own cached keys: no barrier needed before
        const unsigned k = key_at(s);
        if ((k & mask) == threshold) atomicAdd(&hist[pass][(k >> shift) & (bins - 1)], 1u);
      }
      sync();
      // Bins from the top, two per thread; the bin where the count reaches `need`.
      unsigned v[2] = {};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (unsigned(2 * t + j) < bins)
          for (unsigned r = 0; r < ctas; ++r) v[j] += remote_u32(&hist[pass][bins - 1 - (2 * t + j)], r);
      unsigned total, before = block_scan(v[0] + v[1], scan_u, &total);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (before < need && need <= before + v[j]) {
          found[0] = bins - 1 - (2 * t + j);
          found[1] = need - before;
        }
        before += v[j];
      }
      __syncthreads();
      threshold |= found[0] << shift;
      need = found[1];
      mask |= (bins - 1) << shift;
      __syncthreads();
    }
  }
  // Slot order from here on: thread t owns the slots [b0, b1); an odd count
  // spreads neighbouring threads over the shared memory banks.
  const int own = max(1, (chunk + kThreads - 1) / kThreads) | 1;
  const int b0 = min(s1, s0 + t * own), b1 = min(s1, b0 + own);
  unsigned ties = 0;
  if (!all)
    for (int s = b0; s < b1; ++s) ties += key_at(s) == threshold;
  unsigned cta_ties, tie0 = block_scan(ties, scan_u, &cta_ties);
  if (t == 0) tie_total = cta_ties;
  sync();
  unsigned unused;
  tie0 += cluster_offset(&tie_total, rank, ctas, &unused);
  // kept(s) for s walking upward; `tie` counts the ties passed.
  auto kept = [&](int s, unsigned& tie) {
    if (all) return true;
    const unsigned k = key_at(s);
    return k > threshold || (k == threshold && tie++ < need);
  };
  unsigned long long both = 0;  // holes, movers << 32
  unsigned tie = tie0;
  for (int s = b0; s < b1; ++s) {
    const bool k = kept(s, tie);
    if (s < keep) both += !k;
    else both += (unsigned long long)(k) << 32;
  }
  unsigned long long cta_both, rank0 = block_scan(both, scan_l, &cta_both);
  if (t == 0) {
    hole_total = unsigned(cta_both);
    mover_total = unsigned(cta_both >> 32);
  }
  sync();
  unsigned holes, movers;
  unsigned hole = unsigned(rank0) + cluster_offset(&hole_total, rank, ctas, &holes);
  unsigned mover = unsigned(rank0 >> 32) + cluster_offset(&mover_total, rank, ctas, &movers);
  int* dst = list_of(ws, unit, a.budget);
  int *src = dst + a.budget, *mov = src + a.budget;
  tie = tie0;
  for (int s = b0; s < b1; ++s)
    if (kept(s, tie) && s >= keep) mov[mover++] = s;
  __threadfence();
  sync();  // every mover of the unit is listed; no CTA reads another's shared memory after this
  float* weights_out = a.weights_out + size_t(unit) * a.out_capacity;
  int* positions_out = a.positions_out + size_t(unit) * a.out_capacity;
  tie = tie0;
  for (int s = b0; s < b1 && s < keep; ++s) {
    const bool stays = kept(s, tie);
    const int from = stays ? s : __ldcg(mov + hole);
    const int entry = a.in_place ? int(hole) : s;
    hole += !stays;
    if (stays && a.in_place) continue;
    dst[entry] = s;
    src[entry] = from;
    weights_out[s] = weights[from];
    positions_out[s] = positions[from];
  }
  if (rank == 0 && t == 0)
    list_of(ws, a.caches * a.kv_heads, a.budget)[unit] = a.in_place ? int(holes) : keep;
}

// Block (KV head fastest, then a run of entries, then the cache): the heads'
// 256-byte rows of one slot are moved side by side.  A row's key and value
// are 2 * C 16-byte pieces; each thread moves kPieces of them, loads first.
constexpr int kMoveThreads = 256;
constexpr int kPieces = 4;

template <int C>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a, int* ws, int runs) {
  const int h = blockIdx.x % a.kv_heads, run = blockIdx.x / a.kv_heads % runs, cache = blockIdx.x / a.kv_heads / runs;
  const int unit = cache * a.kv_heads + h, pieces = 2 * (C ? C : a.width / 8);
  wait_prior();
  if (h == 0 && run == 0 && threadIdx.x == 0) {
    const long long n = a.lengths[cache];
    a.lengths_out[cache] = min((long long)a.budget, n < 0 ? 0 : n > a.capacity ? a.capacity : n);
  }
  const long long count = (long long)list_of(ws, a.caches * a.kv_heads, a.budget)[unit] * pieces;
  const int* dst = list_of(ws, unit, a.budget);
  const int* src = dst + a.budget;
  uint4 v[kPieces];
  uint4* to[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const long long i = ((long long)run * kPieces + j) * kMoveThreads + threadIdx.x;
    to[j] = nullptr;
    if (i >= count) continue;
    const int e = int(i / pieces), p = int(i % pieces), c = p % (pieces / 2);
    const bool val = p >= pieces / 2;
    const size_t from = size_t(cache) * a.cache_stride + size_t(src[e]) * a.row_stride + size_t(h) * a.width;
    const size_t into = size_t(cache) * a.out_cache_stride + size_t(dst[e]) * a.out_row_stride + size_t(h) * a.width;
    v[j] = reinterpret_cast<const uint4*>((val ? a.value : a.key) + from)[c];
    to[j] = reinterpret_cast<uint4*>((val ? a.value_out : a.key_out) + into) + c;
  }
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    if (to[j]) *to[j] = v[j];
}

}  // namespace

size_t cache_evict_workspace_bytes(int caches, int kv_heads, int budget) {
  return size_t(caches) * kv_heads * (3 * size_t(budget) + 1) * 4;
}

cudaError_t launch_cache_evict(const EvictArgs& a, void* workspace, cudaStream_t stream) {
  const int units = a.caches * a.kv_heads;
  int ctas = 1;
  while (ctas < 8 && a.capacity > 4096 * ctas) ctas *= 2;
  const int cached = std::min((a.capacity + ctas - 1) / ctas, kMaxCached);
  if (cached > 4096) {  // beyond the 48 KB that need no opt-in (a setting of the current device)
    const cudaError_t s = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kMaxCached * 4);
    if (s != cudaSuccess) return s;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(cached) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int* ws = static_cast<int*>(workspace);
  cudaError_t e = cudaLaunchKernelEx(&cfg, evict_select_kernel, a, ws, cached);
  if (e != cudaSuccess) return e;
  const int pieces = 2 * (a.width / 8);
  const int runs = int((size_t(a.budget) * pieces + kMoveThreads * kPieces - 1) / (kMoveThreads * kPieces));
  cudaLaunchConfig_t mv = {};
  mv.gridDim = dim3(unsigned(units) * runs);
  mv.blockDim = dim3(kMoveThreads);
  mv.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  mv.attrs = attr;
  mv.numAttrs = 1;
  if (a.width == 128) return cudaLaunchKernelEx(&mv, evict_move_kernel<16>, a, ws, runs);
  if (a.width == 64) return cudaLaunchKernelEx(&mv, evict_move_kernel<8>, a, ws, runs);
  return cudaLaunchKernelEx(&mv, evict_move_kernel<0>, a, ws, runs);
}

}  // namespace dl
