// Eviction from KV caches by accumulated attention weight (see
// dl_cache_evict in the public header for the definition).
//
// evict_select_kernel: one cluster of 1-8 CTAs per (cache, KV head) gives each
// slot a 32-bit key (protected highest, then the weight's order-preserving
// bits, NaN lowest) and finds the last slot that stays: histograms of 11, 11
// and 10 bits narrow the keys down until at most 512 slots share the bits found
// so far, those are ranked against one another by (key, slot); only more than
// 512 equal keys need the ties counted in slot order.  Then a slot stays if its
// (key, slot) is at least the cut's, and prefix sums in slot order pair vacated
// slots ("holes", below the kept count) with kept slots beyond it ("movers"):
// hole i receives mover i.  Weights and positions move with the pairing; rows
// are copied by the same CTAs when that is little work, and by
// evict_move_kernel, spread over all SMs, otherwise.  Sources lie at or above
// the kept count and destinations below it, so moving in place needs no order
// between rows.  Integer counts and prefix sums only: results do not depend on
// scheduling.
//
// Measured, 8 heads of width 128, out of place: 32 caches of 2304 slots to 2048
// in 95 us (5.7 TB/s: bound by the copy), of 1051 to 2304 slots in 80; one
// cache of 32768 to 8192 in 36 us, two thirds of it the selection, whose dozen
// cluster-wide steps of 1 to 2 us each bound it; two caches of 320 to 256 in 6.4
// us, two launches.  In place: the same 32 caches in 41 and 37 us (58380 and 6300
// rows move, a floor of 10 and 1.5 us: the selection, then blocks for every slot
// of the budget that mostly find nothing to move), the others in 34 and 7.1 us.
// Adding the histograms up in slices, one per CTA, instead of all by each CTA: no
// gain.
#include <algorithm>
#include <climits>

#include "cache_evict.h"
#include "tcgen05.cuh"

namespace dl {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kRanked = 512;       // slots of a unit ranked one against all
constexpr int kMostTiles = 1024;   // runs of kThreads slots per CTA
constexpr int kMaxCtas = 8;

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
    T s = lane < kWarps ? warp_sums[lane] : T(0), e = s;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const T y = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) e += y;
    }
    if (lane < kWarps) warp_sums[lane] = e - s;
    if (lane == 31) warp_sums[32] = e;
  }
  __syncthreads();
  const T r = warp_sums[warp] + x - v;
  *total = warp_sums[32];
  __syncthreads();
  return r;
}

// Words of shared memory at p in CTA `rank` of the cluster; MULTI = false: this CTA is alone.
template <bool MULTI>
__device__ __forceinline__ uint4 remote_u32x4(const unsigned* p, unsigned rank) {
  if constexpr (!MULTI) return *reinterpret_cast<const uint4*>(p);
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(tc::mapa_shared(smem_addr(p), rank)));
  return v;
}
template <bool MULTI>
__device__ __forceinline__ unsigned remote_u32(const unsigned* p, unsigned rank) {
  if constexpr (!MULTI) return *p;
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(tc::mapa_shared(smem_addr(p), rank)));
  return v;
}
// The word at p in every CTA of the cluster (0 past the last), loads in flight together.
template <bool MULTI>
__device__ __forceinline__ void remote_all(const unsigned* p, unsigned ctas, unsigned (&v)[kMaxCtas]) {
#pragma unroll
  for (int r = 0; r < kMaxCtas; ++r) v[r] = r < ctas ? remote_u32<MULTI>(p, r) : 0u;
}

// Larger = kept first.  -0 counts as +0, NaN below -infinity.
__device__ __forceinline__ unsigned slot_key(float w, int position, int first, long long recent_from) {
  if (position < first || position > recent_from) return 0xffffffffu;
  if (w != w) return 0u;
  const unsigned b = __float_as_uint(w + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ void move_sums(const EvictArgs& a, int unit, int from, int to) {
  a.weights_out[size_t(unit) * a.out_capacity + to] = a.weights[size_t(unit) * a.capacity + from];
  a.positions_out[size_t(unit) * a.out_capacity + to] = a.positions[size_t(unit) * a.capacity + from];
}

// TILES: runs of kThreads slots per CTA, a slot per thread, their keys in
// registers; 0: any number, keys made again from global memory each time.  MULTI:
// a cluster of CTAs per unit.
// Dynamic shared memory: counts [tiles * kWarps] (64 bits), then, with TILES,
// the movers of the CTA [tiles * kThreads] and, to move, the slots that its rows come from.
template <int TILES, bool MULTI>
__global__ void __launch_bounds__(kThreads, TILES > 8 ? 1 : 2) evict_select_kernel(const EvictArgs a, int* ws, int tiles_by_capacity,
                                                               bool move) {
  extern __shared__ __align__(16) unsigned long long counts[];
  int* const own_movers = reinterpret_cast<int*>(counts + tiles_by_capacity * kWarps);
  int* const from_slot = own_movers + tiles_by_capacity * kThreads;
  __shared__ __align__(16) unsigned hist[kBins];
  __shared__ unsigned long long near_order[kRanked], scan_l[33], cut_s;
  __shared__ unsigned scan_u[33], found[3], newest_s, listed, hole_total, mover_total;
  static_assert(sizeof(hist) >= sizeof(near_order) && kRanked <= kThreads,
                "the histogram's memory takes the unit's list afterwards, a thread ranks a slot");
  const unsigned ctas = MULTI ? gridDim.x / (a.caches * a.kv_heads) : 1, rank = MULTI ? tc::cluster_ctarank() : 0;
  const int unit = blockIdx.x / ctas, cache = unit / a.kv_heads, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  for (int i = t; i < kBins; i += kThreads) hist[i] = 0;
  if (t == 0) {
    newest_s = 0;
    listed = 0;
    cut_s = 0;
  }
  wait_prior();
  allow_next();
  const long long len = a.lengths[cache];
  const int n = int(len < 0 ? 0 : len > a.capacity ? a.capacity : len);
  const int keep = min(n, a.budget);
  const int chunk = (n + ctas - 1) / ctas, tiles = (chunk + kThreads - 1) / kThreads;
  const int s0 = min(n, int(rank) * chunk), s1 = min(n, s0 + chunk);
  const float* weights = a.weights + size_t(unit) * a.capacity;
  const int* positions = a.positions + size_t(unit) * a.capacity;
  const bool all = n <= a.budget;  // nothing is evicted
  auto sync = [&] {
    if constexpr (MULTI) tc::cluster_sync();
    else __syncthreads();
  };
  // f(e, slot) for this thread's slot of tile e, in slot order; with TILES also
  // for tiles past the last one, whose slots are at or beyond s1.
  auto each = [&](auto f) {
    if constexpr (TILES > 0) {
#pragma unroll
      for (int e = 0; e < TILES; ++e) f(e, s0 + e * kThreads + t);
    } else {
      for (int e = 0; e < tiles; ++e) f(e, s0 + e * kThreads + t);
    }
  };

  constexpr int held = TILES ? TILES : 1;
  unsigned keys[held] = {};
  long long recent_from = 0;
  unsigned long long cut = 0;  // order of the last slot that stays
  auto key_at = [&](int e, int s) {
    return TILES ? keys[TILES ? e : 0] : slot_key(weights[s], positions[s], a.first, recent_from);
  };
  // Slots from first kept to first evicted: by key, then the lowest slot.
  auto order = [](unsigned k, int s) { return (unsigned long long)k << 32 | (0xffffffffu - unsigned(s)); };
  auto cut_of_all = [&] {  // one CTA of the cluster found it
    unsigned v[kMaxCtas], u[kMaxCtas];
    remote_all<MULTI>(reinterpret_cast<const unsigned*>(&cut_s), ctas, u);
    remote_all<MULTI>(reinterpret_cast<const unsigned*>(&cut_s) + 1, ctas, v);
    unsigned long long c = 0;
#pragma unroll
    for (int r = 0; r < kMaxCtas; ++r) c = max(c, (unsigned long long)v[r] << 32 | u[r]);
    return c;
  };
  __syncthreads();
  if (!all) {
    // Positions as unsigned with the order of int, 0 where there is none.
    unsigned newest = 0;
    float w[held];
    int pos[held];
    each([&](int e, int s) {
      if (s >= s1) return;
      const int p = positions[s];
      newest = max(newest, unsigned(p) ^ 0x80000000u);
      if constexpr (TILES > 0) {
        pos[e] = p;
        w[e] = weights[s];
      }
    });
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) atomicMax(&newest_s, newest);
    sync();
    unsigned v[kMaxCtas];
    remote_all<MULTI>(&newest_s, ctas, v);
    for (int r = 0; r < kMaxCtas; ++r) newest = max(newest, v[r]);
    recent_from = (long long)int(newest ^ 0x80000000u) - a.recent;
    if constexpr (TILES > 0)
      each([&](int e, int s) { keys[e] = s < s1 ? slot_key(w[e], pos[e], a.first, recent_from) : 0u; });

    unsigned mask = 0, prefix = 0, need = keep, near = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const unsigned bins = pass == 2 ? 1024 : 2048;
      each([&](int e, int s) {
        const unsigned k = s < s1 ? key_at(e, s) : 0u;
        const bool in = s < s1 && (k & mask) == prefix;
        // The two keys that many slots share, never looked at and protected,
        // are counted per warp: adds to one word queue up.
        const unsigned none = __ballot_sync(0xffffffffu, in && k == 0x80000000u);
        const unsigned safe = __ballot_sync(0xffffffffu, in && k == 0xffffffffu);
        if (in && (k != 0x80000000u || lane == __ffs(none) - 1) && (k != 0xffffffffu || lane == __ffs(safe) - 1))
          atomicAdd(&hist[(k >> shift) & (bins - 1)],
                    k == 0x80000000u ? __popc(none) : k == 0xffffffffu ? __popc(safe) : 1);
      });
      sync();
      // Bins from the top, four per thread (one load from each CTA); the bin
      // where the count reaches `need`.
      unsigned c[4] = {};
      const int top = int(bins) - 4 - 4 * t;
      if (top >= 0) {
        uint4 y[kMaxCtas];
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) y[r] = r < ctas ? remote_u32x4<MULTI>(&hist[top], r) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) {
          c[0] += y[r].w;
          c[1] += y[r].z;
          c[2] += y[r].y;
          c[3] += y[r].x;
        }
      }
      unsigned total, before = block_scan(c[0] + c[1] + c[2] + c[3], scan_u, &total);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (before < need && need <= before + c[j]) {
          found[0] = top + 3 - j;
          found[1] = need - before;
          found[2] = c[j];
        }
        before += c[j];
      }
      sync();  // also: every CTA has read every histogram
      prefix |= found[0] << shift;
      need = found[1];
      near = found[2];
      mask |= (bins - 1) << shift;
      if (near <= kRanked || pass == 2) break;
      for (int i = t; i < kBins; i += kThreads) hist[i] = 0;
      __syncthreads();
    }
    if (near <= kRanked) {
      unsigned mine = 0, at = 0;
      each([&](int e, int s) { mine += s < s1 && (key_at(e, s) & mask) == prefix; });
      if (mine) at = atomicAdd(&listed, mine);  // the slots' ranks do not depend on it
      each([&](int e, int s) {
        if (s >= s1) return;
        const unsigned k = key_at(e, s);
        if ((k & mask) == prefix) near_order[at++] = order(k, s);
      });
      sync();
      // Every CTA lists the unit's and ranks them, a thread each.
      unsigned long long* list = reinterpret_cast<unsigned long long*>(hist);
      remote_all<MULTI>(&listed, ctas, v);
      for (unsigned i = t; i < near; i += kThreads) {
        unsigned j = i, r = 0;
#pragma unroll
        for (unsigned u = 0; u + 1 < kMaxCtas; ++u)
          if (r == u && j >= v[u]) {
            j -= v[u];
            r = u + 1;
          }
        const unsigned* word = reinterpret_cast<const unsigned*>(&near_order[j]);
        list[i] = (unsigned long long)remote_u32<MULTI>(word + 1, r) << 32 | remote_u32<MULTI>(word, r);
      }
      __syncthreads();
      if (t < near) {
        unsigned better = 0;
#pragma unroll 8
        for (unsigned j = 0; j < near; ++j) better += list[j] > list[t];
        if (better == need - 1) cut_s = list[t];
      }
      __syncthreads();
      cut = cut_s;
    } else {  // more than kRanked equal keys: the need-th of them in slot order
      each([&](int e, int s) {
        const unsigned m = __ballot_sync(0xffffffffu, s < s1 && key_at(e, s) == prefix);
        if (lane == 0 && e < tiles) counts[e * kWarps + warp] = __popc(m);
      });
      __syncthreads();
      unsigned long long run = 0;
      for (int i0 = 0; i0 < tiles * kWarps; i0 += kThreads) {
        const int i = i0 + t;
        unsigned long long total;
        const unsigned long long x = block_scan(i < tiles * kWarps ? counts[i] : 0ull, scan_l, &total);
        if (i < tiles * kWarps) counts[i] = run + x;
        run += total;
      }
      if (t == 0) listed = unsigned(run);
      sync();
      remote_all<MULTI>(&listed, ctas, v);
      unsigned before = 0;
      for (int r = 0; r < int(rank); ++r) before += remote_u32<MULTI>(&listed, r);
      each([&](int e, int s) {
        const bool tie = s < s1 && key_at(e, s) == prefix;
        const unsigned m = __ballot_sync(0xffffffffu, tie);
        if (tie && before + unsigned(counts[e * kWarps + warp]) + __popc(m & ((1u << lane) - 1)) == need - 1)
          cut_s = order(prefix, s);
      });
      sync();
      cut = cut_of_all();
    }
  }
  auto stays = [&](int e, int s) { return all || order(key_at(e, s), s) >= cut; };
  // Ranks of holes and movers: counts per (tile, warp), summed in slot order.
  const int used = tiles * kWarps;
  each([&](int e, int s) {
    const bool in = s < s1, k = in && stays(e, s);
    const unsigned h = __ballot_sync(0xffffffffu, in && s < keep && !k);
    const unsigned m = __ballot_sync(0xffffffffu, in && s >= keep && k);
    if (lane == 0 && e < tiles) counts[e * kWarps + warp] = __popc(h) | (unsigned long long)(__popc(m)) << 32;
  });
  __syncthreads();
  unsigned long long run = 0;
  for (int i0 = 0; i0 < used; i0 += kThreads) {
    const int i = i0 + t;
    unsigned long long total;
    const unsigned long long x = block_scan(i < used ? counts[i] : 0ull, scan_l, &total);
    if (i < used) counts[i] = run + x;
    run += total;
  }
  if (t == 0) {
    hole_total = unsigned(run);
    mover_total = unsigned(run >> 32);
  }
  sync();
  unsigned hole0 = 0, mover0 = 0, holes = 0, movers[kMaxCtas];
  {
    unsigned h[kMaxCtas];
    remote_all<MULTI>(&hole_total, ctas, h);
    remote_all<MULTI>(&mover_total, ctas, movers);
#pragma unroll
    for (unsigned r = 0; r < kMaxCtas; ++r) {
      hole0 += int(r) < int(rank) ? h[r] : 0;
      mover0 += int(r) < int(rank) ? movers[r] : 0;
      holes += h[r];
    }
  }
  // Movers in slot order: each CTA's in its shared memory (with TILES), or the
  // unit's in global memory.
  int* dst = list_of(ws, unit, a.budget);
  int *src = dst + a.budget, *mov = TILES ? own_movers : src + a.budget + mover0;
  each([&](int e, int s) {
    const bool mover = s < s1 && s >= keep && stays(e, s);
    const unsigned m = __ballot_sync(0xffffffffu, mover);
    if (mover) mov[unsigned(counts[e * kWarps + warp] >> 32) + __popc(m & ((1u << lane) - 1))] = s;
  });
  if (!TILES) __threadfence();
  sync();  // every mover of the unit is listed
  auto mover_at = [&](unsigned i) {
    if constexpr (TILES > 0) {
      unsigned r = 0;
#pragma unroll
      for (unsigned u = 0; u + 1 < kMaxCtas; ++u)
        if (r == u && i >= movers[u]) {
          i -= movers[u];
          r = u + 1;
        }
      return int(remote_u32<MULTI>(reinterpret_cast<const unsigned*>(own_movers) + i, r));
    } else {
      return *reinterpret_cast<volatile int*>(src + a.budget + i);
    }
  };
  each([&](int e, int s) {
    const bool in = s < s1 && s < keep, k = in && stays(e, s);
    const unsigned h = __ballot_sync(0xffffffffu, in && !k);
    if (!in) return;
    const unsigned hole = hole0 + unsigned(counts[e * kWarps + warp]) + __popc(h & ((1u << lane) - 1));
    const int from = k ? s : mover_at(hole);
    if (move) {
      from_slot[s - s0] = k && a.in_place ? -1 : from;
    } else if (!k && a.in_place) {
      dst[hole] = s;
      src[hole] = from;
    } else if (!a.in_place) {
      src[s] = from;  // its destination is s
    }
  });
  if constexpr (MULTI) tc::cluster_sync();  // no CTA leaves while another reads its shared memory
  if (!move) {
    if (rank == 0 && t == 0)
      list_of(ws, a.caches * a.kv_heads, a.budget)[unit] = a.in_place ? int(holes) : keep;
    return;
  }
  const int h = unit % a.kv_heads;
  if (rank == 0 && h == 0 && t == 0) a.lengths_out[cache] = keep;  // not the input lengths: see the launch
  __syncthreads();
  const int rows = max(0, min(s1, keep) - s0), pieces = a.width / 4;  // 16-byte pieces of a row's key, then its value
  constexpr int kAhead = 4;
  for (int row = t; row < rows; row += kThreads)
    if (from_slot[row] >= 0) move_sums(a, unit, from_slot[row], s0 + row);
#pragma unroll 1
  for (int i0 = 0; i0 < rows * pieces; i0 += kAhead * kThreads) {
    uint4 v[kAhead];
    uint4* to[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kThreads + t, row = i / pieces, p = i % pieces, c = p % (pieces / 2);
      const bool val = p >= pieces / 2;
      to[j] = nullptr;
      if (i >= rows * pieces || from_slot[row] < 0) continue;
      const size_t from = size_t(cache) * a.cache_stride + size_t(from_slot[row]) * a.row_stride + size_t(h) * a.width;
      const size_t into =
          size_t(cache) * a.out_cache_stride + size_t(s0 + row) * a.out_row_stride + size_t(h) * a.width;
      v[j] = reinterpret_cast<const uint4*>((val ? a.value : a.key) + from)[c];
      to[j] = reinterpret_cast<uint4*>((val ? a.value_out : a.key_out) + into) + c;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (to[j]) *to[j] = v[j];
  }
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
  // The weights and positions of the entries whose first piece is this block's.
  constexpr int span = kPieces * kMoveThreads;
  const long long e1 = ((long long)(run + 1) * span + pieces - 1) / pieces;
  for (long long e = ((long long)run * span + pieces - 1) / pieces + threadIdx.x; e < e1 && e * pieces < count;
       e += kMoveThreads)
    move_sums(a, unit, src[e], a.in_place ? dst[e] : int(e));
  uint4 v[kPieces];
  uint4* to[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const long long i = ((long long)run * kPieces + j) * kMoveThreads + threadIdx.x;
    to[j] = nullptr;
    if (i >= count) continue;
    const int e = int(i / pieces), p = int(i % pieces), c = p % (pieces / 2);
    const bool val = p >= pieces / 2;
    const int source = src[e], slot = a.in_place ? dst[e] : e;
    const size_t from = size_t(cache) * a.cache_stride + size_t(source) * a.row_stride + size_t(h) * a.width;
    const size_t into = size_t(cache) * a.out_cache_stride + size_t(slot) * a.out_row_stride + size_t(h) * a.width;
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

int cache_evict_most_slots() { return kMaxCtas * kMostTiles * kThreads; }

cudaError_t launch_cache_evict(const EvictArgs& a, void* workspace, int sms, cudaStream_t stream) {
  // A CTA takes up to eight slots per thread, in registers; more CTAs per head
  // beyond that, and four rather than two while SMs are idle (21 heads of 7544
  // slots 25.7 us with four, 27.4 with two, 43 with eight; 8 of 8192 21.0, 22.8
  // and 21.6; 8 of 32768 50.6 with four, 35.1 with eight).
  const int units = a.caches * a.kv_heads;
  int ctas = 1;
  while (ctas < kMaxCtas && a.capacity > 8 * kThreads * ctas) ctas *= 2;
  if (ctas == 2 && units <= sms / 4) ctas = 4;
  const int tiles = (a.capacity + ctas * kThreads - 1) / (ctas * kThreads);
  // Moving in the selecting CTAs when they fill the SMs, in one wave, with few
  // rows each: some copy while others still select.  Below that the second
  // kernel's even spread is faster (microseconds, moving there / here: 2 caches
  // of 320 slots to 256 6.3 / 9.3, 20 of 1024 to 512 25.7 / 29.8, 32 of 320 to
  // 256 18.9 / 17.3, 36 of 1024 to 512 36.3 / 34.1).  Not when the lengths are
  // updated in place, since a CTA of another head may still have to read them.
  const int own_rows = std::min(a.budget, tiles * kThreads);
  const size_t bytes = size_t(own_rows) * a.width * 4;
  const bool move = tiles <= 8 && bytes <= (size_t(256) << 10) && units * ctas > sms && units * ctas <= 2 * sms &&
                    a.lengths_out != a.lengths;
  const size_t smem = size_t(tiles) * kWarps * 8 + (tiles <= 32 ? size_t(tiles) * kThreads * 4 : 0) +
                      (move ? size_t(own_rows) * 4 : 0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  int* ws = static_cast<int*>(workspace);
  cudaError_t e;
  if (ctas == 1) {  // at most eight tiles
    e = tiles <= 1 ? cudaLaunchKernelEx(&cfg, evict_select_kernel<1, false>, a, ws, tiles, move)
                   : cudaLaunchKernelEx(&cfg, evict_select_kernel<8, false>, a, ws, tiles, move);
  } else if (tiles <= 8) {
    e = cudaLaunchKernelEx(&cfg, evict_select_kernel<8, true>, a, ws, tiles, move);
  } else if (tiles <= 32) {  // up to 68 KB: an opt-in of the current device
    e = cudaFuncSetAttribute(evict_select_kernel<32, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             32 * (kWarps * 8 + kThreads * 4));
    if (e != cudaSuccess) return e;
    e = cudaLaunchKernelEx(&cfg, evict_select_kernel<32, true>, a, ws, tiles, move);
  } else {
    e = cudaFuncSetAttribute(evict_select_kernel<0, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMostTiles * kWarps * 8);
    if (e != cudaSuccess) return e;
    e = cudaLaunchKernelEx(&cfg, evict_select_kernel<0, true>, a, ws, tiles, move);
  }
  if (e != cudaSuccess || move) return e;
  const int pieces = 2 * (a.width / 8);
  const int runs = int((size_t(a.budget) * pieces + kMoveThreads * kPieces - 1) / (kMoveThreads * kPieces));
  cfg.gridDim = dim3(unsigned(units) * runs);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  if (a.width == 128) return cudaLaunchKernelEx(&cfg, evict_move_kernel<16>, a, ws, runs);
  if (a.width == 64) return cudaLaunchKernelEx(&cfg, evict_move_kernel<8>, a, ws, runs);
  return cudaLaunchKernelEx(&cfg, evict_move_kernel<0>, a, ws, runs);
}

}  // namespace dl
