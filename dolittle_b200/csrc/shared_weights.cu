// Sums of the weight each cached key received from the rows of a call.
//
// The rows' norms are known by then, so a key's sum needs its scores once more
// and nothing else: weight = exp2(s * scale - m[row]) * r[row].  One CTA takes
// 256 keys of one KV head and walks the query rows in tiles of up to 128,
//
//   S^T [2 x 128 keys x 128 rows] = K Q^T   (tcgen05, both K-major)
//
// with the keys as TMEM lanes: two threads own a key and add up half of its row
// of S^T each, in order, joined at the end: no exchange in between, no atomics.
// The latencies around the exponentials bound it: sixteen warps cover one
// another's, two key tiles share each query tile that comes through L2, scores
// and queries are double-buffered, and the next key tiles load under the sums of
// the ones before.  When there are few key tiles and many rows, the row tiles of
// a pair are cut into parts and a second kernel adds the parts' sums in order.
// The keys were just read by the attention, so they come from L2 while the
// caches fit it.
//
// Measured: 8192 keys x 8 heads against 256 tokens x 4 heads (67 M weights) 38
// us, 47 % of the exponential unit while a CTA has work; 256 pairs over 148 SMs
// leave a seventh of the time idle.  Slower: scores of 64 columns in registers
// at once (108 us against 94 for the whole call), the keys in TMEM (98.3 / 97.6),
// the norms as one more product step (105.7 / 97.5).
#include "shared_attention.cuh"

#include <algorithm>

namespace dl {
namespace sa {
namespace {

using namespace tc;

constexpr int kWork = 2 * kPair;      // threads that sum, two per key
constexpr int kThreads = kWork + 32;  // and a warp that loads and issues
constexpr int kIssueWarp = kWork / 32;
constexpr int kAtom = kKeys * 128;
constexpr uint32_t kTmemCols = 512;  // scores: [key tile][buffer]

struct alignas(64) WeightArgs {
  CUtensorMap q, pk, sk;
  SharedAttnArgs a;
  const RowNorm* norm;
  int per_tile, prefix_pairs, suffix_pairs;  // pairs of key tiles by capacity
  int prefix_parts, suffix_parts;            // of a pair's row tiles
  float *prefix_sums, *suffix_sums;          // of the parts, if there is more than one: [part][(b,) h][256 keys x pairs]
  int prefix_units, units;                   // parts x pairs x KV heads (x sequences)
  float scale_log2;
};

// The longest and shortest prefix of any sequence; whole warps.
__device__ __forceinline__ void prefix_extent(const SharedAttnArgs& a, int& longest, int& shortest) {
  longest = 0;
  shortest = a.pcap;
  for (int s = threadIdx.x & 31; s < a.batch; s += 32) {
    const int l = prefix_len(a, s);
    longest = max(longest, l);
    shortest = min(shortest, l);
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  shortest = __reduce_min_sync(0xffffffffu, shortest);
}

// Row tiles [first, first + span) that see keys from j0 on, of `tokens` tokens:
// all of them for a prefix, of a sequence's rows for its suffix of n keys.
__device__ __forceinline__ int row_span(const WeightArgs& w, bool suffix, int tokens, int j0, int n, int& first) {
  first = suffix ? max(0, j0 - n + w.a.rows) / w.per_tile : 0;
  return j0 >= n ? 0 : max(0, (tokens + w.per_tile - 1) / w.per_tile - first);
}
__device__ __forceinline__ int part_start(int span, int part, int parts) {
  return span / parts * part + min(part, span % parts);
}
// The sums of a part of pair (b, h, j0).
__device__ __forceinline__ float* part_sums(const WeightArgs& w, bool suffix, int part, int b, int h, int j0) {
  const size_t head = suffix ? (size_t(part) * w.a.batch + b) * w.a.kv_heads + h : size_t(part) * w.a.kv_heads + h;
  return (suffix ? w.suffix_sums : w.prefix_sums) + head * kPair * (suffix ? w.suffix_pairs : w.prefix_pairs) + j0;
}

// A pair of key tiles of one KV head and the row tiles [i0, i0 + n) that this
// CTA takes it through: of all tokens for a prefix key, of the sequence's rows
// that can see the first tile for a suffix key.
struct Unit {
  bool suffix;
  int h, b, j0, tokens, token0, i0, n, part;
  int longest, shortest;  // prefix lengths of all sequences; a suffix's own
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) shared_weights_kernel(const __grid_constant__ WeightArgs w) {
  constexpr int slot = D / 64 * kAtom;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t k_full[2], q_full[2], q_free[2], s_full[2][2], s_free[2][2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_s;
  __shared__ __align__(16) RowNorm norms[2][2][kRows];
  __shared__ int seen_s[2][2][kRows];
  __shared__ float sums[kWork];
  volatile int* failed = &failed_s;
  const SharedAttnArgs& a = w.a;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;  // two pairs of key tiles, two query tiles
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&q_full[i], 1);
      mbar_init(&q_free[i], 1);
      for (int p = 0; p < 2; ++p) {
        mbar_init(&s_full[p][i], 1);
        mbar_init(&s_free[p][i], kPair / 32);
      }
    }
    failed_s = 0;
    fence_barrier_init();
  }
  if (warp == kIssueWarp) {
    tmem_alloc(&tmem_slot, kTmemCols);
    if (lane == 0) {
      prefetch_map(&w.q);
      if (w.prefix_pairs) prefetch_map(&w.pk);
      if (w.suffix_pairs) prefetch_map(&w.sk);
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_slot;

  int longest, shortest;
  prefix_extent(a, longest, shortest);
  auto unit_of = [&](int at) {
    Unit u;
    u.suffix = at >= w.prefix_units;
    if (u.suffix) at -= w.prefix_units;
    const int parts = u.suffix ? w.suffix_parts : w.prefix_parts;
    u.h = at % a.kv_heads;
    at /= a.kv_heads;
    u.part = at % parts;
    at /= parts;
    u.b = u.suffix ? at / w.suffix_pairs : 0;
    u.j0 = (u.suffix ? at % w.suffix_pairs : at) * kPair;
    u.tokens = u.suffix ? a.rows : a.batch * a.rows;
    u.token0 = u.suffix ? u.b * a.rows : 0;
    u.longest = u.suffix ? suffix_len(a, u.b) : longest;
    u.shortest = shortest;
    int first;
    const int span = row_span(w, u.suffix, u.tokens, u.j0, u.longest, first);
    u.i0 = first + part_start(span, u.part, parts);
    u.n = first + part_start(span, u.part + 1, parts) - u.i0;
    return u;
  };
  // The units of this CTA that have row tiles.
  auto next = [&](int& at, Unit& u) {
    for (; at < w.units; at += gridDim.x) {
      u = unit_of(at);
      if (u.n > 0) {
        at += gridDim.x;
        return true;
      }
    }
    return false;
  };
  auto active = [](const Unit& u, int p) { return u.j0 + p * kKeys < u.longest; };

  if (warp == kIssueWarp) {
    if (elect_one()) {
      auto mem = [&](uint32_t off) { return smem_raw + (base + off - smem_addr(smem_raw)); };
      const unsigned q_bytes = unsigned(w.per_tile * a.group * 128 * (D / 64));
      // Row tiles issued and loaded, of all units in turn; scores issued per key
      // tile; units whose keys were loaded.  The x-th use of a pair of buffers is
      // of buffer x & 1, for its (x >> 1)-th time.
      unsigned x = 0, loaded = 0, scored[2] = {0, 0}, unit = 0, keys = 0;
      bool ok = true;
      auto load_keys = [&](const Unit& u) {
        uint64_t* bar = &k_full[keys & 1];
        const int tiles = active(u, 1) ? 2 : 1;
        mbar_arrive_expect_tx(bar, unsigned(tiles * slot));
        for (int p = 0; p < tiles; ++p)
          for (int c = 0; c < D / 64; ++c) {
            unsigned char* dst = mem(((keys & 1) * 2 + p) * slot + c * kAtom);
            if (u.suffix) tma_4d(dst, &w.sk, 64 * c, u.h, u.j0 + p * kKeys, one_suffix(a) ? 0 : u.b, bar);
            else tma_3d(dst, &w.pk, 64 * c, u.h, u.j0 + p * kKeys, bar);
          }
        ++keys;
      };
      auto load_query = [&](const Unit& u, int i) {
        const int s = loaded & 1;
        if (loaded >= 2 && !role_wait(&q_free[s], ((loaded >> 1) + 1) & 1, failed)) return false;
        mbar_arrive_expect_tx(&q_full[s], q_bytes);
        for (int c = 0; c < D / 64; ++c)
          tma_3d(mem((4 + s) * slot + c * kAtom), &w.q, 64 * c, u.h * a.group, u.token0 + (u.i0 + i) * w.per_tile,
                 &q_full[s]);
        ++loaded;
        return true;
      };
      Unit u, v;
      int at = blockIdx.x, li = 0;  // li: next row tile to load, of u or (ahead) of v
      bool have = next(at, u), more = false, ahead = false;
      if (have) {
        load_keys(u);
        more = next(at, v);
      }
      auto load_more = [&] {  // two row tiles ahead of the products, into the next unit if need be
        while (ok && loaded < x + 2) {
          if (!ahead && li >= u.n) {
            if (!more) return;
            ahead = true;
            li = 0;
          }
          if (ahead && li >= v.n) return;
          ok = load_query(ahead ? v : u, li++);
        }
      };
      while (have && ok) {
        load_more();
        ok = ok && role_wait(&k_full[unit & 1], (unit >> 1) & 1, failed);
        for (int i = 0; i < u.n && ok; ++i) {
          const int s = x & 1;
          ok = role_wait(&q_full[s], (x >> 1) & 1, failed);
          for (int p = 0; p < 2 && ok; ++p) {
            if (!active(u, p)) continue;
            const int sb = scored[p] & 1;
            if (scored[p] >= 2) ok = role_wait(&s_free[p][sb], ((scored[p] >> 1) + 1) & 1, failed);
            if (!ok) break;
            fence_after_sync();
            const uint32_t kt = base + ((unit & 1) * 2 + p) * slot, qt = base + (4 + s) * slot;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t atom = uint32_t(kk >> 2) * kAtom;
              const uint64_t off = uint64_t((kk & 3) * 2);
              mma_bf16(tmem + (p * 2 + sb) * kRows, smem_desc_sw128(kt + atom) + off, smem_desc_sw128(qt + atom) + off,
                       instr_desc_bf16(kKeys, kRows), kk ? 1u : 0u);
            }
            mma_commit(&s_full[p][sb]);
            ++scored[p];
          }
          if (!ok) break;
          mma_commit(&q_free[s]);
          ++x;
          if (i == 0 && more) {  // the other keys' buffer: its last product is over
            if (x >= 2) ok = role_wait(&q_free[x & 1], ((x - 2) >> 1) & 1, failed);
            if (ok) load_keys(v);
          }
          load_more();
        }
        if (!ok) break;
        have = more;
        u = v;
        if (!ahead) li = 0;
        ahead = false;
        more = have && next(at, v);
        ++unit;
      }
      if (!ok) {  // copies and products still in flight use this CTA's memory
        for (unsigned k = keys > 2 ? keys - 2 : 0; k < keys; ++k) mbar_wait(&k_full[k & 1], (k >> 1) & 1);
        for (unsigned k = loaded > 2 ? loaded - 2 : 0; k < loaded; ++k) mbar_wait(&q_full[k & 1], (k >> 1) & 1);
        mma_commit(&q_free[x & 1]);  // completes with the products issued so far
        if (x >= 1) mbar_wait(&q_free[(x - 1) & 1], ((x - 1) >> 1) & 1);
        mbar_wait(&q_free[x & 1], (x >> 1) & 1);
      }
    }
    __syncwarp();
  } else {
    // Key r of tile p, columns (rows of the queries) from half * 64 on.
    const int r = threadIdx.x % kKeys, half = threadIdx.x / kKeys % 2, p = threadIdx.x / kPair;
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16) + p * 2 * kRows + half * (kRows / 2);
    const uint64_t scale2 = pair(w.scale_log2, w.scale_log2);
    // Row r of row tile i, if it exists; its norm is on its way from one turn to the next.
    auto row_of = [&](const Unit& u, int i, int& local) {
      local = (u.i0 + i) * w.per_tile + r / a.group;
      return r / a.group < w.per_tile && local < u.tokens;
    };
    auto fetch = [&](const Unit& u, int i) {
      int local;
      RowNorm nm = {0.f, 0.f};
      if (half == 0 && row_of(u, i, local))
        nm = w.norm[size_t(u.token0 + local) * a.query_heads + u.h * a.group + r % a.group];
      return nm;
    };
    auto next_active = [&](int& at, Unit& u) {
      while (next(at, u))
        if (active(u, p)) return true;
      return false;
    };
    // Only the norms come from the kernel before this one.  It began when what
    // came before it was over, so keys, queries and lengths are there already:
    // the first products run while it ends.
    wait_prior();
    allow_next();
    Unit u, following;
    int at = blockIdx.x;
    unsigned g = 0;
    bool ok = true, more = next_active(at, u);
    RowNorm nm = {0.f, 0.f};
    if (more) nm = fetch(u, 0);
    sums[threadIdx.x] = 0.f;
    while (more) {
      const int j0 = u.j0 + p * kKeys, key = j0 + r;
      float sum = 0.f;
      more = next_active(at, following);
#pragma unroll 1
      for (int i = 0; i < u.n; ++i, ++g) {
        const int s = g & 1;
        if (half == 0) norms[p][s][r] = RowNorm{-nm.m, nm.r};
        // Does every row of the tile exist and see every key of it?
        const int head = (u.i0 + i) * w.per_tile;
        const bool plain = w.per_tile * a.group == kRows && head + w.per_tile <= u.tokens &&
                           j0 + kKeys <= (u.suffix ? suffix_seen(u.longest, a.rows, head) : u.shortest);
        if (!plain && half == 0) {
          int local;
          seen_s[p][s][r] = !row_of(u, i, local) ? 0
                            : u.suffix           ? suffix_seen(u.longest, a.rows, local)
                                                 : prefix_len(a, (u.token0 + local) / a.rows);
        }
        named_sync(1 + p, kPair);
        if (i + 1 < u.n) nm = fetch(u, i + 1);
        else if (more) nm = fetch(following, 0);
        // After a failure the remaining turns only keep the barrier above met.
        ok = ok && role_wait_warp(&s_full[p][s], (g >> 1) & 1, failed);
        if (!ok) continue;
        fence_after_sync();
        uint64_t part[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (int c = 0; c < kRows / 2; c += 32) {
          uint32_t v[32];
          tmem_ld32_async(lanes + s * kRows + c, v);
          tmem_ld_wait32(v);
          const int from = half * (kRows / 2) + c;
          const float4* nv = reinterpret_cast<const float4*>(norms[p][s] + from);
          if (plain) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float4 y = nv[k];
              float x0, x1;
              unpair(fma2(pair(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), scale2, pair(y.x, y.z)), x0,
                     x1);
              part[k & 3] = fma2(pair(exp2_approx(x0), exp2_approx(x1)), pair(y.y, y.w), part[k & 3]);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const RowNorm y = norms[p][s][from + k];
              const float e = exp2_approx(fmaf(__uint_as_float(v[k]), w.scale_log2, y.m));
              part[k & 3] = fma2(pair(key < seen_s[p][s][from + k] ? e : 0.f, 0.f), pair(y.r, 0.f), part[k & 3]);
            }
          }
        }
        float x0, x1;
        unpair(add2(add2(part[0], part[1]), add2(part[2], part[3])), x0, x1);
        sum += x0 + x1;
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[p][s]);
      }
      if (!ok) sum = NAN;
      sums[threadIdx.x] = sum;
      named_sync(1 + p, kPair);
      if ((u.suffix ? w.suffix_parts : w.prefix_parts) > 1) {
        if (half == 0)
          part_sums(w, u.suffix, u.part, u.b, u.h, u.j0)[key - u.j0] = sum + sums[threadIdx.x + kKeys];
      } else if (half == 0 && key < (u.suffix ? a.scap : a.pcap)) {
        float* out = u.suffix ? a.sw + (size_t(u.b) * a.kv_heads + u.h) * a.scap : a.pw + size_t(u.h) * a.pcap;
        out[key] += sum + sums[threadIdx.x + kKeys];
      }
      u = following;
    }
    fence_before_sync();
  }
  __syncthreads();
  if (warp == kIssueWarp) tmem_dealloc(tmem, kTmemCols);
}

// Adds the parts' sums of a pair, a thread per key, in order: a block for each
// pair that was cut, prefix pairs first.
__global__ void __launch_bounds__(kPair) shared_weights_add_kernel(const __grid_constant__ WeightArgs w) {
  const SharedAttnArgs& a = w.a;
  const int prefix = w.prefix_parts > 1 ? w.prefix_pairs * a.kv_heads : 0;
  const bool suffix = int(blockIdx.x) >= prefix;
  int at = blockIdx.x - (suffix ? prefix : 0), first;
  const int h = at % a.kv_heads;
  at /= a.kv_heads;
  const int b = suffix ? at / w.suffix_pairs : 0, j0 = (suffix ? at % w.suffix_pairs : at) * kPair;
  const int key = j0 + int(threadIdx.x), parts = suffix ? w.suffix_parts : w.prefix_parts;
  // Lengths and sums are from before the weights kernel, which began when what
  // came before it was over; only the parts' sums have to be waited for.
  int n, shortest;
  if (suffix) n = suffix_len(a, b);
  else prefix_extent(a, n, shortest);
  const int span = row_span(w, suffix, suffix ? a.rows : a.batch * a.rows, j0, n, first);
  const bool live = key < n && span > 0;
  float* out = suffix ? a.sw + (size_t(b) * a.kv_heads + h) * a.scap : a.pw + size_t(h) * a.pcap;
  const float old = live ? out[key] : 0.f;
  wait_prior();
  allow_next();
  if (!live) return;
  float total = 0.f;
#pragma unroll 8
  for (int p = 0; p < min(parts, span); ++p) total += part_sums(w, suffix, p, b, h, j0)[threadIdx.x];
  out[key] = old + total;
}

}  // namespace

cudaError_t launch_weights(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, int sms, cudaStream_t stream) {
  WeightArgs w = {};
  w.a = a;
  w.norm = ws.norm;
  w.per_tile = p.per_tile;
  w.prefix_pairs = a.pw ? (a.pcap + kPair - 1) / kPair : 0;
  w.suffix_pairs = a.sw && !p.pooled ? (a.scap + kPair - 1) / kPair : 0;
  w.prefix_parts = p.prefix_parts;
  w.suffix_parts = p.suffix_parts;
  w.prefix_sums = ws.prefix_sums;
  w.suffix_sums = ws.suffix_sums;
  w.scale_log2 = attention_scale(a.width) * kLog2e;
  if (!encode_query_map(&w.q, a, p.per_tile)) return cudaErrorInvalidValue;
  if (w.prefix_pairs && !encode_prefix_map(&w.pk, a, a.pk)) return cudaErrorInvalidValue;
  if (w.suffix_pairs && !encode_suffix_map(&w.sk, a, a.sk)) return cudaErrorInvalidValue;
  const long long prefix = (long long)w.prefix_pairs * a.kv_heads, suffix = (long long)w.suffix_pairs * a.batch * a.kv_heads;
  const long long units = prefix * w.prefix_parts + suffix * w.suffix_parts;
  if (units == 0) return cudaSuccess;
  if (units > (1 << 30)) return cudaErrorInvalidValue;
  w.prefix_units = int(prefix * w.prefix_parts);
  w.units = int(units);
  // At least half of an SM's memory: each block takes all of the SM's TMEM.
  const int smem = std::max(6 * (a.width / 64) * kAtom + 1024, 120 << 10);
  cudaError_t e = a.width == 64 ? allow_smem<shared_weights_kernel<64>>(smem) : allow_smem<shared_weights_kernel<128>>(smem);
  if (e != cudaSuccess) return e;
  DependentLaunch d(dim3(unsigned(std::min(w.units, sms))), kThreads, smem, stream);
  e = a.width == 64 ? cudaLaunchKernelEx(&d.cfg, shared_weights_kernel<64>, w)
                    : cudaLaunchKernelEx(&d.cfg, shared_weights_kernel<128>, w);
  const long long cut = (w.prefix_parts > 1 ? prefix : 0) + (w.suffix_parts > 1 ? suffix : 0);
  if (e != cudaSuccess || cut == 0) return e;
  DependentLaunch add(dim3(unsigned(cut)), kPair, 0, stream);
  return cudaLaunchKernelEx(&add.cfg, shared_weights_add_kernel, w);
}

}  // namespace sa
}  // namespace dl
