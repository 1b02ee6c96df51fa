// Sums of the weight each cached key received from the rows of a call.
//
// The rows' norms are known by then, so a key's sum needs its scores once more
// and nothing else: weight = exp2(s * scale - m[row]) * r[row].  One CTA takes
// 128 keys of one KV head and walks the query rows in tiles of up to 128,
//
//   S^T [128 keys x 128 rows] = K Q^T   (tcgen05, both K-major)
//
// with the keys as TMEM lanes: a thread owns one key and adds up its row of
// S^T in order, with no exchange between threads and no atomics.  Scores and
// queries are double-buffered, so the next product runs under the sums.  When
// there are few key tiles, a cluster shares the rows of one and rank 0 adds
// the ranks' sums in order.  The keys were just read by the attention, so they
// come from L2 while the caches fit it.
#include "shared_attention.cuh"

namespace dl {
namespace sa {
namespace {

using namespace tc;

constexpr int kThreads = 160;  // 4 warps of keys, one that loads and issues
constexpr int kAtom = kKeys * 128;
constexpr uint32_t kTmemCols = 256;

struct alignas(64) WeightArgs {
  CUtensorMap q, pk, sk;
  SharedAttnArgs a;
  const RowNorm* norm;
  int per_tile, prefix_tiles, suffix_tiles, ranks;  // key tiles by capacity; CTAs per key tile
  float scale_log2;
};

template <int D>
__global__ void __launch_bounds__(kThreads) shared_weights_kernel(const __grid_constant__ WeightArgs w) {
  constexpr int slot = D / 64 * kAtom;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t k_full, q_full[2], q_free[2], s_full[2], s_free[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_s, whole[2][4];
  __shared__ __align__(16) RowNorm norms[2][kRows];
  __shared__ int seen_s[2][kRows];
  __shared__ float sums[kKeys];
  volatile int* failed = &failed_s;
  const SharedAttnArgs& a = w.a;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;  // K, then two query tiles
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = cluster_ctarank();

  int at = blockIdx.x / w.ranks;
  const bool suffix = at >= w.prefix_tiles * a.kv_heads;
  if (suffix) at -= w.prefix_tiles * a.kv_heads;
  const int h = at % a.kv_heads;
  at /= a.kv_heads;
  const int tile = suffix ? at % w.suffix_tiles : at, b = suffix ? at / w.suffix_tiles : 0;
  const int j0 = tile * kKeys;

  if (threadIdx.x == 0) {
    mbar_init(&k_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_free[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kKeys);
    }
    failed_s = 0;
    fence_barrier_init();
  }
  if (warp == 4) tmem_alloc(&tmem_slot, kTmemCols);
  wait_prior();
  allow_next();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_slot;

  // Row tiles of this CTA: all tokens for a prefix key, the sequence's rows
  // that can see the tile for a suffix key.
  const int tokens = suffix ? a.rows : a.batch * a.rows, token0 = suffix ? b * a.rows : 0;
  int row_tiles = (tokens + w.per_tile - 1) / w.per_tile, first = 0;
  if (suffix) {
    const int n = suffix_len(a, b);
    if (j0 >= n) row_tiles = 0;
    first = max(0, j0 - n + a.rows) / w.per_tile;
  } else {
    int longest = 0;
    for (int s = lane; s < a.batch; s += 32) longest = max(longest, prefix_len(a, s));
    if (j0 >= __reduce_max_sync(0xffffffffu, longest)) row_tiles = 0;
  }
  const int span = max(0, row_tiles - first);
  const int i0 = first + int((long long)span * rank / w.ranks);
  const int n = first + int((long long)span * (rank + 1) / w.ranks) - i0;

  float sum = 0.f;
  if (warp == 4) {
    if (n > 0 && elect_one()) {
      auto mem = [&](uint32_t off) { return smem_raw + (base + off - smem_addr(smem_raw)); };
      const unsigned q_bytes = unsigned(w.per_tile * a.group * 128 * (D / 64));
      auto load_q = [&](int i) {
        mbar_arrive_expect_tx(&q_full[i & 1], q_bytes);
        for (int c = 0; c < D / 64; ++c)
          tma_3d(mem((1 + (i & 1)) * slot + c * kAtom), &w.q, 64 * c, h * a.group, token0 + (i0 + i) * w.per_tile,
                 &q_full[i & 1]);
      };
      mbar_arrive_expect_tx(&k_full, unsigned(slot));
      for (int c = 0; c < D / 64; ++c) {
        if (suffix) tma_4d(mem(c * kAtom), &w.sk, 64 * c, h, j0, b, &k_full);
        else tma_3d(mem(c * kAtom), &w.pk, 64 * c, h, j0, &k_full);
      }
      load_q(0);
      int loaded = 1;
      if (n > 1) {
        load_q(1);
        loaded = 2;
      }
      bool ok = role_wait(&k_full, 0, failed);
      int issued = 0;
      for (int i = 0; i < n && ok; ++i) {
        ok = role_wait(&q_full[i & 1], (i >> 1) & 1, failed) &&
             (i < 2 || role_wait(&s_free[i & 1], ((i >> 1) + 1) & 1, failed));
        if (!ok) break;
        fence_after_sync();
        const uint32_t kt = base, qt = base + (1 + (i & 1)) * slot;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t atom = uint32_t(kk >> 2) * kAtom;
          const uint64_t off = uint64_t((kk & 3) * 2);
          mma_bf16(tmem + (i & 1) * kRows, smem_desc_sw128(kt + atom) + off, smem_desc_sw128(qt + atom) + off,
                   instr_desc_bf16(kKeys, kRows), kk ? 1u : 0u);
        }
        mma_commit(&s_full[i & 1]);
        mma_commit(&q_free[i & 1]);
        issued = i + 1;
        if (i + 2 < n) {
          ok = role_wait(&q_free[i & 1], (i >> 1) & 1, failed);
          if (!ok) break;
          load_q(i + 2);
          loaded = i + 3;
        }
      }
      if (!ok) {  // copies and products still in flight use this CTA's memory
        mbar_wait(&k_full, 0);
        for (int i = max(0, loaded - 2); i < loaded; ++i) mbar_wait(&q_full[i & 1], (i >> 1) & 1);
        for (int i = max(0, issued - 2); i < issued; ++i) mbar_wait(&q_free[i & 1], (i >> 1) & 1);
      }
    }
    __syncwarp();
  } else {
    const int r = threadIdx.x, key = j0 + r;
    const uint32_t lanes = tmem + (uint32_t(warp * 32) << 16);
    // Row r of row tile i: its norm and the keys it sees.
    auto fetch = [&](int i, RowNorm& nm, int& seen) {
      const int local = (i0 + i) * w.per_tile + r / a.group, token = token0 + local;
      nm = RowNorm{0.f, 0.f};
      seen = 0;
      if (i >= n || r / a.group >= w.per_tile || local >= tokens) return;
      nm = w.norm[size_t(token) * a.query_heads + h * a.group + r % a.group];
      seen = suffix ? suffix_seen(suffix_len(a, b), a.rows, local) : prefix_len(a, token / a.rows);
    };
    RowNorm nm;
    int seen;
    fetch(0, nm, seen);
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int s = i & 1;
      norms[s][r] = RowNorm{-nm.m, nm.r};
      seen_s[s][r] = seen;
      const bool all = __all_sync(0xffffffffu, seen >= j0 + kKeys);
      if (lane == 0) whole[s][warp] = all;
      named_sync(1, kKeys);
      fetch(i + 1, nm, seen);
      // After a failure the remaining turns only keep the barrier above met.
      ok = ok && role_wait_warp(&s_full[s], (i >> 1) & 1, failed);
      if (!ok) continue;
      fence_after_sync();
      const bool unmasked = whole[s][0] && whole[s][1] && whole[s][2] && whole[s][3];
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int c = 0; c < kRows; c += 32) {
        uint32_t v[32];
        tmem_ld32_async(lanes + s * kRows + c, v);
        tmem_ld_wait32(v);
        const float4* nv = reinterpret_cast<const float4*>(norms[s] + c);
        if (unmasked) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float4 y = nv[k];
            part[(2 * k) & 3] =
                fmaf(exp2_approx(fmaf(__uint_as_float(v[2 * k]), w.scale_log2, y.x)), y.y, part[(2 * k) & 3]);
            part[(2 * k + 1) & 3] =
                fmaf(exp2_approx(fmaf(__uint_as_float(v[2 * k + 1]), w.scale_log2, y.z)), y.w, part[(2 * k + 1) & 3]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const RowNorm y = norms[s][c + k];
            const float e = exp2_approx(fmaf(__uint_as_float(v[k]), w.scale_log2, y.m));
            part[k & 3] = key < seen_s[s][c + k] ? fmaf(e, y.r, part[k & 3]) : part[k & 3];
          }
        }
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      fence_before_sync();
      mbar_arrive(&s_free[s]);
    }
    if (!ok) sum = NAN;
    sums[r] = sum;
  }
  fence_before_sync();
  if (w.ranks > 1) cluster_sync();
  else __syncthreads();
  if (warp < 4 && rank == 0 && span > 0) {
    const int key = j0 + int(threadIdx.x), cap = suffix ? a.scap : a.pcap;
    float total = 0.f;
    for (int r = 0; r < w.ranks; ++r) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];"
                   : "=f"(v)
                   : "r"(mapa_shared(smem_addr(&sums[threadIdx.x]), r))
                   : "memory");
      total += v;
    }
    if (key < cap) {
      float* out = suffix ? a.sw + (size_t(b) * a.kv_heads + h) * a.scap : a.pw + size_t(h) * a.pcap;
      out[key] += total;
    }
  }
  if (w.ranks > 1) cluster_sync();
  if (warp == 4) tmem_dealloc(tmem, kTmemCols);
}

}  // namespace

cudaError_t launch_weights(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  WeightArgs w = {};
  w.a = a;
  w.norm = ws.norm;
  w.per_tile = p.per_tile;
  w.prefix_tiles = a.pw ? (a.pcap + kKeys - 1) / kKeys : 0;
  w.suffix_tiles = a.sw && !p.pooled ? (a.scap + kKeys - 1) / kKeys : 0;
  w.ranks = p.weight_ranks;
  w.scale_log2 = attention_scale(a.width) * kLog2e;
  if (!encode_query_map(&w.q, a, p.per_tile)) return cudaErrorInvalidValue;
  if (w.prefix_tiles && !encode_prefix_map(&w.pk, a, a.pk)) return cudaErrorInvalidValue;
  if (w.suffix_tiles && !encode_suffix_map(&w.sk, a, a.sk)) return cudaErrorInvalidValue;
  const long long units = (long long)(w.prefix_tiles + (long long)w.suffix_tiles * a.batch) * a.kv_heads;
  if (units == 0) return cudaSuccess;
  const int smem = 3 * (a.width / 64) * kAtom + 1024;
  const cudaError_t e = a.width == 64 ? allow_smem<shared_weights_kernel<64>>(smem)
                                      : allow_smem<shared_weights_kernel<128>>(smem);
  if (e != cudaSuccess) return e;
  DependentLaunch d(dim3(unsigned(units * w.ranks)), kThreads, smem, stream, w.ranks);
  return a.width == 64 ? cudaLaunchKernelEx(&d.cfg, shared_weights_kernel<64>, w)
                       : cudaLaunchKernelEx(&d.cfg, shared_weights_kernel<128>, w);
}

}  // namespace sa
}  // namespace dl
