// Few-row kernel of the shared-prefix attention: at most 32 query rows (the
// new tokens of one sequence x the query heads of one KV head) against that
// sequence's suffix, joined with the prefix ranges the tile kernel left.
//
// Bound by reading the suffix caches once, so the products run on the warp
// tensor instructions, whose small fragments fit a few rows: a warp takes 16
// keys at a time, with the keys as the 16-row operand of both products and the
// query rows as the 8-wide one,
//
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [features x 8 rows] += V^T P^T,
//
// so one 8-row block costs half of what padding the rows to 16 would, and K
// and V fragments are read once for all row blocks.  Warps do not meet until
// the end: each streams its own keys through a private ring of three 16-row
// slots (K, V, K, ...; cp.async, two slots ahead) and keeps its own running
// maximum and sum.  The four warps of a CTA, the CTAs of a cluster (one key
// range each, over distributed shared memory) and the tile kernel's ranges
// are then joined in a fixed order.  Rows past the length are loaded as zeros.
#include "shared_attention.cuh"

namespace dl {
namespace sa {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 16;  // keys of a warp's step
constexpr int kSlots = 3;
constexpr float kRescale = 8.f;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  const int bytes = real ? 16 : 0;  // 0: zero fill, nothing read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float remote_f32(const float* p, unsigned rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::mapa_shared(smem_addr(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 remote_f32x4(const float* p, unsigned rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(tc::mapa_shared(smem_addr(p), rank))
               : "memory");
  return v;
}

template <int D, int NB>
struct RowsShape {
  static constexpr int rows = 8 * NB;
  static constexpr int ring = kWarps * kSlots * kStep * D * 2;
  static constexpr int join = kWarps * rows * D * 4;  // the warps' outputs, over the ring
  static constexpr int smem = ring > join ? ring : join;
};

template <int D, int NB>
__global__ void __launch_bounds__(kThreads) shared_rows_kernel(const SharedAttnArgs a, const Plan pl,
                                                              const Workspace ws, const float scale_log2) {
  constexpr int R = 8 * NB;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float warp_m[kWarps][R], warp_l[kWarps][R], cta_m[R], cta_l[R], row_m[R], row_r[R];
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int g4 = lane >> 2, c2 = (lane & 3) * 2;
  const int live = a.rows * a.group;  // row = new token * group + query head of the group
  // The suffix and the queries come from before the tile kernel, whose blocks
  // have all waited for them; its own results are waited for below.
  if (pl.splits == 0) {
    wait_prior();
    allow_next();
  }
  const int n = suffix_len(a, b);
  const int per = ((n + pl.suffix_splits - 1) / pl.suffix_splits + kStep - 1) / kStep * kStep;
  const int j0 = min(n, split * per), j1 = min(n, j0 + per);
  const int steps = (j1 - j0 + kStep * kWarps - 1) / (kStep * kWarps);
  // Step i of this warp: keys j0 + (i * kWarps + warp) * 16 ...
  auto key0 = [&](int i) { return j0 + (i * kWarps + warp) * kStep; };

  const uint32_t ring = smem_addr(smem) + warp * (kSlots * kStep * D * 2);
  const bf16* base_k = a.sk + size_t(b) * a.s_seq + size_t(h) * D;
  const bf16* base_v = a.sv + size_t(b) * a.s_seq + size_t(h) * D;
  constexpr int P = D / 8;  // 16-byte pieces of a row; piece c of row k lies at c ^ (k & 7)
  auto load = [&](int item) {  // items: K of step 0, V of step 0, K of step 1, ...
    const int i = item >> 1, slot = item % kSlots;
    if (i < steps) {
      const bf16* src = item & 1 ? base_v : base_k;
      const uint32_t dst = ring + slot * (kStep * D * 2);
#pragma unroll
      for (int u = 0; u < kStep * P / 32; ++u) {
        const int idx = u * 32 + lane, k = idx / P, c = idx % P, j = key0(i) + k;
        const bool real = j < j1;
        cp16(dst + k * (D * 2) + ((c ^ (k & 7)) << 4), src + size_t(real ? j : 0) * a.s_row + c * 8, real);
      }
    }
    cp_commit();
  };
  load(0);
  load(1);

  // Query fragments: row 8 nb + g4 (zero past the live rows), features 16 kk + c2, + 8.
  uint32_t q[NB][D / 16][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row = 8 * nb + g4;
    const bf16* src = a.q + (size_t(b) * a.rows + row / a.group) * a.ldq + size_t(h * a.group + row % a.group) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      q[nb][kk][0] = row < live ? *reinterpret_cast<const uint32_t*>(src + 16 * kk + c2) : 0u;
      q[nb][kk][1] = row < live ? *reinterpret_cast<const uint32_t*>(src + 16 * kk + 8 + c2) : 0u;
    }
  }
  // Rows 8 nb + c2, + 1 of the score fragments: how many keys they see.
  int seen[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = 8 * nb + c2 + u;
      seen[nb][u] = row < live ? suffix_seen(n, a.rows, row / a.group) : 0;
    }
  float o[NB][D / 16][4], m[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = -INFINITY;  // unscaled references
    l[nb][0] = l[nb][1] = 0.f;        // this lane's keys only
#pragma unroll
    for (int f = 0; f < D / 16; ++f) o[nb][f][0] = o[nb][f][1] = o[nb][f][2] = o[nb][f][3] = 0.f;
  }
  float* scores = a.sw ? ws.scores + (size_t(b) * a.kv_heads + h) * live * a.scap : nullptr;

#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    load(2 * i + 2);
    cp_wait<2>();
    __syncwarp();
    float s[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
    {
      const uint32_t slot = ring + (2 * i) % kSlots * (kStep * D * 2);
      const int k = lane & 15;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t ka[4];
        ldsm4(ka, slot + k * (D * 2) + (((2 * kk + (lane >> 4)) ^ (k & 7)) << 4));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16816(s[nb], ka, q[nb][kk][0], q[nb][kk][1]);
      }
    }
    __syncwarp();  // every lane has read the slot that the next load refills
    const int ka = key0(i) + g4, kb = ka + 8;
    uint32_t p_hi[NB][2], p_lo[NB][2];
    bool grow = false;
    float top[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int end = min(seen[nb][u], j1), row = 8 * nb + c2 + u;
        if (scores && row < live) {
          if (ka < j1) scores[size_t(row) * a.scap + ka] = s[nb][u];
          if (kb < j1) scores[size_t(row) * a.scap + kb] = s[nb][2 + u];
        }
        if (ka >= end) s[nb][u] = -INFINITY;
        if (kb >= end) s[nb][2 + u] = -INFINITY;
        float x = fmaxf(s[nb][u], s[nb][2 + u]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        top[nb][u] = x;
        grow = grow || (x - m[nb][u]) * scale_log2 > kRescale;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float alpha[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool up = (top[nb][u] - m[nb][u]) * scale_log2 > kRescale;
          alpha[u] = up ? exp2_approx((m[nb][u] - top[nb][u]) * scale_log2) : 1.f;
          if (up) m[nb][u] = top[nb][u];
          l[nb][u] *= alpha[u];
        }
#pragma unroll
        for (int f = 0; f < D / 16; ++f) {
          o[nb][f][0] *= alpha[0];
          o[nb][f][1] *= alpha[1];
          o[nb][f][2] *= alpha[0];
          o[nb][f][3] *= alpha[1];
        }
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float e[4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float shift = m[nb][u] == -INFINITY ? 0.f : -m[nb][u] * scale_log2;
        e[u] = exp2_approx(fmaf(s[nb][u], scale_log2, shift));
        e[2 + u] = exp2_approx(fmaf(s[nb][2 + u], scale_log2, shift));
        l[nb][u] += e[u] + e[2 + u];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t hi, lo;
        split_bf16(pair(e[2 * u], e[2 * u + 1]), hi, lo);
        p_hi[nb][u] = transpose8(hi);
        p_lo[nb][u] = transpose8(lo);
      }
    }
    load(2 * i + 3);
    cp_wait<2>();
    __syncwarp();
    {
      const uint32_t slot = ring + (2 * i + 1) % kSlots * (kStep * D * 2);
      const int k = (lane & 7) + ((lane >> 4) & 1) * 8;
#pragma unroll
      for (int f = 0; f < D / 16; ++f) {
        uint32_t va[4];
        ldsm4_trans(va, slot + k * (D * 2) + (((2 * f + ((lane >> 3) & 1)) ^ (k & 7)) << 4));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma16816(o[nb][f], va, p_hi[nb][0], p_hi[nb][1]);
          mma16816(o[nb][f], va, p_lo[nb][0], p_lo[nb][1]);
        }
      }
    }
    __syncwarp();
  }
  cp_wait<0>();

  // This warp's maxima (base 2) and sums, then its outputs over the ring.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x = l[nb][u];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g4 == 0) {
        warp_m[warp][8 * nb + c2 + u] = m[nb][u] == -INFINITY ? -INFINITY : m[nb][u] * scale_log2;
        warp_l[warp][8 * nb + c2 + u] = x;
      }
    }
  __syncthreads();  // all warps are done with their rings
  float* joined = reinterpret_cast<float*>(smem);  // [warps][R][D]; piece c of row r at c ^ (r & 7)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = 8 * nb + c2 + (u & 1), feature = 16 * f + g4 + (u >> 1) * 8;
        joined[(warp * R + row) * D + (((feature >> 2) ^ (row & 7)) << 2) + (feature & 3)] = o[nb][f][u];
      }
  __syncthreads();
  if (t < R) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w][t]);
    for (int w = 0; w < kWarps; ++w) {
      const float f = warp_m[w][t] == -INFINITY ? 0.f : exp2_approx(warp_m[w][t] - top);
      sum = fmaf(warp_l[w][t], f, sum);
      warp_m[w][t] = f;  // from here on: the warp's factor
    }
    cta_m[t] = top;
    cta_l[t] = sum;
  }
  __syncthreads();
  constexpr int pieces = R * D / 4;
  float4* cta_o = reinterpret_cast<float4*>(smem);  // over warp 0's part
  for (int i = t; i < pieces; i += kThreads) {
    const int row = i / (D / 4);
    if (row >= live) break;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = warp_m[w][row];
      const float4 y = reinterpret_cast<const float4*>(joined)[w * pieces + i];
      v.x = fmaf(y.x, f, v.x);
      v.y = fmaf(y.y, f, v.y);
      v.z = fmaf(y.z, f, v.z);
      v.w = fmaf(y.w, f, v.w);
    }
    cta_o[i] = v;
  }
  if (pl.splits) {
    wait_prior();  // the prefix ranges are complete
    allow_next();
  }
  const unsigned ctas = pl.suffix_splits;
  if (ctas > 1) tc::cluster_sync();
  else __syncthreads();

  // The row's whole softmax, the same in every CTA of the cluster: the
  // cluster's ranges in order, then the prefix ranges in order.
  auto part_of = [&](int row, int s) {
    const int token = b * a.rows + row / a.group;
    return ((size_t(s) * pl.units + h) * pl.tiles + token / pl.per_tile) * kRows +
           token % pl.per_tile * a.group + row % a.group;
  };
  if (t < live) {
    float top = -INFINITY, sum = 0.f;
    for (unsigned r = 0; r < ctas; ++r) top = fmaxf(top, remote_f32(&cta_m[t], r));
    for (int s = 0; s < pl.splits; ++s) top = fmaxf(top, ws.part_ml[part_of(t, s)].x);
    for (unsigned r = 0; r < ctas; ++r) {
      const float x = remote_f32(&cta_m[t], r);
      if (x != -INFINITY) sum = fmaf(remote_f32(&cta_l[t], r), exp2_approx(x - top), sum);
    }
    for (int s = 0; s < pl.splits; ++s) {
      const float2 ml = ws.part_ml[part_of(t, s)];
      sum = fmaf(ml.y, ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top), sum);
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
    row_m[t] = sum == 0.f ? 0.f : top;
    row_r[t] = inv;
    if (split == 0) {
      const size_t row = (size_t(b) * a.rows + t / a.group) * a.query_heads + h * a.group + t % a.group;
      if (a.lse) a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
      if (a.pw) ws.norm[row] = RowNorm{row_m[t], inv};
    }
  }
  __syncthreads();
  for (int i = split * kThreads + t; i < live * (D / 4); i += int(ctas) * kThreads) {
    const int row = i / (D / 4), c = i % (D / 4);  // c: where the piece lies, c ^ (row & 7): the piece
    const float mr = row_m[row], inv = row_r[row];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float4 y, float f) {
      v.x = fmaf(y.x, f, v.x);
      v.y = fmaf(y.y, f, v.y);
      v.z = fmaf(y.z, f, v.z);
      v.w = fmaf(y.w, f, v.w);
    };
    for (unsigned r = 0; r < ctas; ++r) {
      const float x = remote_f32(&cta_m[row], r);
      if (x != -INFINITY) add(remote_f32x4(joined + i * 4, r), exp2_approx(x - mr));
    }
    const int feature = (c ^ (row & 7)) * 4;
#pragma unroll 4
    for (int s = 0; s < pl.splits; ++s) {
      const size_t part = part_of(row, s);
      const float x = ws.part_ml[part].x;
      const int r = int(part % kRows);
      if (x != -INFINITY)
        add(reinterpret_cast<const float4*>(ws.part_o + part * D)[(feature >> 2) ^ (r & 7)], exp2_approx(x - mr));
    }
    bf16* out = a.out + (size_t(b) * a.rows + row / a.group) * a.ldo + size_t(h * a.group + row % a.group) * D + feature;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
  }
  if (a.sw) {
    float* sums = a.sw + (size_t(b) * a.kv_heads + h) * a.scap;
    for (int j = j0 + t; j < j1; j += kThreads) {
      float w = 0.f;
      for (int row = 0; row < live; ++row)
        if (j < suffix_seen(n, a.rows, row / a.group))
          w = fmaf(exp2_approx(fmaf(scores[size_t(row) * a.scap + j], scale_log2, -row_m[row])), row_r[row], w);
      sums[j] += w;
    }
  }
  if (ctas > 1) tc::cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int D, int NB>
cudaError_t launch_shape(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  constexpr int smem = RowsShape<D, NB>::smem;
  const cudaError_t e = allow_smem<shared_rows_kernel<D, NB>>(smem);
  if (e != cudaSuccess) return e;
  DependentLaunch d(dim3(p.suffix_splits, a.kv_heads, a.batch), kThreads, smem, stream, p.suffix_splits);
  return cudaLaunchKernelEx(&d.cfg, shared_rows_kernel<D, NB>, a, p, ws, attention_scale(D) * kLog2e);
}

template <int D>
cudaError_t launch_width(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  const int live = a.rows * a.group;
  return live <= 8    ? launch_shape<D, 1>(a, p, ws, stream)
         : live <= 16 ? launch_shape<D, 2>(a, p, ws, stream)
                      : launch_shape<D, 4>(a, p, ws, stream);
}

}  // namespace

cudaError_t launch_rows(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  return a.width == 64 ? launch_width<64>(a, p, ws, stream) : launch_width<128>(a, p, ws, stream);
}

}  // namespace sa
}  // namespace dl
