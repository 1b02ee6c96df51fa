// Attention of a batch of sequences over one shared prefix cache and their
// own suffix caches, and the sums of the weight each key receives.
//
//   s[t, h, j] = q[t, h] . k[j, h / group] / sqrt(d),  lse = log sum_j exp(s),
//   out = sum_j exp(s - lse) v[j],  weight[j] += sum over t, h of exp(s - lse)
//
// Plain form: one CTA per (token, query head), its warps striding the keys
// with a running maximum and sum each; the weights are a second kernel, one
// warp per key that walks the rows in order.
#include <cmath>

#include "shared_attention.h"

namespace dl {
namespace {

__device__ __forceinline__ int clamp_len(long long n, int cap) { return int(n < 0 ? 0 : n > cap ? cap : n); }

// Prefix and suffix keys that row i of sequence b sees.
__device__ __forceinline__ int prefix_seen(const SharedAttnArgs& a, int b) {
  return a.pcap ? clamp_len(a.plens[b], a.pcap) : 0;
}
__device__ __forceinline__ int suffix_seen(const SharedAttnArgs& a, int b, int i) {
  return a.scap ? max(0, clamp_len(a.slens[b], a.scap) - (a.rows - 1 - i)) : 0;
}

// q . k over the warp, lane l holding features l, l + 32, ...
template <int D>
__device__ __forceinline__ float warp_dot(const float (&q)[D / 32], const bf16* k, int lane) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) s = fmaf(q[c], widen(k[lane + 32 * c]), s);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <int D>
__global__ void __launch_bounds__(128) attend_kernel(SharedAttnArgs a, float* lse_out, float scale) {
  __shared__ float ms[4], ls[4], os[4][D];
  const int token = blockIdx.x, hq = blockIdx.y, b = token / a.rows, i = token % a.rows, h = hq / a.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float q[D / 32], o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    q[c] = widen(a.q[token * a.ldq + size_t(hq) * D + lane + 32 * c]);
    o[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int np = prefix_seen(a, b), n = np + suffix_seen(a, b, i);
  for (int j = warp; j < n; j += 4) {
    const size_t at = (j < np ? size_t(j) * a.p_row : size_t(b) * a.s_seq + size_t(j - np) * a.s_row) + size_t(h) * D;
    const float s = warp_dot<D>(q, (j < np ? a.pk : a.sk) + at, lane) * scale;
    const bf16* v = (j < np ? a.pv : a.sv) + at;
    const float mn = fmaxf(m, s), alpha = expf(m - mn), p = expf(s - mn);
    l = l * alpha + p;
    m = mn;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = fmaf(p, widen(v[lane + 32 * c]), o[c] * alpha);
  }
  if (lane == 0) {
    ms[warp] = m;
    ls[warp] = l;
  }
#pragma unroll
  for (int c = 0; c < D / 32; ++c) os[warp][lane + 32 * c] = o[c];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, ms[w]);
  for (int w = 0; w < 4; ++w) L += M == -INFINITY ? 0.f : ls[w] * expf(ms[w] - M);
  for (int f = threadIdx.x; f < D; f += 128) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += M == -INFINITY ? 0.f : os[w][f] * expf(ms[w] - M);
    a.out[token * a.ldo + size_t(hq) * D + f] = narrow(L > 0.f ? x / L : 0.f);
  }
  if (threadIdx.x == 0) lse_out[size_t(token) * a.query_heads + hq] = M + logf(L);
}

// Keys [0, pcap) of the prefix (b = -1) or [0, scap) of sequence b's suffix.
template <int D>
__global__ void __launch_bounds__(128) weights_kernel(SharedAttnArgs a, const float* lse, float scale, bool suffix) {
  const int lane = threadIdx.x & 31, j = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  if (j >= (suffix ? a.scap : a.pcap)) return;
  const bf16* k = (suffix ? a.sk + size_t(b) * a.s_seq + size_t(j) * a.s_row : a.pk + size_t(j) * a.p_row) + size_t(h) * D;
  float sum = 0.f;
  const int t0 = suffix ? b * a.rows : 0, t1 = suffix ? t0 + a.rows : a.batch * a.rows;
  for (int t = t0; t < t1; ++t) {
    if (j >= (suffix ? suffix_seen(a, b, t - t0) : prefix_seen(a, t / a.rows))) continue;
    for (int hq = h * a.group; hq < (h + 1) * a.group; ++hq) {
      float q[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) q[c] = widen(a.q[t * a.ldq + size_t(hq) * D + lane + 32 * c]);
      sum += expf(warp_dot<D>(q, k, lane) * scale - lse[size_t(t) * a.query_heads + hq]);
    }
  }
  if (lane == 0) {
    if (suffix) a.sw[(size_t(b) * a.kv_heads + h) * a.scap + j] += sum;
    else a.pw[size_t(h) * a.pcap + j] += sum;
  }
}

template <int D>
cudaError_t launch(const SharedAttnArgs& a, float* ws, cudaStream_t stream) {
  float* lse = a.lse ? a.lse : ws;
  const float scale = attention_scale(D);
  attend_kernel<D><<<dim3(a.batch * a.rows, a.query_heads), 128, 0, stream>>>(a, lse, scale);
  if (a.pw && a.pcap)
    weights_kernel<D><<<dim3((a.pcap + 3) / 4, a.kv_heads), 128, 0, stream>>>(a, lse, scale, false);
  if (a.sw && a.scap)
    weights_kernel<D><<<dim3((a.scap + 3) / 4, a.kv_heads, a.batch), 128, 0, stream>>>(a, lse, scale, true);
  return cudaGetLastError();
}

}  // namespace

size_t shared_attention_workspace_bytes(const SharedAttnArgs& a, bool, int) {
  return size_t(a.batch) * a.rows * a.query_heads * 4;
}

cudaError_t launch_shared_attention(const SharedAttnArgs& a, void* workspace, int, cudaStream_t stream) {
  return a.width == 64 ? launch<64>(a, static_cast<float*>(workspace), stream)
                       : launch<128>(a, static_cast<float*>(workspace), stream);
}

}  // namespace dl
