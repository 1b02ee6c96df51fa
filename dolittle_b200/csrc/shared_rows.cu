// Few-row kernels of the shared-prefix attention: at most 32 query rows (the
// new tokens of one sequence x the query heads of one KV head), 8 or 16 of them
// per CTA.
//
// shared_rows_kernel streams that sequence's suffix beside the tile kernel's
// prefix and leaves the part of each key range; shared_join_kernel joins the
// prefix and suffix parts.  For small calls (SOLO) it streams prefix and suffix
// both and ends the rows itself, one launch in all.
//
// Bound by reading the caches once, so the products run on the warp tensor
// instructions, whose small fragments fit a few rows: a warp takes 16 keys at
// a time, with the keys as the 16-row operand of both products and the query
// rows as the 8-wide one,
//
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [features x 8 rows] += V^T P^T,
//
// so one 8-row block costs half of what padding the rows to 16 would, and K
// and V fragments are read once for all row blocks.  Warps do not meet until
// the end: each streams its own keys through a private ring of three 16-row
// slots (K, V, K, ...; cp.async, two slots ahead) and keeps its own running
// maximum and sum.  The four warps of a CTA, then the CTAs that share a row
// are joined in a fixed order.  Rows past the length are loaded as zeros.
//
// Measured: the suffixes of 64 sequences of up to 2048 keys (271 MB) by
// themselves take 53 us, 5.1 TB/s; a small call (64 sequences on 256 + 64 keys,
// 84 MB mostly from L2) 14.0 us, 6.0 TB/s.  Two branches of 256 + 64 keys take 6.0
// us, nearly all of it launch, first loads and join.  A row block of 32 rows
// instead of two of 16 had to wait for the tile kernel's shared memory: batch 8
// of 8 tokens on 8192 + 256 keys 63 us against 36.  A ring of four slots left
// room for fewer CTAs: batch 32 on 8192 + 256 keys 26.4 against 22.7 us.
#include "shared_attention.cuh"

#include <algorithm>
#include <climits>

namespace dl {
namespace sa {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 16;  // keys of a warp's step
constexpr int kSlots = 3;
constexpr float kRescale = 8.f;
constexpr int kMaxParts = kMaxSplits + kMaxSuffixSplits;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool real) {
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
  static constexpr int smem = kWarps * kSlots * kStep * D * 2;
  static_assert(NB <= kMostRows / 8 && (kWarps + 1) * rows * D * 4 <= smem, "the outputs fit the ring");
};

// The whole softmax of one row from its parts' (maximum, sum), by one warp:
// lanes hold two parts each, joined by a fixed tree.  factor[s]: of part s in
// the normalised output.
struct RowJoin {
  float m, inv, lse;
};
template <class Part>
__device__ __forceinline__ RowJoin join_row(int parts, Part&& part, float* factor) {
  const int lane = threadIdx.x & 31;
  float m[2], l[2], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int s = lane + 32 * u;
    const float2 ml = s < parts ? part(s) : make_float2(-INFINITY, 0.f);
    m[u] = ml.x;
    l[u] = ml.y;
    top = fmaxf(top, m[u]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    m[u] = m[u] == -INFINITY ? 0.f : exp2_approx(m[u] - top);
    sum = fmaf(l[u], m[u], sum);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 32 * u < parts) factor[lane + 32 * u] = m[u] * inv;
  return {sum == 0.f ? 0.f : top, inv, sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2};
}

// out += y * f; a part of factor 0 may be undefined.
__device__ __forceinline__ void add_part(float4& out, float4 y, float f) {
  if (f == 0.f) return;
  out.x = fmaf(y.x, f, out.x);
  out.y = fmaf(y.y, f, out.y);
  out.z = fmaf(y.z, f, out.z);
  out.w = fmaf(y.w, f, out.w);
}

// The same for four rows of at most eight parts, eight lanes each: lane = 8 x
// row + part.  Only the lane's own part is read; its factor comes back.
template <class Part>
__device__ __forceinline__ RowJoin join_four_rows(bool real, Part&& part, float& factor) {
  const float2 ml = real ? part() : make_float2(-INFINITY, 0.f);
  float top = ml.x;
#pragma unroll
  for (int o = 4; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
  float sum = ml.y * f;
#pragma unroll
  for (int o = 4; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
  factor = f * inv;
  return {sum == 0.f ? 0.f : top, inv, sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2};
}

// Row `row` (new token * group + query head of the group) of unit (b, h).
__device__ __forceinline__ size_t row_index(const SharedAttnArgs& a, int b, int h, int row) {
  return (size_t(b) * a.rows + row / a.group) * a.query_heads + h * a.group + row % a.group;
}
template <int D>
__device__ __forceinline__ void store_piece(const SharedAttnArgs& a, int b, int h, int row, int piece, float4 v) {
  bf16* out = a.out + (size_t(b) * a.rows + row / a.group) * a.ldo + size_t(h * a.group + row % a.group) * D + piece * 4;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// Adds the weights of suffix keys [j0, j1) of unit (b, h) to their sums, from
// the stored scores and the rows' norms in shared memory, which are there when
// ready() returns; one of `threads`, which all call ready() once.  j0 is a
// multiple of 4, j1 at most the suffix length n.  The scores of four rows x
// eight keys are in flight together (one key after another took as long as a
// kernel: 9 us of a step of batch 32).
template <class Ready>
__device__ __forceinline__ void add_suffix_weights(const SharedAttnArgs& a, const Workspace& ws, float scale_log2, int b,
                                                   int h, int n, int j0, int j1, const float* row_m,
                                                   const float* row_r, int thread, int threads, Ready&& ready) {
  constexpr int kPieces = 1, kAtOnce = 4;  // of 4 keys; rows
  const int live = a.rows * a.group, pitch = score_pitch(a);
  float* sums = a.sw + (size_t(b) * a.kv_heads + h) * a.scap;
  const float* scores = ws.scores + (size_t(b) * a.kv_heads + h) * live * pitch;
  bool waiting = true;
  for (int base = j0; base < j1 || waiting; base += 4 * kPieces * threads) {
    float w[kPieces][4] = {}, old[kPieces][4];
    int j[kPieces];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      j[p] = base + 4 * (thread + p * threads);
#pragma unroll
      for (int k = 0; k < 4; ++k) old[p][k] = j[p] + k < j1 ? sums[j[p] + k] : 0.f;
    }
#pragma unroll 1
    for (int r0 = 0; r0 < live; r0 += kAtOnce) {
      float4 y[kAtOnce][kPieces];
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r)
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
          if (r0 + r < live && j[p] < j1)
            y[r][p] = *reinterpret_cast<const float4*>(scores + size_t(r0 + r) * pitch + j[p]);
      if (waiting) {
        ready();
        waiting = false;
      }
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
        if (r0 + r >= live) break;
        const int seen = min(j1, suffix_seen(n, a.rows, (r0 + r) / a.group));
        const float m = row_m[r0 + r], f = row_r[r0 + r];
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          const float x[4] = {y[r][p].x, y[r][p].y, y[r][p].z, y[r][p].w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (j[p] + k < seen) w[p][k] = fmaf(exp2_approx(fmaf(x[k], scale_log2, -m)), f, w[p][k]);
        }
      }
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j[p] + k < j1) sums[j[p] + k] = old[p][k] + w[p][k];
  }
}

template <int D, int NB, bool SOLO>
__global__ void __launch_bounds__(kThreads, SOLO && NB == 2 ? 3 : 4)
    shared_rows_kernel(const SharedAttnArgs a, const Plan pl, const Workspace ws, const float scale_log2) {
  constexpr int R = 8 * NB;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float warp_m[kWarps][R], warp_l[kWarps][R], cta_m[R], cta_l[R], row_m[R], row_r[R];
  __shared__ float part_f[R][kMaxSuffixSplits];
  const int split = blockIdx.x % pl.suffix_splits, h = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int g4 = lane >> 2, c2 = (lane & 3) * 2;
  // Row = new token * group + query head of the group; this CTA's from row0 on.
  const int unit_rows = a.rows * a.group, row0 = blockIdx.x / pl.suffix_splits * R, live = min(R, unit_rows - row0);
  int np = 0, n = 0, ps = 0, g0 = 0, g1 = 0, steps = 0;  // keys of prefix and suffix; steps of 16: prefix steps, this CTA's [g0, g1), per warp
  float o[NB][D / 16][4], m[NB][2], l[NB][2];
  const uint32_t ring = smem_addr(smem) + warp * (kSlots * kStep * D * 2);
  constexpr int P = D / 8;  // 16-byte pieces of a row; piece c of row k lies at c ^ (k & 7)
  auto load = [&](int item) {  // items: K of step 0, V of step 0, K of step 1, ...
    const int i = item >> 1, slot = item % kSlots, g = g0 + i * kWarps + warp;
    if (g < g1) {
      const bool pre = g < ps;
      const bf16* base = item & 1 ? (pre ? a.pv : a.sv) : (pre ? a.pk : a.sk);
      const bf16* src = base + (pre ? 0 : size_t(b) * a.s_seq) + size_t(h) * D;
      const int j0 = (pre ? g : g - ps) * kStep, end = pre ? np : n;
      const size_t stride = pre ? a.p_row : a.s_row;
      // Lane: piece lane % P of rows lane / P, + 32 / P, ...
      constexpr int kApart = 32 / P;
      const int k0 = lane / P, c = lane % P;
      const bf16* from = src + size_t(j0 + k0) * stride + c * 8;
      const uint32_t dst = ring + slot * (kStep * D * 2) + k0 * (D * 2);
      const bool whole = j0 + kStep <= end;
#pragma unroll
      for (int u = 0; u < kStep / kApart; ++u) {
        const uint32_t to = dst + u * kApart * (D * 2) + (((c ^ k0) ^ (u * kApart & 7)) << 4);
        if (whole) {
          cp16(to, from);
          from += kApart * stride;
        } else {
          const int j = j0 + k0 + u * kApart;
          cp16_or_zero(to, src + size_t(j < end ? j : 0) * stride + c * 8, j < end);
        }
      }
    }
    cp_commit();
  };
  // Turn -1 (SOLO) runs one step on no keys while the kernel before this one
  // ends, which brings the loop's code in: a small call runs it only a few
  // times.  Beside the tile kernel nothing has to be waited for: the suffix and
  // the queries come from before it, and its blocks, which had to start before
  // this kernel could, have waited for them.
#pragma unroll 1
  for (int turn = SOLO ? -1 : 0; turn < 1; ++turn) {
    const int rows = turn < 0 ? 0 : live;
    if (SOLO && turn == 0) wait_prior();
    if (turn == 0) allow_next();
    // Keys in steps of 16: the prefix's (SOLO), then the suffix's; this CTA has
    // the steps [g0, g1), its warps every fourth.
    np = SOLO && rows ? prefix_len(a, b) : 0;
    n = rows ? suffix_len(a, b) : 0;
    ps = (np + kStep - 1) / kStep;
    const int all = ps + (n + kStep - 1) / kStep;
    g0 = int((long long)all * split / pl.suffix_splits);
    g1 = int((long long)all * (split + 1) / pl.suffix_splits);
    steps = rows ? (g1 - g0 + kWarps - 1) / kWarps : 1;
    load(0);
    load(1);

    // Query fragments: row 8 nb + g4 (zero past the live rows), features 16 kk + c2, + 8.
    uint32_t q[NB][D / 16][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = row0 + 8 * nb + g4;
      const bool real = 8 * nb + g4 < rows;
      const bf16* src = a.q + (size_t(b) * a.rows + row / a.group) * a.ldq + size_t(h * a.group + row % a.group) * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        q[nb][kk][0] = real ? *reinterpret_cast<const uint32_t*>(src + 16 * kk + c2) : 0u;
        q[nb][kk][1] = real ? *reinterpret_cast<const uint32_t*>(src + 16 * kk + 8 + c2) : 0u;
      }
    }
    // Rows 8 nb + c2, + 1 of the score fragments: how many suffix keys they see.
    int seen[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = 8 * nb + c2 + u;
        seen[nb][u] = row < rows ? suffix_seen(n, a.rows, (row0 + row) / a.group) : 0;
      }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb][0] = m[nb][1] = -INFINITY;  // unscaled references
      l[nb][0] = l[nb][1] = 0.f;        // this lane's keys only
#pragma unroll
      for (int f = 0; f < D / 16; ++f) o[nb][f][0] = o[nb][f][1] = o[nb][f][2] = o[nb][f][3] = 0.f;
    }
    float* scores = a.sw && pl.pooled ? ws.scores + ((size_t(b) * a.kv_heads + h) * unit_rows + row0) * score_pitch(a) : nullptr;

#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const int g = g0 + i * kWarps + warp;
      const bool pre = g < ps;
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
      if (g >= g1 && rows) continue;  // this warp's last step may be empty
      const int ka = (pre ? g : g - ps) * kStep + g4, kb = ka + 8;
      uint32_t p_hi[NB][2], p_lo[NB][2];
      bool grow = false;
      float top[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 8 * nb + c2 + u, end = row < rows ? (pre ? np : seen[nb][u]) : 0;
          if (scores && row < rows && !pre) {
            if (ka < n) scores[size_t(row) * score_pitch(a) + ka] = s[nb][u];
            if (kb < n) scores[size_t(row) * score_pitch(a) + kb] = s[nb][2 + u];
          }
          if (ka >= end) s[nb][u] = -INFINITY;
          if (kb >= end) s[nb][2 + u] = -INFINITY;
          top[nb][u] = fmaxf(s[nb][u], s[nb][2 + u]);  // of this lane's keys
          grow = grow || (top[nb][u] - m[nb][u]) * scale_log2 > kRescale;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float alpha[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x = top[nb][u];  // of the row's
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const bool up = (x - m[nb][u]) * scale_log2 > kRescale;
            alpha[u] = up ? exp2_approx((m[nb][u] - x) * scale_log2) : 1.f;
            if (up) m[nb][u] = x;
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
  }

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
  float* cta_o = reinterpret_cast<float*>(smem);  // [R][D], then [warps][R][D]; piece c of row r at c ^ (r & 7)
  float* joined = cta_o + R * D;
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
  const size_t part0 = ((size_t(split) * a.batch + b) * a.kv_heads + h) * unit_rows + row0;
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
    if (SOLO) reinterpret_cast<float4*>(cta_o)[i] = v;
    else reinterpret_cast<float4*>(ws.suffix_o + (part0 + row) * D)[(i % (D / 4)) ^ (row & 7)] = v;
  }
  if constexpr (!SOLO) {
    if (t < live) ws.suffix_ml[part0 + t] = make_float2(cta_m[t], cta_l[t]);
    // One block outlasts the tile kernel, so that this kernel's end, which the
    // join waits for, is the end of both; the others make room at once.
    if (blockIdx.x == gridDim.x - 1 && h == int(gridDim.y) - 1 && b == int(gridDim.z) - 1) wait_prior();
    return;
  }
  const int ctas = pl.suffix_splits;
  if (ctas > 1) tc::cluster_sync();
  else __syncthreads();
  static_assert(kMaxSuffixSplits == 8 && R <= 4 * kWarps, "a warp joins four rows of eight parts");
  if (4 * warp < live) {
    const int row = 4 * warp + lane / 8, part = lane % 8;
    float f;
    const RowJoin j = join_four_rows(
        row < live && part < ctas,
        [&] { return make_float2(remote_f32(&cta_m[row], part), remote_f32(&cta_l[row], part)); }, f);
    part_f[row][part] = f;
    if (part == 0 && row < live) {
      row_m[row] = j.m;
      row_r[row] = j.inv;
      if (split == 0) {
        if (a.lse) a.lse[row_index(a, b, h, row0 + row)] = j.lse;
        if (a.pw || (a.sw && !pl.pooled)) ws.norm[row_index(a, b, h, row0 + row)] = RowNorm{j.m, j.inv};
      }
    }
  }
  __syncthreads();
  for (int i = split * kThreads + t; i < live * (D / 4); i += ctas * kThreads) {
    const int row = i / (D / 4);
    float4 y[kMaxSuffixSplits], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kMaxSuffixSplits; ++r)
      if (r < ctas) y[r] = remote_f32x4(cta_o + i * 4, r);
#pragma unroll
    for (int r = 0; r < kMaxSuffixSplits; ++r)
      if (r < ctas) add_part(v, y[r], part_f[row][r]);
    store_piece<D>(a, b, h, row0 + row, (i % (D / 4)) ^ (row & 7), v);
  }
  if (a.sw && pl.pooled)  // of this CTA's suffix keys
    add_suffix_weights(a, ws, scale_log2, b, h, n, max(0, g0 - ps) * kStep, min(n, max(0, g1 - ps) * kStep), row_m, row_r, t,
                       kThreads, [] {});
  if (ctas > 1) tc::cluster_sync();  // no CTA leaves while another reads its shared memory
}

// Joins the prefix ranges and the suffix ranges of each row (3 to 5 us of a
// step of batch 32).  Bound by latency
// (a few KB per block), so the work is spread thin: W warps share a row, each
// every W-th part with all its loads in flight, lane = 16-byte piece of the row;
// every one of them makes the row's factors itself.  With weights, the first
// blocks add the sums of the suffix keys, two warps for each chunk of a
// (sequence, KV head).
constexpr int kJoinThreads = 512;
constexpr int kInFlight = 5;  // parts that a warp has in flight
constexpr int kChunkThreads = 128, kChunkKeys = 512, kChunks = kJoinThreads / kChunkThreads;  // of a block

template <int D, int W>
__global__ void __launch_bounds__(kJoinThreads, 2) shared_join_kernel(const SharedAttnArgs a, const Plan pl,
                                                                  const Workspace ws, const float scale_log2,
                                                                  const int weight_blocks, const int chunks) {
  __shared__ float row_m[kChunks][kFewRows], row_r[kChunks][kFewRows], factors[kJoinThreads / 32][kMaxParts];
  __shared__ float4 sums[kJoinThreads / 32][D / 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit_rows = a.rows * a.group, parts = pl.splits + pl.suffix_splits;
  const size_t stride = size_t(pl.tasks) * pl.per_cta * kRows;            // rows between two prefix ranges
  const size_t suffix_stride = size_t(a.batch) * a.kv_heads * unit_rows;  // and two suffix ranges
  // Row of query head hq of a token: its tile's first row in a prefix range, its
  // place in the tile, its place in a suffix range.
  size_t first, suffix_row;
  int r;
  auto place = [&](int token, int hq) {
    const int h = hq / a.group, tile = token / pl.per_tile;
    r = token % pl.per_tile * a.group + hq % a.group;
    first = (size_t(h * pl.groups + tile / pl.per_cta) * pl.per_cta + tile % pl.per_cta) * kRows;
    suffix_row = (size_t(token / a.rows) * a.kv_heads + h) * unit_rows + token % a.rows * a.group + hq % a.group;
  };
  auto join = [&] {
    return join_row(
        parts,
        [&](int s) {
          return s < pl.splits ? ws.part_ml[first + r + s * stride]
                               : ws.suffix_ml[suffix_row + (s - pl.splits) * suffix_stride];
        },
        factors[warp]);
  };
  wait_prior();
  allow_next();
  if (int(blockIdx.x) < weight_blocks) {
    const int mine = threadIdx.x / kChunkThreads, thread = threadIdx.x % kChunkThreads;
    const int at = blockIdx.x * kChunks + mine, unit = at / chunks, chunk = at % chunks;
    const int h = unit % a.kv_heads, b = unit / a.kv_heads;
    const int n = b < a.batch ? suffix_len(a, b) : 0;
    add_suffix_weights(a, ws, scale_log2, min(b, a.batch - 1), h, n, chunk * kChunkKeys, min(n, (chunk + 1) * kChunkKeys),
                       row_m[mine], row_r[mine], thread, kChunkThreads, [&] {
                         for (int row = thread / 32; row < unit_rows && b < a.batch; row += kChunkThreads / 32) {
                           place(b * a.rows + row / a.group, h * a.group + row % a.group);
                           const RowJoin j = join();
                           if (lane == 0) {
                             row_m[mine][row] = j.m;
                             row_r[mine][row] = j.inv;
                           }
                         }
                         __syncthreads();
                       });
    return;
  }
  const int row = (blockIdx.x - weight_blocks) * (kJoinThreads / 32 / W) + warp / W, sub = warp % W;
  const int token = row / a.query_heads, hq = row % a.query_heads;
  const bool live = token < a.batch * a.rows;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    place(token, hq);
    const float* pre = ws.part_o + first * D + part_offset<D>(r, lane * 4);
    const float* suf = ws.suffix_o + suffix_row * D + lane * 4;
    float4 y[kInFlight];
    auto load = [&](int s0) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int s = s0 + u * W;
        if (s < parts && lane < D / 4)
          y[u] = *reinterpret_cast<const float4*>(s < pl.splits ? pre + s * stride * D
                                                                : suf + (s - pl.splits) * suffix_stride * D);
      }
    };
    load(sub);
    const RowJoin j = join();
    __syncwarp();
#pragma unroll 1
    for (int s0 = sub; s0 < parts; s0 += kInFlight * W) {
      if (s0 != sub) load(s0);
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int s = s0 + u * W;
        if (s < parts) add_part(v, y[u], factors[warp][s]);
      }
    }
    if (lane == 0 && sub == 0) {
      if (a.lse) a.lse[row] = j.lse;
      if (a.pw) ws.norm[row] = RowNorm{j.m, j.inv};
    }
  }
  if constexpr (W > 1) {
    if (lane < D / 4) sums[warp][lane] = v;
    __syncthreads();
  }
  if (live && sub == 0 && lane < D / 4) {
#pragma unroll
    for (int w = 1; w < W; ++w) add_part(v, sums[warp + w][lane], 1.f);
    reinterpret_cast<uint2*>(a.out + size_t(token) * a.ldo + size_t(hq) * D)[lane] =
        make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
  }
}

template <int D, int NB, bool SOLO>
cudaError_t launch_shape(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  constexpr int smem = RowsShape<D, NB>::smem;
  const cudaError_t e = allow_smem<shared_rows_kernel<D, NB, SOLO>>(smem);
  if (e != cudaSuccess) return e;
  const int blocks = (a.rows * a.group + 8 * NB - 1) / (8 * NB);
  DependentLaunch d(dim3(p.suffix_splits * blocks, a.kv_heads, a.batch), kThreads, smem, stream,
                    SOLO ? p.suffix_splits : 1);
  return cudaLaunchKernelEx(&d.cfg, shared_rows_kernel<D, NB, SOLO>, a, p, ws, attention_scale(D) * kLog2e);
}

template <int D, bool SOLO>
cudaError_t launch_width(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  return a.rows * a.group <= 8 ? launch_shape<D, 1, SOLO>(a, p, ws, stream)
                               : launch_shape<D, 2, SOLO>(a, p, ws, stream);
}

template <int D, int W>
cudaError_t launch_join_shape(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  const cudaError_t e = allow_smem<shared_join_kernel<D, W>>(0);
  if (e != cudaSuccess) return e;
  constexpr int at_once = kJoinThreads / 32 / W;
  const long long blocks = ((long long)a.batch * a.rows * a.query_heads + at_once - 1) / at_once;
  const int chunks = a.sw ? (a.scap + kChunkKeys - 1) / kChunkKeys : 0;
  const long long weight_blocks = ((long long)a.batch * a.kv_heads * chunks + kChunks - 1) / kChunks;
  const long long grid = blocks + weight_blocks;
  if (grid > INT_MAX / kChunks) return cudaErrorInvalidValue;
  DependentLaunch d(dim3(unsigned(grid)), kJoinThreads, 0, stream);
  return cudaLaunchKernelEx(&d.cfg, shared_join_kernel<D, W>, a, p, ws, attention_scale(D) * kLog2e,
                            int(weight_blocks), chunks);
}

}  // namespace

cudaError_t launch_rows(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  if (p.splits == 0) return a.width == 64 ? launch_width<64, true>(a, p, ws, stream) : launch_width<128, true>(a, p, ws, stream);
  return a.width == 64 ? launch_width<64, false>(a, p, ws, stream) : launch_width<128, false>(a, p, ws, stream);
}

cudaError_t launch_join(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, int sms, cudaStream_t stream) {
  const bool four = join_cost(double(a.batch) * a.rows * a.query_heads, p.splits + p.suffix_splits, sms).warps == 4;
  if (a.width == 64) return four ? launch_join_shape<64, 4>(a, p, ws, stream) : launch_join_shape<64, 1>(a, p, ws, stream);
  return four ? launch_join_shape<128, 4>(a, p, ws, stream) : launch_join_shape<128, 1>(a, p, ws, stream);
}

}  // namespace sa
}  // namespace dl
