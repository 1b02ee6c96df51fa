// What the kernels of the shared-prefix attention have in common: row and
// length arithmetic, the workspace, tensor-core and copy primitives.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>

#include "shared_attention.h"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace dl {
namespace sa {

constexpr int kRows = 128;   // query rows of a tile = TMEM lanes
constexpr int kKeys = 128;   // keys of a tile
constexpr int kMaxSplits = 32;  // key ranges of a row tile
constexpr int kMaxSuffixSplits = 8;
constexpr int kPair = 2 * kKeys;  // keys of a unit of the weights kernel
constexpr int kMaxWeightParts = 64;
constexpr int kFewRows = 32;    // rows of a unit (new tokens x group) that the few-row kernels take
constexpr int kMostRows = 16;   // and one CTA of them
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A query row's softmax in the base-2 domain: weight = exp2(s * scale - m) * r.
// A row without keys has m = 0, r = 0.
struct RowNorm {
  float m, r;
};

// Workspace: FP32 partial outputs of key ranges, one 128-row tile per (range,
// split task, row tile of it) in the layout of part_offset, their running
// maximum (base 2) and sum, the rows' norms [tokens][Hq] and, for the weights,
// the suffix scores of the few-row kernel.
struct Workspace {
  float* part_o;    // [splits][tasks - full][per_cta][128 x D]
  float2* part_ml;  // [splits][tasks - full][per_cta][128]
  float* suffix_o;    // [suffix splits][B][Hkv][rows x group][D]
  float2* suffix_ml;  // [suffix splits][B][Hkv][rows x group]
  RowNorm* norm;    // [tokens * Hq]
  float* scores;    // [B][Hq * rows][score_pitch]
  float *prefix_sums, *suffix_sums;  // of the weights kernel's parts: [parts][Hkv][keys], [parts][B][Hkv][keys]
};

// Suffix scores of a row, in 16-byte pieces.
__host__ __device__ __forceinline__ int score_pitch(const SharedAttnArgs& a) { return (a.scap + 3) / 4 * 4; }

// How a call is cut into work, from sizes alone.
struct Plan {
  bool pooled;    // row tiles hold tokens of several sequences and cover the prefix; the few-row kernel adds the
                  // suffixes and their weights
  int per_tile;   // tokens of a row tile: 128 / group
  int tiles;      // row tiles of a unit: a KV head (pooled) or a sequence's KV head
  int per_cta;    // 2: two row tiles share a CTA's key tiles; 1: one row tile, key tiles in two interleaved streams
  int groups;     // CTA tasks of a unit: tiles / per_cta, rounded up
  int tasks;      // groups x units
  int full;       // tasks done whole, by the first CTAs; the rest are cut into key ranges
  int splits;     // key ranges of the rest (0: no tile kernel; the few-row kernel reads the prefix too)
  int suffix_splits;  // CTAs (a cluster if there is no tile kernel) per sequence and KV head in the few-row kernel
  int prefix_parts, suffix_parts;  // of the row tiles that a pair of key tiles goes through in the weights kernel
};

// Warps that share a row in the join kernel (four, or one when that would take
// several waves of blocks and there are few parts: 4096 rows of 6 parts 12 us
// with four and 5 us with one, 2048 rows of 22 parts 7 us and 11 us), and the
// time of the join in microseconds.
struct JoinCost {
  int warps;
  double time;
};
inline JoinCost join_cost(double rows, int parts, int sms) {
  const double four = std::max(1.0, rows / (8 * sms)) * (2 + 1.5 * ((parts + 19) / 20));
  const double one = std::max(1.0, rows / (32 * sms)) * (2 + 1.5 * ((parts + 4) / 5));
  return {four <= one ? 4 : 1, std::min(four, one) + 2.56e-4 * rows * parts};
}

cudaError_t launch_tiles(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream);
cudaError_t launch_merge(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream);
cudaError_t launch_rows(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream);
cudaError_t launch_join(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, int sms, cudaStream_t stream);
cudaError_t launch_weights(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, int sms, cudaStream_t stream);

// Launch configuration of a programmatic dependent launch.  The first kernel of
// a call waits for its predecessor before it touches global memory and only then
// lets the next one start, and so on: a later kernel may read the call's inputs
// at once and waits before it touches what the kernels before it write.
struct DependentLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  DependentLaunch(dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster = 1) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = cluster;
      attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
      cfg.numAttrs = 2;
    }
  }
};

// Dynamic shared memory above 48 KB, allowed once per kernel and device; and
// the same split of the SM's memory for every kernel here, all of it shared
// memory: blocks of two kernels fit side by side only within one split, and an
// SM changes its split only when it is empty.
template <auto Kernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};  // devices 0 .. 63
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Tiles of [rows][64 features], one KV head: `per_tile` tokens x the head
// group, and 128 positions of a cache.
inline bool encode_query_map(CUtensorMap* m, const SharedAttnArgs& a, int per_tile) {
  const uint64_t dims[3] = {uint64_t(a.width), uint64_t(a.query_heads), uint64_t(a.batch) * a.rows};
  const uint64_t strides[2] = {uint64_t(a.width), a.ldq};
  const uint32_t box[3] = {64, uint32_t(a.group), uint32_t(per_tile)};
  return encode_bf16_map(m, a.q, 3, dims, strides, box);
}
inline bool encode_prefix_map(CUtensorMap* m, const SharedAttnArgs& a, const bf16* base) {
  const uint64_t dims[3] = {uint64_t(a.width), uint64_t(a.kv_heads), uint64_t(a.pcap)};
  const uint64_t strides[2] = {uint64_t(a.width), a.p_row};
  const uint32_t box[3] = {64, 1, kKeys};
  return encode_bf16_map(m, base, 3, dims, strides, box);
}
// A suffix that all sequences share (sequence stride 0) is a map of one
// sequence: strides of 0 are not for tensor maps.
__host__ __device__ __forceinline__ bool one_suffix(const SharedAttnArgs& a) { return a.batch == 1 || a.s_seq == 0; }
inline bool encode_suffix_map(CUtensorMap* m, const SharedAttnArgs& a, const bf16* base) {
  const bool one = one_suffix(a);
  const uint64_t dims[4] = {uint64_t(a.width), uint64_t(a.kv_heads), uint64_t(a.scap), uint64_t(one ? 1 : a.batch)};
  const uint64_t strides[3] = {uint64_t(a.width), a.s_row, one ? a.s_row * a.scap : a.s_seq};
  const uint32_t box[4] = {64, 1, kKeys, 1};
  return encode_bf16_map(m, base, 4, dims, strides, box);
}

__device__ __forceinline__ int clamp_len(long long n, int cap) { return int(n < 0 ? 0 : n > cap ? cap : n); }
__device__ __forceinline__ int prefix_len(const SharedAttnArgs& a, int b) {
  return a.pcap ? clamp_len(a.plens[b], a.pcap) : 0;
}
__device__ __forceinline__ int suffix_len(const SharedAttnArgs& a, int b) {
  return a.scap ? clamp_len(a.slens[b], a.scap) : 0;
}
// Suffix keys that row i sees of a suffix of n keys.
__device__ __forceinline__ int suffix_seen(int n, int rows, int i) { return max(0, n - (rows - 1 - i)); }

// Feature f of row r within a partial tile: two halves of the features, row by
// row, 16-byte piece c of a row's half at c ^ (r & 7) (so that neither the
// staging of rows by threads nor the bulk copy meets bank conflicts).
template <int D>
__device__ __forceinline__ int part_offset(int r, int f) {
  const int half = f / (D / 2), c = f % (D / 2) / 4;
  return (half * kRows + r) * (D / 2) + ((c ^ (r & 7)) << 2) + (f & 3);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs of FP32 numbers in one 64-bit register (one instruction for both).
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Two softmax weights as BF16 pairs hi + lo: the upper halves of the numbers
// and of what they leave, so hi + lo is good to 2^-14 (the dropped rest is
// below 2^-7 of lo, lo below 2^-7 of the weight) and the second product, run
// with both, keeps the accuracy of FP32 weights.  One BF16 rounding alone,
// 2^-8, would cost as much as the rounding of the output itself.  Byte
// permutes instead of conversions, which share the exponential's slow pipe.
__device__ __forceinline__ void split_bf16(uint64_t ab, uint32_t& hi, uint32_t& lo) {
  float a, b, ra, rb;
  unpair(ab, a, b);
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  hi = __byte_perm(x, y, 0x7632);
  const uint64_t rest = add2(ab, pair(__uint_as_float((x & 0xffff0000u) ^ 0x80000000u),
                                      __uint_as_float((y & 0xffff0000u) ^ 0x80000000u)));
  unpair(rest, ra, rb);
  lo = __byte_perm(__float_as_uint(ra), __float_as_uint(rb), 0x7632);
}

// True in one lane of a converged warp; the compiler then knows that a single
// thread issues (a tensor instruction under `lane == 0` issues at half the rate).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Position in a ring of N buffers and the parity of the pass over it.
template <int N>
struct RingPos {
  int slot = 0;
  unsigned parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      parity ^= 1;
    }
  }
};

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
      "%5}], [%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
      : "memory");
}

// MN-major operand with 128-byte swizzle (64 contiguous elements of M or N per
// 128-byte row, one row per K): leading offset between 64-element columns,
// 1024 bytes between groups of 8 K.
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t addr, uint32_t column_bytes) {
  return tc::smem_desc_sw128(addr) & ~(uint64_t(0x3FFF) << 16) | (uint64_t(column_bytes >> 4) << 16);
}

// D (TMEM) += A (TMEM, BF16 pairs) * B (shared memory).
__device__ __forceinline__ void mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of this warp's lanes, not yet waited for.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Waits for the loads issued so far; the values in r are only valid after it.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Wait of one role of a warp-specialised kernel: bounded (~2 s), and over at
// once when another role already gave up.  *failed is shared memory.
__device__ __forceinline__ bool role_wait(uint64_t* bar, unsigned parity, volatile int* failed) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  while (!*failed) {
    if (mbar_try_wait(bar, parity)) return true;
    if (clock64() - start > (1ll << 32)) break;
  }
  *failed = 1;
  return false;
}

// The same for a whole warp: one answer for all lanes, which stay together.
__device__ __forceinline__ bool role_wait_warp(uint64_t* bar, unsigned parity, volatile int* failed) {
  return __all_sync(0xffffffffu, role_wait(bar, parity, failed));
}

}  // namespace sa
}  // namespace dl
