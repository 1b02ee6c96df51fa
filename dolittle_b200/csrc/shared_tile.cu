// Tensor-core kernel of the shared-prefix attention: 128-row tiles of query
// rows against 128-key tiles, online softmax, on tcgen05.
//
// The rows of a tile are tokens x the query heads of one KV head.  Pooled
// tiles take the tokens of several sequences (a decode step's batch), so the
// prefix is read once for all of them; otherwise a tile's tokens belong to one
// sequence and its key tiles run through the prefix and on into that
// sequence's suffix.  Roles of a CTA: one warp loads tiles by TMA into a ring,
// one issues the products, and two groups of four warps ("streams") own the
// softmax of a 128 x 128 score tile each, one thread per row.  Wide CTAs give
// the streams two row tiles that share the key tiles; with a single row tile
// the streams take alternate key tiles and are joined at the end.  While one
// stream is in its softmax the tensor core works for the other:
//
//   S[x] = Q K^T       (both operands in shared memory, K-major)
//   P[x] = exp2(S * scale - m), two BF16 halves written over S[x] in TMEM
//   O[x] += (Phi + Plo)[x] V   (P from TMEM, V as it lies in the cache: the
//                       MN-major form of the operand needs no transposed copy)
//
// S[x] of the next key tile is issued behind O[x] += P[x] V: products run in
// issue order, so it cannot overwrite P[x] early, and when S[x] is ready O[x]
// is too.  The row's reference m only moves when its maximum has grown by more
// than 2^8, then the thread rescales its row of O in TMEM; sums stay FP32 far
// from overflow.  The tensor core wants P in the type of V: P is split in two
// BF16 numbers, half again as many products, for FP32's accuracy.
//
// Bound by the tensor core: a 128 x 128 tile of width 128 takes 824 cycles of
// Q K^T (both operands from shared memory, 103 cycles per 128 x 128 x 16 where
// the products alone are 64) and 1024 of P V, two of them 3700; measured 3960
// to 4300 for a pair.  Eight sequences of 512 tokens on 8192 + 512 keys, 32
// heads of 128: 620 us with the SMs at 1965 MHz, 914 TFLOP/s of useful work and
// 1371 with the second half of P; called in a row 714 us, 794 TFLOP/s, since the
// power cap then holds the SMs at 1.6 GHz.  Calls of one or two steps are bound
// by the start instead: 9.6 us for 5 x 74 tokens on 28 + 101 keys.
#include "shared_attention.cuh"

namespace dl {
namespace sa {
namespace {

using namespace tc;

constexpr int kThreads = 352;  // 8 softmax warps, one each for loads, products and clearing
constexpr int kTmaWarp = 8, kMmaWarp = 9, kClearWarp = 10;
constexpr int kAtom = kRows * 128;  // [128 rows][64 BF16]
constexpr uint32_t kTmemCols = 512;  // S0, S1, O0, O1
constexpr float kRescale = 8.f;     // base-2 growth of the maximum that moves the reference

// WIDE: two row tiles share the key tiles, which halves the bytes through L2 per
// product; otherwise one row tile (which CTA shape a call gets is planned in
// shared_attention.cu, with both measured).  BESIDE: one row tile in a CTA that
// leaves room for one of the few-row kernel on its SM (65 KB of shared memory,
// a quarter of the registers), which then streams the suffixes while this one
// is busy with products.
template <int D, bool WIDE, bool BESIDE>
struct Shape {
  static_assert(!(WIDE && BESIDE), "room for a few-row block is left by one row tile only");
  static constexpr int slot = D / 64 * kAtom;  // a K, V or Q tile
  static constexpr int queries = WIDE ? 2 : 1;
  // Parts in which the weights of a tile are handed over: products begin sooner
  // with four (batch 64 on 32768 keys 87.8 -> 85.4 us, turns of 48 tokens 51.4 ->
  // 49.1), but two cost less where the tensor core is busy (tails of 512 tokens
  // 620.5 against 629; all at 1965 MHz).
  static constexpr int parts = WIDE ? 2 : 4;
  static constexpr int stages = D == 64 ? 8 : WIDE ? 5 : 4;
  static constexpr int smem = (queries + stages) * slot + 1024;
  static constexpr int bound = BESIDE ? 512 : kThreads;  // threads that the registers are shared out for
};

struct alignas(64) TileArgs {
  CUtensorMap q, pk, pv, sk, sv;
  SharedAttnArgs a;
  Plan plan;
  Workspace ws;
  float scale_log2;
  bool norms;  // write the rows' norms (the weights follow)
};

template <int D>
__device__ __forceinline__ void mma_scores(uint32_t tmem_s, uint32_t q_tile, uint32_t k_tile) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t atom = uint32_t(kk >> 2) * kAtom;
    const uint64_t off = uint64_t((kk & 3) * 2);
    mma_bf16(tmem_s, smem_desc_sw128(q_tile + atom) + off, smem_desc_sw128(k_tile + atom) + off,
             instr_desc_bf16(kRows, kKeys), kk ? 1u : 0u);
  }
}

// A half or a quarter of the key tile's keys (kk of 8 steps of 16).
template <int D, int PARTS>
__device__ __forceinline__ void mma_output(uint32_t tmem_o, uint32_t tmem_p, uint32_t v_tile, int part,
                                           bool accumulate) {
  constexpr uint32_t idesc = instr_desc_bf16(kRows, D) | (1u << 16);  // B is MN-major
#pragma unroll
  for (int i = 0; i < 8 / PARTS; ++i) {
    const int kk = 8 / PARTS * part + i;
    const uint64_t v = smem_desc_sw128_mn(v_tile + uint32_t(kk * 2048), kAtom);
    const uint32_t p = tmem_p + uint32_t((kk >> 1) * 32 + (kk & 1) * 8);  // 32 keys: 16 columns hi, 16 lo
    mma_bf16_ts(tmem_o, p, v, idesc, (accumulate || i) ? 1u : 0u);
    mma_bf16_ts(tmem_o, p + 16, v, idesc, 1u);
  }
}

// ONE: all sequences share one suffix cache.  A kernel of its own, since the
// loading thread asking for it cost the others 3 % (turns of 48 tokens on 4096
// keys 48.4 -> 50.0 us).
template <int D, bool WIDE, bool BESIDE, bool ONE>
__global__ void __launch_bounds__(Shape<D, WIDE, BESIDE>::bound, 1)
    shared_tile_kernel(const __grid_constant__ TileArgs t) {
  using S = Shape<D, WIDE, BESIDE>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t q_full, full[S::stages], empty[S::stages], s_full[2], p_part[2][S::parts], o_full[2];
  __shared__ uint64_t begun, dirty, clean, drained;
  __shared__ uint32_t dirty_from, dirty_to;  // bytes of a value tile's first 64 features to clear
  __shared__ uint32_t tmem_slot;
  __shared__ int most[2];  // keys of the prefix / suffix that any row sees
  __shared__ int failed_s;
  __shared__ float2 stream_ml[2][kRows];
  volatile int* failed = &failed_s;
  const SharedAttnArgs& a = t.a;
  const Plan& pl = t.plan;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring = base + S::queries * S::slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Task of this CTA (row tiles fastest, so CTAs side by side read the same
  // keys), whole or one of its key ranges.
  const int cta = blockIdx.x, rest = pl.tasks - pl.full;
  const int task = cta < pl.full ? cta : pl.full + (cta - pl.full) % rest;
  const int split = cta < pl.full ? 0 : (cta - pl.full) / rest, splits = cta < pl.full ? 1 : pl.splits;
  const int tile0 = task % pl.groups * pl.per_cta, h = task / pl.groups % a.kv_heads;
  const int seq = task / pl.groups / a.kv_heads;  // 0 when pooled
  const int unit_tokens = pl.pooled ? a.batch * a.rows : a.rows;
  const int streams = WIDE && tile0 + 1 >= pl.tiles ? 1 : 2;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int i = 0; i < S::stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      for (int j = 0; j < S::parts; ++j) mbar_init(&p_part[x][j], 4);
      mbar_init(&o_full[x], 1);
    }
    mbar_init(&begun, 1);
    mbar_init(&dirty, 1);
    mbar_init(&clean, 1);
    mbar_init(&drained, 1);
    failed_s = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_slot, kTmemCols);
  if (warp == kTmaWarp && lane == 0) {
    prefetch_map(&t.q);
    if (a.pcap) prefetch_map(&t.pk), prefetch_map(&t.pv);
    if (a.scap && !BESIDE) prefetch_map(&t.sk), prefetch_map(&t.sv);
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_slot;

  // Row of a softmax thread.
  const int x = (warp >> 2) & 1, r = threadIdx.x & (kRows - 1);
  const int tile = WIDE ? tile0 + x : tile0;
  const int local = tile * pl.per_tile + r / a.group;  // token within the unit
  const bool live = warp < kTmaWarp && r / a.group < pl.per_tile && local < unit_tokens && tile < pl.tiles;
  const int token = pl.pooled ? local : seq * a.rows + local;
  int np = 0, k0 = 0, n = 0;  // prefix tiles; the range's tiles
  // Every role calls this before it touches what other kernels wrote.  The
  // loading warp finds how far the rows see, so that the first tiles are under
  // way while the softmax warps still fetch their code.
  auto begin = [&] {
    wait_prior();
    allow_next();  // after the wait: the next kernel may read what this one's inputs are before it waits itself
    if (warp == kTmaWarp) {
      const int end = min((tile0 + (WIDE ? streams : 1)) * pl.per_tile, unit_tokens);  // the CTA's tokens
      int p = 0, s = 0;
      if (pl.pooled) {
        for (int b = tile0 * pl.per_tile / a.rows + lane; b <= (end - 1) / a.rows; b += 32) p = max(p, prefix_len(a, b));
        p = __reduce_max_sync(0xffffffffu, p);
      } else {
        p = prefix_len(a, seq);
        s = suffix_seen(suffix_len(a, seq), a.rows, end - 1);
      }
      if (lane == 0) {
        most[0] = p;
        most[1] = s;
        mbar_arrive(&begun);
      }
      __syncwarp();
    }
    if (!role_wait_warp(&begun, 0, failed)) return;  // n stays 0
    np = (most[0] + kKeys - 1) / kKeys;
    const int nt = np + (most[1] + kKeys - 1) / kKeys;
    k0 = int((long long)nt * split / splits);
    n = int((long long)nt * (split + 1) / splits) - k0;
  };
  // Key tiles of stream s, and the i-th one's place among the n.
  auto count = [&](int s) { return WIDE ? (s < streams ? n : 0) : (n + 1 - s) / 2; };
  auto nth = [&](int s, int i) { return WIDE ? i : 2 * i + s; };
  // Keys of the i-th tile that exist; a tile that holds fewer than 128 ends its side.
  auto filled = [&](int i) {
    const int g = k0 + i;
    return g < np ? most[0] - g * kKeys : most[1] - (g - np) * kKeys;
  };

  if (warp == kTmaWarp) {
    begin();
    const int steps = count(0);  // count(1) is at most that
    if (n > 0 && elect_one()) {
      const int boxes = D / 64, q_bytes = pl.per_tile * a.group * 128 * boxes;
      RingPos<S::stages> at;
      unsigned c = 0;
      auto load = [&](int i, bool value) {
        if (c >= S::stages && !role_wait(&empty[at.slot], at.parity ^ 1, failed)) return false;
        uint64_t* bar = &full[at.slot];
        mbar_arrive_expect_tx(bar, unsigned(S::slot));
        unsigned char* dst = smem_raw + (ring + at.slot * S::slot - smem_addr(smem_raw));
        const int g = k0 + i;
        for (int b = 0; b < boxes; ++b) {
          if (g < np) tma_3d(dst + b * kAtom, value ? &t.pv : &t.pk, 64 * b, h, g * kKeys, bar);
          else tma_4d(dst + b * kAtom, value ? &t.sv : &t.sk, 64 * b, h, (g - np) * kKeys, ONE ? 0 : seq, bar);
        }
        at.next();
        ++c;
        return true;
      };
      mbar_arrive_expect_tx(&q_full, unsigned(q_bytes * (WIDE ? streams : 1)));
      for (int s = 0; s < (WIDE ? streams : 1); ++s)
        for (int b = 0; b < boxes; ++b)
          tma_3d(smem_raw + (base + s * S::slot + b * kAtom - smem_addr(smem_raw)), &t.q, 64 * b, h * a.group,
                 (pl.pooled ? 0 : seq * a.rows) + (tile0 + s) * pl.per_tile, &q_full);
      // The order in which the products use them.
      const int feeds = WIDE ? 1 : 2;
      bool ok = true;
      for (int s = 0; s < feeds && ok; ++s)
        if (count(s) > 0) ok = load(nth(s, 0), false);
      for (int i = 0; i < steps && ok; ++i)
        for (int s = 0; s < feeds && ok; ++s) {
          if (i < count(s)) ok = load(nth(s, i), true);
          if (ok && i + 1 < count(s)) ok = load(nth(s, i + 1), false);
        }
      if (!ok) {  // gave up: the copies in flight still land in this CTA's memory
        mbar_wait(&q_full, 0);
        for (unsigned j = c > S::stages ? c - S::stages : 0; j < c; ++j)
          mbar_wait(&full[j % S::stages], (j / S::stages) & 1);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    begin();
    const int steps = count(0);
    if (n > 0 && elect_one()) {
      RingPos<S::stages> at;
      unsigned cleared = 0;
      bool ok = role_wait(&q_full, 0, failed);
      auto slot_addr = [&](int slot) { return ring + uint32_t(slot) * S::slot; };
      auto wait_key = [&] {
        ok = ok && role_wait(&full[at.slot], at.parity, failed);
        fence_after_sync();
      };
      auto wait_value = [&](int i) {
        ok = ok && role_wait(&full[at.slot], at.parity, failed);
        const int left = filled(i);
        if (ok && left < kKeys) {
          dirty_from = slot_addr(at.slot) + uint32_t(left) * 128;
          dirty_to = slot_addr(at.slot) + kAtom;
          mbar_arrive(&dirty);
          ok = role_wait(&clean, cleared++ & 1, failed);
        }
        fence_after_sync();
      };
      auto scores = [&](int s, int slot) {
        mma_scores<D>(tmem + s * kKeys, base + (WIDE ? s : 0) * S::slot, slot_addr(slot));
        mma_commit(&s_full[s]);
      };
      auto output = [&](int s, int slot, int i) {
        const uint32_t o = tmem + 256 + s * 128, p = tmem + s * kKeys, v = slot_addr(slot);
#pragma unroll
        for (int j = 0; j < S::parts; ++j) {
          ok = role_wait(&p_part[s][j], i & 1, failed);
          fence_after_sync();
          if (!ok) return;
          mma_output<D, S::parts>(o, p, v, j, i > 0 || j > 0);
        }
      };
      if constexpr (WIDE) {
        wait_key();
        if (ok) {
          for (int s = 0; s < streams; ++s) scores(s, at.slot);
          mma_commit(&empty[at.slot]);
          at.next();
        }
        for (int i = 0; i < n && ok; ++i) {
          wait_value(i);
          const int v = at.slot;
          at.next();
          for (int s = 0; s < streams && ok; ++s) {
            output(s, v, i);
            if (!ok) break;
            if (s == streams - 1) mma_commit(&empty[v]);
            if (i + 1 == n) {
              mma_commit(&o_full[s]);
              continue;
            }
            if (s == 0) wait_key();
            if (!ok) break;
            scores(s, at.slot);
            if (s == streams - 1) mma_commit(&empty[at.slot]);
          }
          if (i + 1 < n) at.next();
        }
      } else {
        for (int s = 0; s < 2; ++s) {
          if (!ok || count(s) == 0) continue;
          wait_key();
          if (!ok) break;
          scores(s, at.slot);
          mma_commit(&empty[at.slot]);
          at.next();
        }
        for (int i = 0; i < steps && ok; ++i)
          for (int s = 0; s < 2 && ok; ++s) {
            if (i >= count(s)) continue;
            wait_value(nth(s, i));
            if (ok) output(s, at.slot, i);
            if (!ok) break;
            mma_commit(&empty[at.slot]);
            at.next();
            if (i + 1 == count(s)) {
              mma_commit(&o_full[s]);
              continue;
            }
            wait_key();
            if (!ok) break;
            scores(s, at.slot);
            mma_commit(&empty[at.slot]);
            at.next();
          }
      }
      if (!ok) {  // products in flight read shared memory and write TMEM
        mma_commit(&drained);
        mbar_wait(&drained, 0);
      }
    }
    __syncwarp();
  } else if (warp == kClearWarp) {
    // Value rows past every length hold anything: times a weight of zero they
    // would still count, so the products wait until they are zeros.
    begin();
    unsigned events = 0;
    for (int i = 0; i < n; ++i) events += filled(i) < kKeys;
    for (unsigned e = 0; e < events; ++e) {
      if (!role_wait_warp(&dirty, e & 1, failed)) break;
      for (int b = 0; b < D / 64; ++b)
        for (uint32_t o = dirty_from + b * kAtom + lane * 16; o < dirty_to + b * kAtom; o += 512)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(o), "r"(0) : "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&clean);
    }
  } else if (warp < kTmaWarp) {
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + 256 + x * 128;
    const float c = t.scale_log2;
    float m = -INFINITY, l = 0.f;  // m: unscaled reference of the row
    int seen_p = 0, seen_s = 0;    // keys the row sees
    bool ok = true;
    // Turn -1 (BESIDE) runs the code once on whatever the tensor memory holds,
    // while the kernel before this one ends and the first tiles load: a decode
    // step has only a few turns, and fetching the loop from memory that other
    // kernels' data went through took longer than they do (batch 32 on 8192
    // keys: 4900 and 3400 cycles for the two passes of the first turn, 720 and
    // 2400 after it).
#pragma unroll 1
    for (int i = BESIDE ? -1 : 0;; ++i) {
      if (i == 0) {
        begin();
        if (live) {
          seen_p = prefix_len(a, token / a.rows);
          if (!pl.pooled) seen_s = suffix_seen(suffix_len(a, seq), a.rows, local);
        }
        m = -INFINITY;
        l = 0.f;
      }
      if (i >= 0 && i >= count(x)) break;
      const int g = k0 + nth(x, i);
      // The scores' columns; in turn -1 those of the output, which nothing uses
      // before this warp has handed over its first weights.
      const uint32_t t_s = i < 0 ? t_o : tmem + lanes + x * kKeys;
      int lim = kKeys;  // keys of the tile this row sees
      if (i >= 0) {
        lim = g < np ? seen_p - g * kKeys : seen_s - (g - np) * kKeys;
        ok = role_wait_warp(&s_full[x], i & 1, failed);
        if (!ok) break;
        fence_after_sync();
      }
      const bool masked = __any_sync(0xffffffffu, lim < kKeys);
      // BESIDE: two rolled passes over the scores, 32 at a time, for a quarter of
      // the registers and of the code (a decode step runs each loop only a few
      // times, so fetching unrolled code would take longer than running it).
      // Otherwise all 128 scores in registers, unrolled.
      constexpr int held = BESIDE ? 1 : 4;
      uint32_t s[held][32];
      auto mask = [&](int j) {
        if (masked) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (32 * j + k >= lim) s[j % held][k] = 0xff800000u;  // -infinity
        }
      };
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      auto raise = [&](int j) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          mx[k & 3] =
              fmaxf(mx[k & 3], fmaxf(__uint_as_float(s[j % held][k]), __uint_as_float(s[j % held][16 + k])));
      };
      if constexpr (BESIDE) {
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          tmem_ld32_async(t_s + 32 * j, s[0]);
          tmem_ld_wait32(s[0]);
          mask(j);
          raise(j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) tmem_ld32_async(t_s + 32 * j, s[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          tmem_ld_wait32(s[j]);
          mask(j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) raise(j);
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = (top - m) * c > kRescale;  // also from -infinity
      if (i <= 0) {
        m = top;
      } else if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? exp2_approx((m - top) * c) : 1.f;
#pragma unroll 1
        for (int j = 0; j < D / 32; ++j) {
          uint32_t o[32];
          tmem_ld32_async(t_o + 32 * j, o);
          tmem_ld_wait32(o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tmem_st32(t_o + 32 * j, o);
        }
        l *= alpha;
        if (grow) m = top;
      }
      const float shift = m == -INFINITY ? 0.f : -m * c;
      const uint64_t c2 = pair(c, c), shift2 = pair(shift, shift);
      uint64_t sum[4] = {0, 0, 0, 0};
      auto weights = [&](int j) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x0, x1;
          unpair(fma2(pair(__uint_as_float(s[j % held][2 * k]), __uint_as_float(s[j % held][2 * k + 1])), c2, shift2),
                 x0, x1);
          const uint64_t e = pair(exp2_approx(x0), exp2_approx(x1));
          sum[k & 3] = add2(sum[k & 3], e);
          split_bf16(e, hi[k], lo[k]);
        }
        tmem_st16(t_s + 32 * j, hi);  // over the 32 scores just used
        tmem_st16(t_s + 32 * j + 16, lo);
        constexpr int chunks = 4 / S::parts;
        if (j % chunks == chunks - 1) {  // a part is there: its products may begin
          tmem_st_wait();
          fence_before_sync();
          __syncwarp();
          if (lane == 0 && i >= 0) mbar_arrive(&p_part[x][j / chunks]);
        }
      };
      if constexpr (BESIDE) {
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          tmem_ld32_async(t_s + 32 * j, s[0]);
          tmem_ld_wait32(s[0]);
          mask(j);
          weights(j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) weights(j);
      }
      float s0, s1;
      unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
      l += s0 + s1;
    }
    // Both streams' products must be over before the operands become scratch.
    for (int s = 0; s < 2; ++s)
      if (count(s) > 0) ok = role_wait_warp(&o_full[s], 0, failed) && ok;
    fence_after_sync();
    // A wide stream ends its own row; the two narrow ones hold parts of one
    // row, and each thread ends half of its features.
    float m2 = m == -INFINITY ? -INFINITY : m * c, f[2] = {1.f, 0.f};
    if constexpr (!WIDE) {
      stream_ml[x][r] = make_float2(m2, l);
      named_sync(1, 2 * kRows);
      const float2 p = stream_ml[0][r], q = stream_ml[1][r];
      m2 = fmaxf(p.x, q.x);
      f[0] = p.x == -INFINITY ? 0.f : exp2_approx(p.x - m2);
      f[1] = q.x == -INFINITY ? 0.f : exp2_approx(q.x - m2);
      l = p.y * f[0] + q.y * f[1];
    } else if (m == -INFINITY) {
      f[0] = 0.f;
    }
    ok = ok && !*failed;
    if (!ok) l = NAN;
    constexpr int columns = WIDE ? D : D / 2;
    const int from = WIDE ? 0 : x * columns;
    const uint32_t t_o0 = tmem + lanes + 256 + (WIDE ? x * 128 : 0) + from;
    auto features = [&](int j, float* v) {  // features from + 32 j ..
      uint32_t o[32];
      __syncwarp();
      tmem_ld32_async(t_o0 + 32 * j, o);
      tmem_ld_wait32(o);
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = f[0] != 0.f ? __uint_as_float(o[k]) * f[0] : 0.f;
      if constexpr (!WIDE) {
        __syncwarp();
        tmem_ld32_async(t_o0 + 128 + 32 * j, o);
        tmem_ld_wait32(o);
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = f[1] != 0.f ? fmaf(__uint_as_float(o[k]), f[1], v[k]) : v[k];
      }
    };
    if (!BESIDE && splits == 1) {  // the whole softmax of the row
      const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
      const int hq = h * a.group + r % a.group;
      bf16* out = a.out + size_t(token) * a.ldo + size_t(hq) * D + from;
#pragma unroll 1
      for (int j = 0; j < columns / 32; ++j) {
        float v[32];
        features(j, v);
        if (live) {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            reinterpret_cast<uint4*>(out)[4 * j + k / 8] =
                make_uint4(pack_bf16(v[k] * inv, v[k + 1] * inv), pack_bf16(v[k + 2] * inv, v[k + 3] * inv),
                           pack_bf16(v[k + 4] * inv, v[k + 5] * inv), pack_bf16(v[k + 6] * inv, v[k + 7] * inv));
        }
      }
      if (live && (WIDE || x == 0)) {
        const size_t row = size_t(token) * a.query_heads + hq;
        if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m2 + log2f(l)) * kLn2;
        if (t.norms) t.ws.norm[row] = l == 0.f ? RowNorm{0.f, 0.f} : RowNorm{m2, inv};
      }
    } else if (tile < pl.tiles) {
      // One range's part, staged in shared memory and copied out in bulk.
      const size_t part = (size_t(split) * rest + task - pl.full) * pl.per_cta + (WIDE ? x : 0);
      const uint32_t stage = base + uint32_t((WIDE ? x * D : from) * kRows * 4);
      if (WIDE || x == 0) t.ws.part_ml[part * kRows + r] = make_float2(m2, l);
#pragma unroll 1
      for (int j = 0; j < columns / 32; ++j) {
        float v[32];
        features(j, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = 8 * j + k, half = i / (D / 8);
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                           stage + uint32_t((half * kRows + r) * (D * 2) + (((i % (D / 8)) ^ (r & 7)) << 4))),
                       "f"(v[4 * k]), "f"(v[4 * k + 1]), "f"(v[4 * k + 2]), "f"(v[4 * k + 3])
                       : "memory");
        }
      }
      fence_proxy_async_smem();
      named_sync(2 + x, kRows);
      if (r == 0) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(t.ws.part_o +
                                                                                          (part * D + from) * kRows),
                     "r"(stage), "r"(kRows * columns * 4)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
      }
    }
    fence_before_sync();
  }
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

// Joins the key ranges of the split tasks: a warp takes four rows (token, query
// head) of a tile at once, all their loads in flight together, lanes hold a
// row's features; the ranges in order.  Bound by the parts' way to L2 and back:
// with writing them 8 us for 128 parts of 128 x 128 and 13 us for 256 (16.8 MB;
// one row per warp at a time 4 us more).
constexpr int kMergeRows = 4, kMergeWarps = 4;

template <int D>
__global__ void __launch_bounds__(32 * kMergeWarps) shared_merge_kernel(const SharedAttnArgs a, const Plan pl,
                                                                       const Workspace ws, bool norms) {
  constexpr int F = D / 32;  // consecutive features of a lane
  const int lane = threadIdx.x & 31, row0 = (blockIdx.x * kMergeWarps + (threadIdx.x >> 5)) * kMergeRows;
  const int rest = pl.tasks - pl.full, task = pl.full + row0 / kRows / pl.per_cta;
  const int tile = task % pl.groups * pl.per_cta + row0 / kRows % pl.per_cta, h = task / pl.groups % a.kv_heads;
  const size_t stride = size_t(rest) * pl.per_cta * kRows;  // rows between two ranges
  wait_prior();
  allow_next();
  const int first = row0 % kRows;
  const float* src = ws.part_o + size_t(row0 / kRows) * kRows * D;
  float2 ml[kMergeRows];
  float top[kMergeRows], l[kMergeRows], o[kMergeRows][F];
#pragma unroll
  for (int j = 0; j < kMergeRows; ++j) {
    ml[j] = lane < pl.splits ? ws.part_ml[row0 + j + lane * stride] : make_float2(-INFINITY, 0.f);
    l[j] = 0.f;
#pragma unroll
    for (int c = 0; c < F; ++c) o[j][c] = 0.f;
  }
  auto load = [&](int s, float (&v)[kMergeRows][F]) {
#pragma unroll
    for (int j = 0; j < kMergeRows; ++j) {
      const float* p = src + s * stride * D + part_offset<D>(first + j, lane * F);
      if constexpr (F == 4) {
        const float4 y = *reinterpret_cast<const float4*>(p);
        v[j][0] = y.x, v[j][1] = y.y, v[j][2] = y.z, v[j][3] = y.w;
      } else {
        const float2 y = *reinterpret_cast<const float2*>(p);
        v[j][0] = y.x, v[j][1] = y.y;
      }
    }
  };
  float v[2][kMergeRows][F];
  load(0, v[0]);
#pragma unroll
  for (int j = 0; j < kMergeRows; ++j) {
    top[j] = ml[j].x;
#pragma unroll
    for (int k = 16; k; k >>= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], k));
    ml[j].x = ml[j].x == -INFINITY ? 0.f : exp2_approx(ml[j].x - top[j]);  // now the range's factor
  }
  auto add = [&](int s, const float (&v)[kMergeRows][F]) {
#pragma unroll
    for (int j = 0; j < kMergeRows; ++j) {
      const float f = __shfl_sync(0xffffffffu, ml[j].x, s);
      l[j] = fmaf(__shfl_sync(0xffffffffu, ml[j].y, s), f, l[j]);
#pragma unroll
      for (int c = 0; c < F; ++c) o[j][c] = fmaf(v[j][c], f, o[j][c]);
    }
  };
#pragma unroll 1
  for (int s = 0; s < pl.splits; s += 2) {
    if (s + 1 < pl.splits) load(s + 1, v[1]);
    add(s, v[0]);
    if (s + 2 < pl.splits) load(s + 2, v[0]);
    if (s + 1 < pl.splits) add(s + 1, v[1]);
  }
#pragma unroll
  for (int j = 0; j < kMergeRows; ++j) {
    const int r = first + j, local = tile * pl.per_tile + r / a.group;
    if (r / a.group >= pl.per_tile || local >= a.rows) continue;
    const int token = task / pl.groups / a.kv_heads * a.rows + local, hq = h * a.group + r % a.group;
    const float inv = l[j] > 0.f ? 1.f / l[j] : l[j] == 0.f ? 0.f : NAN;
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + size_t(token) * a.ldo + size_t(hq) * D + lane * F);
#pragma unroll
    for (int c = 0; c < F; c += 2) out[c / 2] = pack_bf16(o[j][c] * inv, o[j][c + 1] * inv);
    if (lane == 0) {
      const size_t at = size_t(token) * a.query_heads + hq;
      if (a.lse) a.lse[at] = l[j] == 0.f ? -INFINITY : (top[j] + log2f(l[j])) * kLn2;
      if (norms) ws.norm[at] = l[j] == 0.f ? RowNorm{0.f, 0.f} : RowNorm{top[j], inv};
    }
  }
}

template <int D, bool WIDE, bool BESIDE, bool ONE = false>
cudaError_t launch_tiles_shape(const TileArgs& t, cudaStream_t stream) {
  constexpr int smem = Shape<D, WIDE, BESIDE>::smem;
  const cudaError_t e = allow_smem<shared_tile_kernel<D, WIDE, BESIDE, ONE>>(smem);
  if (e != cudaSuccess) return e;
  const unsigned grid = unsigned(t.plan.full + (t.plan.tasks - t.plan.full) * t.plan.splits);
  DependentLaunch d(dim3(grid), kThreads, smem, stream);
  return cudaLaunchKernelEx(&d.cfg, shared_tile_kernel<D, WIDE, BESIDE, ONE>, t);
}

template <int D>
cudaError_t launch_tiles_width(const TileArgs& t, cudaStream_t stream) {
  if (t.plan.pooled) return launch_tiles_shape<D, false, true>(t, stream);
  if (t.a.scap && t.a.batch > 1 && t.a.s_seq == 0)
    return t.plan.per_cta == 2 ? launch_tiles_shape<D, true, false, true>(t, stream)
                               : launch_tiles_shape<D, false, false, true>(t, stream);
  return t.plan.per_cta == 2 ? launch_tiles_shape<D, true, false>(t, stream)
                             : launch_tiles_shape<D, false, false>(t, stream);
}

}  // namespace

cudaError_t launch_tiles(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  TileArgs t = {};
  t.a = a;
  t.plan = p;
  t.ws = ws;
  t.scale_log2 = attention_scale(a.width) * kLog2e;
  t.norms = a.pw || a.sw;
  if (!encode_query_map(&t.q, a, p.per_tile)) return cudaErrorInvalidValue;
  if (a.pcap && !(encode_prefix_map(&t.pk, a, a.pk) && encode_prefix_map(&t.pv, a, a.pv))) return cudaErrorInvalidValue;
  if (a.scap && !p.pooled && !(encode_suffix_map(&t.sk, a, a.sk) && encode_suffix_map(&t.sv, a, a.sv)))
    return cudaErrorInvalidValue;
  return a.width == 64 ? launch_tiles_width<64>(t, stream) : launch_tiles_width<128>(t, stream);
}

cudaError_t launch_merge(const SharedAttnArgs& a, const Plan& p, const Workspace& ws, cudaStream_t stream) {
  DependentLaunch d(dim3(unsigned(p.tasks - p.full) * p.per_cta * (kRows / (kMergeRows * kMergeWarps))),
                    32 * kMergeWarps, 0, stream);
  const bool norms = a.pw || a.sw;
  const cudaError_t e =
      a.width == 64 ? allow_smem<shared_merge_kernel<64>>(0) : allow_smem<shared_merge_kernel<128>>(0);
  if (e != cudaSuccess) return e;
  return a.width == 64 ? cudaLaunchKernelEx(&d.cfg, shared_merge_kernel<64>, a, p, ws, norms)
                       : cudaLaunchKernelEx(&d.cfg, shared_merge_kernel<128>, a, p, ws, norms);
}

}  // namespace sa
}  // namespace dl
