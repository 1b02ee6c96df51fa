// Attention of a batch of sequences over one shared prefix cache and their
// own suffix caches, and the sums of the weight each key receives:
//
//   s[t, h, j] = q[t, h] . k[j, h / group] / sqrt(d),  lse = log sum_j exp(s),
//   out = sum_j exp(s - lse) v[j],  weight[j] += sum over t, h of exp(s - lse)
//
// This file decides how a call is cut and launches its one to four kernels,
// each a programmatic dependent of the one before:
//
//   few new tokens per sequence (rows x group <= 32, a decode step): the tile
//   kernel over the prefix with the rows of all sequences pooled, beside it the
//   few-row kernel over every suffix, the join kernel for the two; the weights
//   kernel for the prefix sums (the join kernel adds the suffix sums);
//   small calls: the few-row kernel alone over prefix and suffix, 16 rows per
//   CTA, and the weights kernel (for the suffixes too with more rows);
//   more (a turn, a document): the tile kernel per sequence over prefix and
//   suffix, the merge kernel if key ranges were split, the weights kernel.
#include "shared_attention.cuh"

#include <algorithm>

namespace dl {
namespace {

using namespace sa;

// How a call is cut is chosen by an estimate of its time in microseconds, from
// the capacities (lengths are on the device), with constants measured on a B200
// (148 SMs; 32 query and 8 KV heads of width 128 unless said otherwise) with
// full caches: room beyond the lengths leads to plans for suffixes that are not
// there (batch 32 on 8192 keys, suffixes of up to 256 in a capacity of 256 22.2,
// of 1024 24.4, of 2048 39.3, of 4096 50.5).  The alternatives measured against
// one another, in a graph of 18 calls at 1965 MHz:
//
//   few-row kernel alone / beside tiles, one token: batch 8 on 1024 + 64 keys
//     10.9 / 12.9, batch 64 on 256 + 64 14.0 / 13.1 (taken: alone); batch 2 on
//     8192 + 64 23.8 / 19.2, batch 16 on 2048 + 64 21.1 / 13.8
//   few-row kernel alone / tiles per sequence: one sequence of 88 tokens, 8
//     query heads, on 291 + 91 keys 10.7 / 13.6; 2 of 33 on 1000 + 64 23.5 / 17.1
//   few rows beside tiles / tiles per sequence: batch 32 of one token on 8192 +
//     256 keys 27 / 178, batch 8 of 8 tokens on 8192 + 256 28 / 57; batch 16 of
//     8 tokens on 1024 + 128 19.5 / 18.9
//   key ranges of the pooled tiles, batch 64 of one token on 32768 + 2048 keys
//     (16 row tiles), the best suffix cut of each: 2 196, 3 144, 4 117, 5 115, 6
//     115, 9 125; suffixes of half that on average 175, 123, 97, 86, 92, 96:
//     with more ranges fewer SMs are left for the suffixes to stream through
//   one / two row tiles per CTA: batch 8 of 48 tokens on 4096 + 112 keys 49.0
//     (whole) / 58.7 (two ranges); batch 8 of 512 on 8192 + 512 637 / 615
inline int ceil_div(long long a, long long b) { return int((a + b - 1) / b); }

// Tiles of row tiles alone (a turn, a document): sets per_cta, groups, tasks,
// full and splits.  A step is a pair of a row tile and a key tile on each
// stream, 2.3 us; a split costs the merge kernel and 42 ns per 128-row part.
double plan_tiles(const SharedAttnArgs& a, int key_tiles, int units, int sms, Plan* best) {
  double best_cost = 0;
  for (int per_cta = 1; per_cta <= (best->tiles > 1 ? 2 : 1); ++per_cta) {
    Plan p = *best;
    p.per_cta = per_cta;
    p.groups = ceil_div(p.tiles, per_cta);
    p.tasks = p.groups * units;
    // Whole tasks fill the SMs as often as they can; what is left is cut into
    // key ranges that fill them once more, if that pays.
    const int whole = p.tasks / sms * sms, rest = p.tasks - whole;
    auto steps = [&](int splits) { return per_cta == 2 ? ceil_div(key_tiles, splits) : ceil_div(key_tiles, 2 * splits); };
    for (int s = 1; s <= std::max(1, std::min({rest ? sms / rest : 1, key_tiles / 2, kMaxSplits})); ++s) {
      const int waves = ceil_div(p.tasks, sms);
      const double cost = 7 + (per_cta == 2 ? 2.3 : 2.37) * (double(whole / sms) * steps(1) + (rest ? steps(s) : 0)) +
                          4 * (waves - 1) + (s > 1 ? 3 + 0.042 * s * rest * per_cta * a.width / 128 : 0);
      if (best_cost && cost >= best_cost) continue;
      best_cost = cost;
      p.splits = s;
      p.full = s == 1 ? p.tasks : whole;
      *best = p;
    }
  }
  return best_cost;
}

// The few-row kernel alone: sets suffix_splits.  A step is 64 keys of a CTA, of
// which four (three of 16 rows) fit an SM.
double plan_solo(const SharedAttnArgs& a, int units, int sms, Plan* best) {
  const bool many = a.rows * a.group > 8;
  const int fit = many ? 3 : 4;
  const long long blocks = (long long)units * ceil_div(a.rows * a.group, many ? kMostRows : 8);
  double best_cost = 0;
  for (int s = 1; s <= kMaxSuffixSplits; s *= 2) {
    const int waves = ceil_div(blocks * s, fit * sms), beside = std::min(fit, ceil_div(blocks * s, sms));
    const double start = many ? 4.8 + 0.8 * beside : 3.4 + 0.4 * beside;
    const double step = (many ? 0.85 + 0.4 * beside : std::max(1.05, 0.45 * beside)) * a.width / 128;
    const double cost = waves * (start + step * ceil_div(a.scap + a.pcap, 64 * s)) + (s > 1 ? 1 : 0);
    if (best_cost && cost >= best_cost) continue;
    best_cost = cost;
    best->suffix_splits = s;
  }
  return best_cost;
}

// The few-row kernel over the suffixes beside the tile kernel over the prefix:
// sets splits and suffix_splits.  An SM holds a tile CTA and a few-row CTA, or
// four of the latter.
double plan_beside(const SharedAttnArgs& a, int key_tiles, int units, int sms, Plan* best) {
  const double width = a.width / 128.0, few = a.rows * a.group > 8 ? 1.5 : 1;
  const double rows = double(a.batch) * a.rows * a.query_heads;
  const double bytes = (double(a.pcap) + double(a.batch) * a.scap) * a.kv_heads * a.width * 4;
  const int blocks = units * ceil_div(a.rows * a.group, a.rows * a.group > 8 ? kMostRows : 8);
  double best_cost = 0;
  for (int splits = 1; splits <= std::max(1, std::min({sms / best->tasks, (key_tiles + 1) / 2, kMaxSplits})); ++splits) {
    const int ctas = best->tasks * splits, waves = ceil_div(ctas, sms);
    const double tile = 6.3 + waves * (0.7 + 3.2 * ceil_div(key_tiles, 2 * splits));
    const int slots = waves == 1 ? ctas + 4 * (sms - ctas) : sms;
    for (int s = 1; s <= kMaxSuffixSplits; s *= 2) {
      const double one = few * (2.8 + 1.6 * width * ceil_div(a.scap, 64 * s));
      double suffix = one * ceil_div((long long)blocks * s, slots);
      if (suffix > tile) suffix = std::max(one, tile + (suffix - tile) * slots / (4 * sms));
      const double cost = std::max({tile, suffix, bytes / 6.9e6}) + join_cost(rows, splits + s, sms).time * width;
      if (best_cost && cost >= best_cost) continue;
      best_cost = cost;
      best->splits = splits;
      best->suffix_splits = s;
    }
  }
  return best_cost;
}

// The parts of the row tiles in the weights kernel, for both caches: the least
// work of the busiest CTA, which takes every sms-th unit, in tiles of 128 rows
// against a pair of key tiles (2.3 us); a unit costs half a tile besides, adding
// the parts up one and a half.  41 sequences of 150 tokens, 2 heads per KV head,
// on 71 keys take 199 us in one part (two CTAs take all rows past the prefix),
// 54 in 8, 41 in 33; 8 of 48 tokens on 4096 keys 81 in one, 85 in 4, 93 in 8.
void plan_weights(const SharedAttnArgs& a, int sms, Plan* p) {
  const long long prefix = (long long)ceil_div(a.pcap, kPair) * a.kv_heads;
  const long long suffix = p->pooled ? 0 : (long long)ceil_div(a.scap, kPair) * a.kv_heads * a.batch;
  const int prefix_rows = ceil_div((long long)a.batch * a.rows, p->per_tile), suffix_rows = ceil_div(a.rows, p->per_tile);
  double best_cost = 0;
  for (int parts = 1; parts <= std::min(prefix_rows, kMaxWeightParts); ++parts) {
    const int longest = ceil_div(prefix_rows, parts);
    const int of_suffix = suffix ? std::min(kMaxWeightParts, ceil_div(suffix_rows, longest)) : 1;
    const long long first = prefix * parts, all = first + suffix * of_suffix;
    auto load = [&](long long cta) {
      const int mine = ceil_div(std::max(0ll, first - cta), sms), rest = ceil_div(std::max(0ll, all - cta), sms) - mine;
      return mine * (longest + 0.5) + rest * (ceil_div(suffix_rows, of_suffix) + 0.5);
    };
    const double cost = std::max(load(0), load(first % sms)) + (parts > 1 || of_suffix > 1 ? 1.5 : 0);
    if (best_cost && cost >= best_cost) continue;
    best_cost = cost;
    p->prefix_parts = parts;
    p->suffix_parts = of_suffix;
  }
}

Plan plan_of(const SharedAttnArgs& a, bool weights, int sms) {
  const int tokens = a.batch * a.rows, units = a.batch * a.kv_heads;
  const int prefix_tiles = ceil_div(a.pcap, kKeys), suffix_tiles = ceil_div(a.scap, kKeys);
  Plan p = {};
  p.per_tile = kRows / a.group;
  p.tiles = ceil_div(a.rows, p.per_tile);
  p.suffix_splits = 1;
  double cost = plan_tiles(a, prefix_tiles + suffix_tiles, units, sms, &p);
  if (a.rows * a.group <= kFewRows) {
    Plan q = p;
    q.pooled = true;
    q.tiles = q.groups = ceil_div(tokens, q.per_tile);
    q.tasks = q.tiles * a.kv_heads;
    q.per_cta = 1;
    q.full = 0;
    const double beside = plan_beside(a, prefix_tiles, units, sms, &q);
    if (beside < cost) {
      p = q;
      cost = beside;
    }
  }
  Plan solo = p;
  const double alone = plan_solo(a, units, sms, &solo);
  if (alone < cost) {
    p = solo;
    p.pooled = a.rows * a.group <= kMostRows;  // rows of several CTAs cannot add a key's weight together
    p.splits = 0;
    p.full = p.tasks;
  }
  p.prefix_parts = p.suffix_parts = 1;
  if (weights) plan_weights(a, sms, &p);
  return p;
}

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

// Lays the workspace out at `base`; returns its size.
size_t lay_out(const SharedAttnArgs& a, const Plan& p, bool weights, char* base, Workspace* ws) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* at_ptr = base + at;
    at += round_up(bytes);
    return at_ptr;
  };
  const size_t part_rows = size_t(p.splits) * (p.tasks - p.full) * p.per_cta * kRows;
  const size_t rows = size_t(a.batch) * a.rows * a.query_heads;
  const size_t suffix_rows = p.pooled && p.splits ? rows * p.suffix_splits : 0;
  ws->part_o = reinterpret_cast<float*>(take(part_rows * a.width * 4));
  ws->part_ml = reinterpret_cast<float2*>(take(part_rows * 8));
  ws->suffix_o = reinterpret_cast<float*>(take(suffix_rows * a.width * 4));
  ws->suffix_ml = reinterpret_cast<float2*>(take(suffix_rows * 8));
  ws->norm = reinterpret_cast<RowNorm*>(take(weights ? rows * 8 : 0));
  const size_t prefix_keys = p.prefix_parts > 1 ? size_t(ceil_div(a.pcap, kPair)) * kPair : 0;
  const size_t suffix_keys = p.suffix_parts > 1 && !p.pooled ? size_t(ceil_div(a.scap, kPair)) * kPair : 0;
  ws->prefix_sums = reinterpret_cast<float*>(take(p.prefix_parts * a.kv_heads * prefix_keys * 4));
  ws->suffix_sums = reinterpret_cast<float*>(take(size_t(p.suffix_parts) * a.batch * a.kv_heads * suffix_keys * 4));
  ws->scores = reinterpret_cast<float*>(take(weights && p.pooled ? rows * score_pitch(a) * 4 : 0));
  return std::max<size_t>(at, 256);
}

}  // namespace

size_t shared_attention_workspace_bytes(const SharedAttnArgs& a, bool weights, int sms) {
  Workspace ws;
  return lay_out(a, plan_of(a, weights, sms), weights, nullptr, &ws);
}

cudaError_t launch_shared_attention(const SharedAttnArgs& a, void* workspace, int sms, cudaStream_t stream) {
  const bool weights = a.pw || a.sw;
  const Plan p = plan_of(a, weights, sms);
  Workspace ws;
  lay_out(a, p, weights, static_cast<char*>(workspace), &ws);
  cudaError_t e = p.splits ? launch_tiles(a, p, ws, stream) : cudaSuccess;
  if (e == cudaSuccess && (p.pooled || !p.splits)) e = launch_rows(a, p, ws, stream);
  if (e == cudaSuccess && p.pooled && p.splits) e = launch_join(a, p, ws, sms, stream);
  if (e == cudaSuccess && !p.pooled && p.full < p.tasks) e = launch_merge(a, p, ws, stream);
  if (e == cudaSuccess && (a.pw || (a.sw && !p.pooled))) e = launch_weights(a, p, ws, sms, stream);
  return e;
}

}  // namespace dl
