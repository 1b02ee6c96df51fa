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
//   kernel for the prefix sums (the join kernel adds the suffix sums).  Small
//   calls: the few-row kernel alone over prefix and suffix.
//   more (a turn, a document): the tile kernel per sequence over prefix and
//   suffix, the merge kernel if key ranges were split, the weights kernel.
#include "shared_attention.cuh"

#include <algorithm>

namespace dl {
namespace {

using namespace sa;

// Prefix elements, over all sequences, up to which reading the prefix once per
// sequence from L2 costs less than a second kernel.
constexpr size_t kSoloElements = size_t(4) << 20;

// CTAs per (sequence, KV head) of the few-row kernel: the fewest waves x time
// of a CTA, in units of a step of 64 keys at the HBM rate shared by three
// resident CTAs (about 2.2 us); start and join cost about 1.4 such steps.
int suffix_splits(long long units, int keys, int slots) {
  int best = 1;
  double best_cost = 0;
  for (int s = 1; s <= kMaxSuffixSplits; s *= 2) {
    const double waves = double((units * s + slots - 1) / slots), steps = (keys + 64 * s - 1) / (64 * s);
    const double cost = waves * (steps + 1.4);
    if (s == 1 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

Plan plan_of(const SharedAttnArgs& a, bool weights, int sms) {
  Plan p = {};
  const int tokens = a.batch * a.rows;
  p.per_tile = kRows / a.group;
  p.pooled = a.rows * a.group <= kFewRows;
  const int unit_tokens = p.pooled ? tokens : a.rows;
  p.tiles = (unit_tokens + p.per_tile - 1) / p.per_tile;
  const int units = a.batch * a.kv_heads;
  p.per_cta = p.tiles > 1 ? 2 : 1;
  p.groups = (p.tiles + p.per_cta - 1) / p.per_cta;
  p.tasks = p.groups * (p.pooled ? a.kv_heads : units);
  const int prefix_tiles = (a.pcap + kKeys - 1) / kKeys, suffix_tiles = (a.scap + kKeys - 1) / kKeys;
  const int key_tiles = prefix_tiles + (p.pooled ? 0 : suffix_tiles);
  // Whole tasks fill the SMs as often as they can; what is left is cut into
  // key ranges (of two key tiles at least) that fill them once more.  Pooled
  // tasks are always joined with a suffix, so they are all cut alike.
  p.full = p.pooled ? 0 : p.tasks / sms * sms;
  const int rest = p.tasks - p.full;
  p.splits = std::max(1, std::min({sms / std::max(1, rest), key_tiles / 2, kMaxSplits}));
  // No more ranges than their longest one needs to stay as short as it is.
  const int longest = (key_tiles + p.splits - 1) / p.splits;
  const int step = p.per_cta == 2 ? longest : (longest + 1) / 2 * 2;  // two streams share a narrow task's key tiles
  if (key_tiles) p.splits = std::min(p.splits, (key_tiles + step - 1) / step);
  if (!p.pooled && p.splits == 1) p.full = p.tasks;
  // (Not with rows for two CTAs, which could not add a key's weight together.)
  if (p.pooled && a.rows * a.group <= kMostRows && units * size_t(a.pcap) * a.width <= kSoloElements) p.splits = 0;
  const int unit_keys = a.scap + (p.splits ? 0 : a.pcap);
  p.suffix_splits = p.pooled ? suffix_splits(units, unit_keys, 3 * sms) : 1;
  p.weight_ranks = 1;
  if (weights) {
    const long long key_units =  // pairs of key tiles
        ((prefix_tiles + 1) / 2 + (long long)(p.pooled ? 0 : (suffix_tiles + 1) / 2) * a.batch) * a.kv_heads;
    const int row_tiles = (tokens + p.per_tile - 1) / p.per_tile;
    while (p.weight_ranks < 8 && key_units * p.weight_ranks * 2 <= sms && row_tiles >= 2 * p.weight_ranks)
      p.weight_ranks *= 2;
  }
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
  ws->scores = reinterpret_cast<float*>(take(weights && p.pooled ? rows * a.scap * 4 : 0));
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
  if (e == cudaSuccess && p.pooled) e = launch_rows(a, p, ws, stream);
  if (e == cudaSuccess && p.pooled && p.splits) e = launch_join(a, p, ws, stream);
  if (e == cudaSuccess && !p.pooled && p.full < p.tasks) e = launch_merge(a, p, ws, stream);
  if (e == cudaSuccess && (a.pw || (a.sw && !p.pooled))) e = launch_weights(a, p, ws, sms, stream);
  return e;
}

}  // namespace dl
