// Attention of a batch of sequences over one shared prefix cache and their
// own suffix caches, and the sums of the weight each key receives:
//
//   s[t, h, j] = q[t, h] . k[j, h / group] / sqrt(d),  lse = log sum_j exp(s),
//   out = sum_j exp(s - lse) v[j],  weight[j] += sum over t, h of exp(s - lse)
//
// This file decides how a call is cut and launches its two to three kernels,
// each a programmatic dependent of the one before:
//
//   few new tokens per sequence (rows x group <= 32, a decode step): the tile
//   kernel over the prefix with the rows of all sequences pooled, beside it the
//   few-row kernel over every suffix, which then joins the two; the weights
//   kernel for the prefix sums (the few-row kernel adds the suffix sums).
//   more (a turn, a document): the tile kernel per sequence over prefix and
//   suffix, the merge kernel if key ranges were split, the weights kernel.
#include "shared_attention.cuh"

#include <algorithm>

namespace dl {
namespace {

using namespace sa;

constexpr int kFewRows = 32;

Plan plan_of(const SharedAttnArgs& a, bool weights, int sms) {
  Plan p = {};
  const int tokens = a.batch * a.rows;
  p.per_tile = kRows / a.group;
  p.pooled = a.rows * a.group <= kFewRows;
  const int unit_tokens = p.pooled ? tokens : a.rows;
  p.tiles = (unit_tokens + p.per_tile - 1) / p.per_tile;
  p.units = p.pooled ? a.kv_heads : a.kv_heads * a.batch;
  p.wide = p.tiles > 1;
  const int prefix_tiles = (a.pcap + kKeys - 1) / kKeys, suffix_tiles = (a.scap + kKeys - 1) / kKeys;
  const int key_tiles = prefix_tiles + (p.pooled ? 0 : suffix_tiles);
  const int ctas = (p.wide ? (p.tiles + 1) / 2 : p.tiles) * p.units;
  // Key ranges until one CTA per SM is reached; a range has two key tiles at least.
  p.splits = key_tiles == 0 ? 0 : std::max(1, std::min({sms / std::max(1, ctas), key_tiles / 2, 32}));
  p.suffix_splits = 1;
  const int units = a.batch * a.kv_heads;
  while (p.pooled && p.suffix_splits < 8 && units * p.suffix_splits < 4 * sms && a.scap >= 256 * p.suffix_splits)
    p.suffix_splits *= 2;
  p.weight_ranks = 1;
  if (weights) {
    const long long key_units = (long long)(prefix_tiles + (p.pooled ? 0 : suffix_tiles * a.batch)) * a.kv_heads;
    const int row_tiles = (tokens + p.per_tile - 1) / p.per_tile;
    while (p.weight_ranks < 8 && key_units * p.weight_ranks < sms && row_tiles >= 2 * p.weight_ranks)
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
  const bool parts = p.pooled || p.splits > 1;
  const size_t part_rows = parts ? size_t(p.splits) * p.units * p.tiles * kRows : 0;
  const size_t rows = size_t(a.batch) * a.rows * a.query_heads;
  ws->part_o = reinterpret_cast<float*>(take(part_rows * a.width * 4));
  ws->part_ml = reinterpret_cast<float2*>(take(part_rows * 8));
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
  if (e == cudaSuccess && !p.pooled && p.splits > 1) e = launch_merge(a, p, ws, stream);
  if (e == cudaSuccess && (a.pw || (a.sw && !p.pooled))) e = launch_weights(a, p, ws, stream);
  return e;
}

}  // namespace dl
