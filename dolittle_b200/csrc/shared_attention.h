// Attention of a batch that shares a prefix (shared_attention.cu and the
// kernels it plans: shared_tile.cu, shared_rows.cu, shared_weights.cu).
#pragma once

#include "launch.h"

namespace dl {

struct SharedAttnArgs {
  const bf16* q;
  bf16* out;
  float* lse;  // natural log, [tokens][Hq], or nullptr
  int batch, rows, query_heads, kv_heads, width, group;
  size_t ldq, ldo;  // elements between tokens
  const bf16 *pk, *pv;
  int pcap;
  size_t p_row;
  const long long* plens;
  const bf16 *sk, *sv;
  int scap;
  size_t s_row, s_seq;
  const long long* slens;
  float* pw;  // [Hkv][pcap] or nullptr
  float* sw;  // [B][Hkv][scap] or nullptr
};

size_t shared_attention_workspace_bytes(const SharedAttnArgs& a, bool weights, int sms);
cudaError_t launch_shared_attention(const SharedAttnArgs& a, void* workspace, int sms, cudaStream_t stream);

}  // namespace dl
