#include "paged_attention_tc.cuh"

namespace htr {

bool attention4_tc_serves(int tokens, int requests, int q_heads, int group, int max_new, long long width, int head_dim) {
  return attention_tc_serves(tokens, requests, q_heads, group, max_new, width, head_dim);
}

int attention4_tc_run(const AttentionArgs& a, int dtype, int head_dim, void* workspace, cudaStream_t st) { return run_of<4>(a, dtype, head_dim, workspace, st); }

}  // namespace htr
