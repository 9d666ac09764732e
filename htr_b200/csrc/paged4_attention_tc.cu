#include "paged_attention_tc.cuh"

namespace htr {

// The other kernel (paged4_kernels.cu) passes over the cache once per 16 rows, but its passes find it in L2 and its thread blocks are many and soon begun; this one
// begins and joins slowly, some 35 us in all.  They are level at about 192 rows of 128 dimensions and 384 of 64, of calls of 1.4e9 elements of scores
// times dimensions (of the tables' whole width: lengths are not known here).  Measured behind a flush of L2, us, the other / this one: 64 requests over up to 2000, 2
// heads of 128: 128 rows 41 / 61, 256 rows 68 / 65, 512 rows 119 / 90; of 64 dimensions: 256 rows 43 / 53, 512 rows 74 / 76, 1024 rows 133 / 109; one over 8000, 2 heads of 128: 512
// rows 35 / 45, 1024 rows 51 / 47; 8 heads: 128 rows 35 / 34, 256 rows 53 / 41; one over 500, 8 heads: 1024 rows 33 / 35, 2048 rows 55 / 43.
// What the rule does not see: tables far wider than their lengths (one piece of 256 tokens behind 500 under a table of 131072, 32 heads of 128 on 8, in a chain: 29 / 32; 64 tokens: 14 / 21), and
// one large piece beside single tokens, whose few rows then fill tiles of 256 (64 tokens beside 63 requests of one, all behind 4000: 100 / 347; 1024 tokens: 434 / 450).
bool attention4_tc_serves(int tokens, int requests, int q_heads, int group, int max_new, long long width, int head_dim) {
  return requests <= kMaxRequests && group <= kRows && (long long)group * max_new * head_dim > 24576 &&
         (double)tokens * q_heads * (double)width * head_dim > 1.4e9;
}

int attention4_tc_run(const AttentionArgs& a, int dtype, int head_dim, void* workspace, cudaStream_t st) { return run_of<4>(a, dtype, head_dim, workspace, st); }

}  // namespace htr
