#include "paged_attention_tc.cuh"

namespace htr {

// The other kernel passes over the cache once per 16 rows; this one takes up to 128 of them for the same time, but begins and joins more slowly.
// In the long run they are level at about 50 rows of 128 dimensions and 90 of 64; and below some 0.9e9 elements of scores times dimensions (of the
// tables' whole width: lengths are not known here) the other is ahead.  Measured behind a flush of L2, us, the other / this one: 64 requests over
// 2000, 2 heads of 128: 32 rows 48 / 66, 48 rows 65 / 67, 64 rows 79 / 67, 128 rows 138 / 67, 256 rows 257 / 77; of 64 dimensions: 64 rows 54 / 63, 96 rows
// 71 / 65, 128 rows 89 / 63, 256 rows 161 / 71; one request over 8000, 2 heads of 128, 256 rows: 30 / 42; 9 over 5000: 64 rows 38 / 42, 128 rows 56 / 42.
bool attention_tc_serves(int tokens, int requests, int q_heads, int group, int max_new, long long width, int head_dim) {
  return requests <= kMaxRequests && group <= kRows && (long long)group * max_new * head_dim > 6144 &&
         (double)tokens * q_heads * (double)width * head_dim > 0.9e9;
}

size_t attention_tc_workspace(int head_dim) {
  return (size_t)current_device_sms() * (sizeof(int4) + 2 * sizeof(float) * (head_dim == 128 ? kPartFloats<128> : kPartFloats<64>));
}

int attention_tc_run(const AttentionArgs& a, int dtype, int head_dim, void* workspace, cudaStream_t st) { return run_of<8>(a, dtype, head_dim, workspace, st); }

}  // namespace htr
