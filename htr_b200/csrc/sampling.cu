// Sampling of one token per row of logits from a given uniform number: temperature, top-k, top-p and min-p.
//
// The tokens of a row are ordered by logit, ties by index.  With w = exp((logit - max) / temperature) each filter keeps a beginning of
// that order: top-k the first k; top-p the shortest beginning of those whose weight reaches p times theirs; min-p all with w >= min_p;
// together the shortest of the three, at least one token.  The token is then the first in the order of the vocabulary at which
// the running weight of the kept ones exceeds u times their sum.
//
// Borders decide about whole tokens, so weights are 64-bit integers, 2^42 exp(x) with exp in double: their sums are exact and do not
// depend on who adds them, and a border can differ from that of real numbers only where u or p lies within 2^-42 of it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/htr_b200.h"
#include "htr_common.cuh"

namespace {

thread_local int t_last_cuda = 0;

struct SampleArgs {
  const void* logits;
  long long row_stride;
  int dtype, rows, vocab;
  const float *u, *temperature;
  const int* top_k;
  const float *top_p, *min_p;
  long long* tokens;
  float* logprobs;
};

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr double kOne = 4398046511104.0;                   // 2^42: sums of up to 2^20 weights fit in 62 bits
using u64 = unsigned long long;

// unsigned order of floats; NaN and -infinity are 0, below everything that can be chosen
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  if (!(x > -__builtin_huge_valf())) return 0;
  return b == 0x80000000u ? 0x80000000u : b & 0x80000000u ? ~b : b | 0x80000000u;     // (-0 is 0)
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

__device__ __forceinline__ float load_logit(const void* row, int dtype, int i) {
  if (dtype == HTR_DTYPE_F32) return static_cast<const float*>(row)[i];
  const uint16_t raw = static_cast<const uint16_t*>(row)[i];
  return dtype == HTR_DTYPE_BF16 ? __uint_as_float((uint32_t)raw << 16) : __half2float(*reinterpret_cast<const __half*>(&raw));
}

struct Weigh {
  double max, inv;
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    if (key == 0) return 0;
    const double x = (double)logit_of(key);
    if (x == max) return (u64)kOne;
    if (isinf(max)) return 0;
    return (u64)rint(exp((x - max) * inv) * kOne);
  }
};

// f * w for 0 <= f < 1, exactly: rounded down, or up
__device__ __forceinline__ u64 part_of(u64 w, float f, bool up) {
  if (!(f > 0.f)) return 0;
  int e;
  const u64 bits = (u64)ldexpf(frexpf(f, &e), 24);         // f = bits * 2^(e - 24), e <= 0
  const u64 hi = __umul64hi(w, bits), lo = w * bits;       // below 2^86
  const int down = 24 - e;
  if (down >= 64) return up && w ? 1 : down < 128 && hi >> (down - 64);
  return (hi << (64 - down) | lo >> down) + (up && (lo & (((u64)1 << down) - 1)) != 0);
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(htr::kFullWarp, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  V t = 0;
  for (int i = 0; i < kWarps; ++i) t += red[i];
  return t;
}

// exclusive sum over the threads before this one
template <typename V>
__device__ __forceinline__ V block_before(V v, V* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(htr::kFullWarp, s, o);
    if (lane >= o) s += x;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  V t = 0;
  for (int i = 0; i < warp; ++i) t += red[i];
  return t + s - v;
}

// One thread block per row, several passes over it (the row stays in L2).
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
  __shared__ u64 red[kWarps];
  __shared__ u64 s_mass[256];
  __shared__ unsigned s_count[256];
  __shared__ u64 s_pick[4];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int r = blockIdx.x, tid = threadIdx.x, V = a.vocab;
  const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.row_stride * (a.dtype == HTR_DTYPE_F32 ? 4 : 2);
  const auto key_at = [&](int i) { return key_of(load_logit(row, a.dtype, i)); };
  // ---- the largest, and the first index that has it
  u64 top = 0;
  for (int i = tid; i < V; i += kThreads) {
    const u64 v = (u64)key_at(i) << 32 | (0xFFFFFFFFu - i);
    top = v > top ? v : top;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 v = __shfl_xor_sync(htr::kFullWarp, top, o);
    top = v > top ? v : top;
  }
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) top = red[i] > top ? red[i] : top;
  __syncthreads();
  const uint32_t top_key = (uint32_t)(top >> 32);
  const float t = a.temperature ? a.temperature[r] : 1.f;
  if (top_key == 0 || !(t > 0.f)) {                        // nothing to choose from; greedy
    if (tid == 0) {
      a.tokens[r] = top_key == 0 ? -1 : (long long)(0xFFFFFFFFu - (uint32_t)top);
      if (a.logprobs) a.logprobs[r] = top_key == 0 ? __int_as_float(0x7FC00000) : 0.f;
    }
    return;
  }
  const Weigh weigh = {(double)logit_of(top_key), 1.0 / (double)t};
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, least = a.min_p ? a.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < V, by_p = p < 1.f;
  // ---- the border: all above `border_key` are kept, and the first `border_ties` of those that equal it
  uint32_t border_key = 0;
  int border_ties = 0x7FFFFFFF;
  // finds the border at which the count reaches `count` or the weight reaches `mass`
  const auto find = [&](bool counts, u64 target, u64* mass_within) {
    uint32_t prefix = 0, mask = 0;
    u64 before = 0, count_before = 0, mass_before = 0;     // of keys above the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) {
        s_mass[tid] = 0;
        s_count[tid] = 0;
      }
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t key = key_at(i);
        if ((key & mask) != prefix || key < border_key) continue;
        const int bin = key >> shift & 255;
        atomicAdd(&s_count[bin], 1u);
        const u64 w = weigh(key);
        if (w) atomicAdd(&s_mass[bin], w);
      }
      __syncthreads();
      if (tid == 0) {
        int bin = 255;
        u64 sum = before, n = count_before, mass = mass_before;
        for (; bin > 0; --bin) {
          const u64 next = sum + (counts ? s_count[bin] : s_mass[bin]);
          if (next >= target) break;
          sum = next;
          n += s_count[bin];
          mass += s_mass[bin];
        }
        s_pick[0] = bin;
        s_pick[1] = sum;
        s_pick[2] = n;
        s_pick[3] = mass;
      }
      __syncthreads();
      prefix |= (uint32_t)s_pick[0] << shift;
      mask |= 255u << shift;
      before = s_pick[1];
      count_before = s_pick[2];
      mass_before = s_pick[3];
      __syncthreads();
    }
    // ties at the border: each weighs the same
    const u64 each = weigh(prefix), missing = target > before ? target - before : 0;
    u64 ties = counts ? missing : each ? (missing + each - 1) / each : 0x7FFFFFFF;
    if (ties < 1) ties = 1;
    if (ties > 0x7FFFFFFF) ties = 0x7FFFFFFF;
    if (prefix > border_key || (prefix == border_key && (int)ties < border_ties)) {
      border_key = prefix;
      border_ties = (int)ties;
    }
    *mass_within = mass_before + each * ties;
  };
  u64 all = 0;
  if (by_k) {
    find(true, (u64)k, &all);
  } else if (by_p) {
    for (int i = tid; i < V; i += kThreads) all += weigh(key_at(i));
    all = block_sum(all, red);
  }
  if (by_p) {
    u64 target = part_of(all, p, true), ignored;
    if (target < 1) target = 1;
    find(false, target, &ignored);
  }
  if (least > 0.f) {                                       // equal keys weigh the same: the border moves by whole keys
    const double bound = (double)fminf(least, 1.f) * kOne;
    uint32_t lowest = 0xFFFFFFFFu;
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t key = key_at(i);
      if (key && (double)weigh(key) >= bound) lowest = key < lowest ? key : lowest;
    }
    lowest = __reduce_min_sync(htr::kFullWarp, lowest);
    if ((tid & 31) == 0) red[tid >> 5] = lowest;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) lowest = (uint32_t)red[i] < lowest ? (uint32_t)red[i] : lowest;
    __syncthreads();
    if (lowest > border_key) {
      border_key = lowest;
      border_ties = 0x7FFFFFFF;
    }
  }
  // ---- the token: a thread takes consecutive tokens
  const int each = (V + kThreads - 1) / kThreads, first = min(tid * each, V), last = min(first + each, V);
  unsigned ties = 0;
  for (int i = first; i < last; ++i) ties += key_at(i) == border_key;
  const unsigned ties_before = (unsigned)block_before((u64)ties, red);
  const auto kept = [&](uint32_t key, unsigned& tie) {
    if (key > border_key) return weigh(key);
    if (key < border_key || key == 0) return (u64)0;
    return tie++ < (unsigned)border_ties ? weigh(key) : (u64)0;
  };
  u64 mine = 0;
  unsigned tie = ties_before;
  for (int i = first; i < last; ++i) mine += kept(key_at(i), tie);
  const u64 total = block_sum(mine, red), before = block_before(mine, red);
  const float u = fminf(fmaxf(a.u[r], 0.f), 0.99999994f);
  const u64 target = part_of(total, u, false);
  if (before <= target && target < before + mine) {
    u64 sum = before;
    tie = ties_before;
    for (int i = first; i < last; ++i) {
      const u64 w = kept(key_at(i), tie);
      sum += w;
      if (sum > target) {
        a.tokens[r] = i;
        if (a.logprobs) {
          const double x = (double)logit_of(key_at(i));
          a.logprobs[r] = (float)((x == weigh.max ? 0.0 : (x - weigh.max) * weigh.inv) - log((double)total / kOne));
        }
        break;
      }
    }
  }
}

}  // namespace

extern "C" {

int htr_sample_last_cuda_error(void) { return t_last_cuda; }

int htr_sample(const void* logits, int dtype, int64_t row_stride, int rows, int vocab, const float* u, const float* temperature, const int* top_k,
               const float* top_p, const float* min_p, int64_t* tokens, float* logprobs, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16 && dtype != HTR_DTYPE_F32) return HTR_ERR_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || row_stride < vocab) return HTR_ERR_BAD_SHAPE;
  if (vocab > 1 << 20) return HTR_ERR_TOO_LARGE;
  if (rows == 0) return HTR_OK;
  if (!logits || !u || !tokens) return HTR_ERR_NULL;
  const SampleArgs a = {logits, row_stride, dtype, rows, vocab, u, temperature, top_k, top_p, min_p, reinterpret_cast<long long*>(tokens), logprobs};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int e = (int)cudaLaunchKernelEx(&cfg, sample_kernel, a);
  if (e) {
    t_last_cuda = e;
    (void)cudaGetLastError();
    return HTR_ERR_CUDA;
  }
  return HTR_OK;
}

}  // extern "C"
