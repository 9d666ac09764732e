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
  int rows, vocab;
  const float *u, *temperature;
  const int* top_k;
  const float *top_p, *min_p;
  long long* tokens;
  float* logprobs;
};

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8, kBins = 2048;
constexpr double kOne = 4398046511104.0;                   // 2^42: sums of up to 2^20 weights fit in 62 bits
using u64 = unsigned long long;
constexpr u64 kMark = 1ull << 63;                          // on the one message of a cluster that counts

// unsigned order of floats; NaN and -infinity are 0, below everything that can be chosen
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  if (!(x > -__builtin_huge_valf())) return 0;
  return b == 0x80000000u ? 0x80000000u : b & 0x80000000u ? ~b : b | 0x80000000u;     // (-0 is 0)
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

template <int DT>
struct Logit {
  static constexpr int kBytes = DT == HTR_DTYPE_F32 ? 4 : 2;
  // keys of two different logits are at least 2^kGap apart
  static constexpr int kGap = DT == HTR_DTYPE_F32 ? 0 : DT == HTR_DTYPE_BF16 ? 16 : 13;
  static __device__ __forceinline__ float wide(uint16_t raw) {
    return DT == HTR_DTYPE_BF16 ? __uint_as_float((uint32_t)raw << 16) : __half2float(*reinterpret_cast<const __half*>(&raw));
  }
  static __device__ __forceinline__ uint32_t key(const char* row, int i) {
    if (DT == HTR_DTYPE_F32) return key_of(reinterpret_cast<const float*>(row)[i]);
    return key_of(wide(reinterpret_cast<const uint16_t*>(row)[i]));
  }
};

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

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(htr::kFullWarp, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(htr::kFullWarp, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

struct Shared {
  unsigned count[kBins], lo[kBins], hi[kBins];             // of a range of keys: tokens, and their weight in two words
  u64 red[2][kWarps];
  u64 mail[2][4];                                          // what the thread blocks of a cluster tell one another, in turns
};

template <typename V>
__device__ __forceinline__ V remote(const V* mine, unsigned rank) {
  uint32_t at;
  V v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  if constexpr (sizeof(V) == 8) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  else asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// A cluster of thread blocks per row, each with a contiguous slice of it, which it reads from memory once, into shared memory (rows too
// long for that are read again from L2).
// What bounds it: the passes over a slice (an exponential in double for every token that a sum needs) and the exchanges between thread
// blocks, about 1 us each, not the bytes.  So:
//  * a border is found by histograms over ranges of keys (the bits of the logits in their order): 2048 bins, first over the tokens
//    within 12 nats of the largest, where borders usually lie, then inside the bin that holds the border until it holds one value:
//    one or two passes for 16-bit logits, two or three for float32, and exponentials only for the tokens inside the range;
//  * thread blocks meet in shared memory of the cluster: sums of bins are split among them, and each tells only a total.
template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a, int per, int staged) {
  using L = Logit<DT>;
  extern __shared__ __align__(16) char stage[];
  __shared__ Shared s;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned rank, size;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int r = blockIdx.x / size, begin = min((int)rank * per, a.vocab), n = min(begin + per, a.vocab) - begin;
  const char* src = static_cast<const char*>(a.logits) + ((size_t)r * a.row_stride + begin) * L::kBytes;
  int turn = 0;                                            // of s.mail: a message is written over two exchanges later, when all have read it
  const auto barrier = [&] {
    if (size > 1) htr::cluster_sync();
    else __syncthreads();
  };
  // ---- the largest, and the first index that has it
  u64 top = 0;
  const auto look = [&](uint32_t key, int i) {
    const u64 v = (u64)key << 32 | (0xFFFFFFFFu - (unsigned)(begin + i));
    top = v > top ? v : top;
  };
  constexpr int kVec = 16 / L::kBytes;
  const int whole = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? n / kVec : 0;
#pragma unroll 4
  for (int x = tid; x < whole; x += kThreads) {
    const uint4 raw = reinterpret_cast<const uint4*>(src)[x];
    if (staged) reinterpret_cast<uint4*>(stage)[x] = raw;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == HTR_DTYPE_F32) {
        look(key_of(__uint_as_float(w[j])), 4 * x + j);
      } else {
        look(key_of(L::wide((uint16_t)w[j])), 8 * x + 2 * j);
        look(key_of(L::wide((uint16_t)(w[j] >> 16))), 8 * x + 2 * j + 1);
      }
    }
  }
#pragma unroll 4
  for (int i = whole * kVec + tid; i < n; i += kThreads) {
    if constexpr (DT == HTR_DTYPE_F32) {
      const float f = reinterpret_cast<const float*>(src)[i];
      if (staged) reinterpret_cast<float*>(stage)[i] = f;
      look(key_of(f), i);
    } else {
      const uint16_t raw = reinterpret_cast<const uint16_t*>(src)[i];
      if (staged) reinterpret_cast<uint16_t*>(stage)[i] = raw;
      look(key_of(L::wide(raw)), i);
    }
  }
  if (staged) src = stage;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 v = __shfl_xor_sync(htr::kFullWarp, top, o);
    top = v > top ? v : top;
  }
  if (lane == 0) s.red[0][warp] = top;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) top = s.red[0][w] > top ? s.red[0][w] : top;
  if (tid == 0) s.mail[turn][0] = top;
  barrier();
  for (unsigned c = 0; c < size; ++c) {
    const u64 v = remote(&s.mail[turn][0], c);
    top = v > top ? v : top;
  }
  turn ^= 1;
  const uint32_t top_key = (uint32_t)(top >> 32);
  const float t = a.temperature ? a.temperature[r] : 1.f;
  if (top_key == 0 || !(t > 0.f)) {                        // nothing to choose from; greedy
    if (tid == 0 && rank == 0) {
      a.tokens[r] = top_key == 0 ? -1 : (long long)(0xFFFFFFFFu - (uint32_t)top);
      if (a.logprobs) a.logprobs[r] = top_key == 0 ? __int_as_float(0x7FC00000) : 0.f;
    }
    barrier();                                             // no thread block leaves while another reads its memory
    return;
  }
  const Weigh weigh = {(double)logit_of(top_key), 1.0 / (double)t};
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, least = a.min_p ? a.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  const double bound = least > 0.f ? (double)fminf(least, 1.f) * kOne : 0.0;
  // ---- the border: keys above `high` are kept, and of those in [low, high], which are all equal, the first `ties`
  uint32_t low = 0, high = 0;
  unsigned ties = 0xFFFFFFFFu;
  // sums of the cluster, of two values of every thread
  const auto sum_all = [&](u64& x, u64& y) {
    x = warp_sum(x);
    y = warp_sum(y);
    if (lane == 0) {
      s.red[0][warp] = x;
      s.red[1][warp] = y;
    }
    __syncthreads();
    if (warp == 0) {
      x = warp_sum(s.red[0][lane]);
      y = warp_sum(s.red[1][lane]);
      if (lane == 0) {
        s.mail[turn][0] = x;
        s.mail[turn][1] = y;
      }
    }
    barrier();
    x = y = 0;
    for (unsigned c = 0; c < size; ++c) {
      x += remote(&s.mail[turn][0], c);
      y += remote(&s.mail[turn][1], c);
    }
    turn ^= 1;
  };
  // the border at which the tokens, or their weight, reach `target`
  const auto find = [&](bool counts, u64 target) {
    u64 above = 0;
    uint32_t hi = top_key, lo = max(key_of((float)(weigh.max - 12.0 * (double)t)), low);
    if (isinf(weigh.max) || lo > hi) lo = hi;
    for (;;) {
      int shift = 32 - __clz(hi - lo) - 11;                // at most kBins bins
      if (shift < 0) shift = 0;
      if (hi - lo >> shift >= kBins) ++shift;
      for (int b = tid; b < kBins; b += kThreads) s.count[b] = s.lo[b] = s.hi[b] = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t key = L::key(src, i);
        if (key < lo || key > hi) continue;
        const int b = (hi - key) >> shift;
        atomicAdd(&s.count[b], 1u);
        if (!counts) {
          const u64 w = weigh(key);
          const unsigned x = (unsigned)w, was = atomicAdd(&s.lo[b], x), y = (unsigned)(w >> 32) + (was + x < x);
          if (y) atomicAdd(&s.hi[b], y);
        }
      }
      barrier();
      // this thread block's share of the bins, over the cluster
      const int share = kBins / size, b = rank * share + tid;
      u64 value = 0, tokens = 0;
      if (tid < share)
        for (unsigned c = 0; c < size; ++c) {
          const unsigned m = remote(&s.count[b], c);
          tokens += m;
          value += counts ? m : (u64)remote(&s.hi[b], c) << 32;
          if (!counts) value += remote(&s.lo[b], c);
        }
      // (with one thread block a thread takes two bins)
      u64 value2 = 0, tokens2 = 0;
      if (share > kThreads) {
        const int b0 = 2 * tid;
        tokens = s.count[b0];
        value = counts ? tokens : ((u64)s.hi[b0] << 32) + s.lo[b0];
        tokens2 = s.count[b0 + 1];
        value2 = counts ? tokens2 : ((u64)s.hi[b0 + 1] << 32) + s.lo[b0 + 1];
      }
      u64 end = warp_scan(value + value2, lane);
      if (lane == 31) s.red[0][warp] = end;
      __syncthreads();
      u64 before = 0, total = 0;
      {
        const u64 v = s.red[0][lane], e = warp_scan(v, lane);
        before = __shfl_sync(htr::kFullWarp, e - v, warp);
        total = __shfl_sync(htr::kFullWarp, e, 31);
      }
      if (tid == 0) s.mail[turn][0] = total;
      barrier();
      u64 all = above;
      for (unsigned c = 0; c < size; ++c) {
        const u64 v = remote(&s.mail[turn][0], c);
        if (c < rank) before += v;
        all += v;
      }
      turn ^= 1;
      if (all < target) {                                  // the border lies below this range
        above = all;
        if (lo <= low || lo == 0) {                        // (a target that rounding puts beyond everything: all are kept)
          return;
        }
        hi = lo - 1;
        lo = low;
        continue;
      }
      before += above + end - value - value2;
      if (before < target && before + value + value2 >= target) {
        const bool second = before + value < target;
        const int at = share > kThreads ? 2 * tid + second : b;
        const u64 from = second ? before + value : before;
        s.mail[turn][0] = at;
        s.mail[turn][1] = from;
        s.mail[turn][2] = second ? value2 : value;
        s.mail[turn][3] = (second ? tokens2 : tokens) | kMark;
      }
      barrier();
      u64 bin = 0, from = 0, mass = 0, in = 0;
      for (unsigned c = 0; c < size; ++c) {
        const u64 m = remote(&s.mail[turn][3], c);
        if (m & kMark) {
          in = m & ~kMark;
          bin = remote(&s.mail[turn][0], c);
          from = remote(&s.mail[turn][1], c);
          mass = remote(&s.mail[turn][2], c);
        }
      }
      barrier();
      if (tid == 0) s.mail[turn][3] = 0;
      const uint32_t new_hi = hi - ((uint32_t)bin << shift), step = (1u << shift) - 1, new_lo = new_hi - lo > step ? new_hi - step : lo;
      if (shift <= L::kGap || in == 1) {                   // one value
        const u64 each = counts ? 1 : mass / in;
        const u64 need = each ? (target - from + each - 1) / each : in;
        low = new_lo;
        high = new_hi;
        ties = (unsigned)min(max(need, (u64)1), (u64)0xFFFFFFFFu);
        return;
      }
      above = from;
      hi = new_hi;
      lo = new_lo;
    }
  };
  if (tid == 0) s.mail[0][3] = s.mail[1][3] = 0;
  __syncthreads();
  if (by_k) find(true, (u64)k);
  if (by_p) {
    u64 all = 0, tied = 0, each = 0;
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t key = L::key(src, i);
      if (key > high) {
        all += weigh(key);
      } else if (key >= low && key) {
        ++tied;
        each = weigh(key);
      }
    }
    u64 none = 0;
    if (by_k) {                                            // every tie weighs the same
      each *= tied;
      sum_all(each, tied);
      if (tied) each = each / tied * min(tied, (u64)ties);
    }
    sum_all(all, none);
    find(false, max(part_of(all + each, p, true), (u64)1));
  }
  // ---- the token: a warp takes consecutive tokens
  const int seg = (n + kWarps - 1) / kWarps, first = min(warp * seg, n), last = min(first + seg, n);
  const auto kept = [&](uint32_t key, bool& tie) -> u64 {   // the weight of a token that is kept, or may be: a tie
    tie = false;
    if (key == 0 || key < low) return 0;
    const u64 w = weigh(key);
    if ((double)w < bound) return 0;
    tie = key <= high;
    return w;
  };
  u64 mine = 0, tied = 0, each = 0;
  for (int i = first + lane; i < last; i += 32) {
    bool tie;
    const u64 w = kept(L::key(src, i), tie);
    if (tie) {
      ++tied;
      each = w;
    } else {
      mine += w;
    }
  }
  mine = warp_sum(mine);
  tied = warp_sum(tied);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 v = __shfl_xor_sync(htr::kFullWarp, each, o);
    each = v > each ? v : each;
  }
  // ties before this warp: over the thread block, then over the cluster
  __syncthreads();
  if (lane == 0) s.red[0][warp] = tied;
  __syncthreads();
  u64 tied_before = 0, tied_block = 0;
  {
    const u64 v = s.red[0][lane], e = warp_scan(v, lane);
    tied_before = __shfl_sync(htr::kFullWarp, e - v, warp);
    tied_block = __shfl_sync(htr::kFullWarp, e, 31);
  }
  if (tid == 0) s.mail[turn][0] = tied_block;
  barrier();
  for (unsigned c = 0; c < rank; ++c) tied_before += remote(&s.mail[turn][0], c);
  turn ^= 1;
  const u64 room = ties > tied_before ? ties - tied_before : 0;
  mine += each * min(tied, room);
  __syncthreads();
  if (lane == 0) s.red[0][warp] = mine;
  __syncthreads();
  u64 before = 0, total = 0;
  {
    const u64 v = s.red[0][lane], e = warp_scan(v, lane);
    before = __shfl_sync(htr::kFullWarp, e - v, warp);
    total = __shfl_sync(htr::kFullWarp, e, 31);
  }
  if (tid == 0) s.mail[turn][0] = total;
  barrier();
  total = 0;
  for (unsigned c = 0; c < size; ++c) {
    const u64 v = remote(&s.mail[turn][0], c);
    if (c < rank) before += v;
    total += v;
  }
  barrier();                                               // nothing remote is read any more
  const float u = fminf(fmaxf(a.u[r], 0.f), 0.99999994f);
  const u64 target = part_of(total, u, false);
  if (before > target || target >= before + mine) return;
  // this warp holds the token
  u64 tied_here = 0;
  for (int base = first; base < last; base += 32) {
    bool tie = false;
    const int i = base + lane;
    const uint32_t key = i < last ? L::key(src, i) : 0;
    u64 w = kept(key, tie);
    const unsigned mark = __ballot_sync(htr::kFullWarp, tie);
    if (tie && tied_here + __popc(mark & ((1u << lane) - 1)) >= room) w = 0;
    tied_here += __popc(mark);
    const u64 end = before + warp_scan(w, lane);
    const unsigned hit = __ballot_sync(htr::kFullWarp, end > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.tokens[r] = begin + i;
        if (a.logprobs) {
          const double x = (double)logit_of(key);
          a.logprobs[r] = (float)((x == weigh.max ? 0.0 : (x - weigh.max) * weigh.inv) - log((double)total / kOne));
        }
      }
      return;
    }
    before = __shfl_sync(htr::kFullWarp, end, 31);
  }
}

template <int DT>
int run(const SampleArgs& a, cudaStream_t st) {
  constexpr int kStage = 160 * 1024;
  // thread blocks per row: as many as the GPU has room for at one per SM; a row in fewer is one with fewer exchanges
  int size = 1;
  while (size < kMaxCluster && (long long)a.rows * size * 2 <= 148 && a.vocab > size * 2048) size *= 2;
  while (size < kMaxCluster && (long long)a.vocab * Logit<DT>::kBytes > (long long)size * kStage) size *= 2;
  const int per = ((a.vocab + size - 1) / size + 15) / 16 * 16;
  const bool staged = (long long)per * Logit<DT>::kBytes <= kStage;
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (!e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStage);
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows * size);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = staged ? (size_t)per * Logit<DT>::kBytes : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (!e) e = (int)cudaLaunchKernelEx(&cfg, sample_kernel<DT>, a, per, (int)staged);
  if (e) {
    t_last_cuda = e;
    (void)cudaGetLastError();
    return HTR_ERR_CUDA;
  }
  return HTR_OK;
}

}  // namespace

extern "C" {

int htr_sample_last_cuda_error(void) { return t_last_cuda; }

int htr_sample(const void* logits, int dtype, int64_t row_stride, int rows, int vocab, const float* u, const float* temperature, const int* top_k,
               const float* top_p, const float* min_p, int64_t* tokens, float* logprobs, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16 && dtype != HTR_DTYPE_F32) return HTR_ERR_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || row_stride < vocab) return HTR_ERR_BAD_SHAPE;
  if (vocab > 1 << 20 || rows > 1 << 24) return HTR_ERR_TOO_LARGE;
  if (rows == 0) return HTR_OK;
  if (!logits || !u || !tokens) return HTR_ERR_NULL;
  const SampleArgs a = {logits, row_stride, rows, vocab, u, temperature, top_k, top_p, min_p, reinterpret_cast<long long*>(tokens), logprobs};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == HTR_DTYPE_BF16 ? run<HTR_DTYPE_BF16>(a, st) : dtype == HTR_DTYPE_F16 ? run<HTR_DTYPE_F16>(a, st) : run<HTR_DTYPE_F32>(a, st);
}

}  // extern "C"
