// Sampling of one token per row of logits from a given uniform number: temperature, top-k, top-p and min-p.
//
// The tokens of a row are ordered by logit, ties by index.  With w = exp((logit - max) / temperature) each filter keeps a beginning of
// that order: top-k the first k; top-p the shortest beginning of those whose weight reaches p times theirs; min-p all with w >= min_p;
// together the shortest of the three, at least one token.  The token is then the first in the order of the vocabulary at which
// the running weight of the kept ones exceeds u times their sum.
//
// Borders decide about whole tokens, so weights are 64-bit integers, 2^42 exp(x) with exp in double: their sums are exact and do not
// depend on who adds them.  Each weight is off by up to 2^-43 of the largest when it is rounded (and 2^-44 before), so that a border lies
// within vocab * 2^-42 of the largest weight of that of real numbers, and what weighs less than 2^-43 of it (29.8 temperatures below) is never chosen: 2^42
// is the most that 2^20 weights and their multiples by 2^24 have room for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

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
constexpr uint32_t kNegative = 0x7FFFFFFFu - 0x3B800000u;   // the key of -2^-8

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
  static constexpr uint32_t kLowest = DT == HTR_DTYPE_F32 ? 0xFF800000u : DT == HTR_DTYPE_BF16 ? 0xFF80u : 0xFC00u;     // -infinity
  // logit j of a vector of 16 bytes
  static __device__ __forceinline__ float at(const uint4& v, int j) {
    const int x = DT == HTR_DTYPE_F32 ? j : j >> 1;
    const uint32_t w = x == 0 ? v.x : x == 1 ? v.y : x == 2 ? v.z : v.w;
    if (DT == HTR_DTYPE_F32) return __uint_as_float(w);
    if (DT == HTR_DTYPE_BF16) return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return j & 1 ? __high2float(h) : __low2float(h);
  }
  // bf16: upper halves of the keys of two logits (of -0: 32767)
  static __device__ __forceinline__ uint32_t two_keys(uint32_t w) { return w ^ ((w >> 15 & 0x00010001u) * 0xFFFFu | 0x80008000u); }
  // the largest of a vector, NaN left aside
  static __device__ __forceinline__ float largest(const uint4& v) {
    if constexpr (DT == HTR_DTYPE_F32) {
      return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else if constexpr (DT == HTR_DTYPE_BF16) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
      const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(f.x, f.y);
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&v);
      const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(f.x, f.y);
    }
  }
  // bf16: which of a vector's logits are at least `from` (bit i: the lower of word i, 16 + i: the upper), and the logit of a bit
  static __device__ __forceinline__ unsigned at_least(const uint4& v, float from) {
    const uint32_t half = __float_as_uint(from) >> 16, pair = half << 16 | half;              // (what is cut off lies between two logits)
    const __nv_bfloat162 f = *reinterpret_cast<const __nv_bfloat162*>(&pair), *w = reinterpret_cast<const __nv_bfloat162*>(&v);
    return (__hge2_mask(w[0], f) & 0x00010001u) | (__hge2_mask(w[1], f) & 0x00020002u) | (__hge2_mask(w[2], f) & 0x00040004u) | (__hge2_mask(w[3], f) & 0x00080008u);
  }
  static __device__ __forceinline__ float of_bit(const uint4& v, int bit) {
    const uint32_t w = bit & 2 ? (bit & 1 ? v.w : v.z) : (bit & 1 ? v.y : v.x);
    return __uint_as_float(bit & 16 ? w & 0xFFFF0000u : w << 16);
  }
  // the key in [low, high], of which there is one: logits of 16 bits end in zeros, keys of negative ones in ones
  static __device__ __forceinline__ uint32_t only(uint32_t low, uint32_t high) {
    const uint32_t rest = (1u << kGap) - 1, positive = high & ~rest;
    return high >= 0x80000000u && positive >= low ? positive : ((min(high, 0x7FFFFFFFu) + 1) & ~rest) - 1;
  }
};

// 2^42 exp((logit - max) / temperature) to the nearest integer, by a table of 2^(j / 64) and a polynomial of the fourth degree between its
// entries (the table-driven exponential of Tang, 1989): off by 2^-44 of the largest weight before it is rounded.  The double exp of the
// math library is right to its last bit and took most of a sample's time.
struct Weigh {
  double max, by;                                          // by = 64 log2(e) / temperature
  bool infinite;
  const double* table;
  uint32_t top_key;
  const u64* known;                                        // bf16: of the 2048 values from the largest on and as many from -2^-8 on; or none
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    if (known) {
      if (top_key - key < (uint32_t)kBins << 16) return known[(top_key - key) >> 16];
      if (kNegative - key < (uint32_t)kBins << 16) return known[kBins + ((kNegative - key) >> 16)];
    }
    return computed(key);
  }
  __device__ __forceinline__ u64 computed(uint32_t key) const {
    if (infinite) return key == top_key ? (u64)kOne : 0;
    constexpr double kShift = 6755399441055744.0;          // 1.5 * 2^52: its low word then holds the rounded sum
    const double d = (double)logit_of(key) - max, z = fma(d, by, kShift);
    const int k = __double2loint(z);
    if (__double2hiint(z) < 0x4337FFFF || k < -45 * 64 || key == 0) return 0;
    const double r = fma(d, by, -(z - kShift)), t = table[k & 63];
    // 2^(r / 64) = 1 + r (c1 + r (c2 + ...)), c_i = (ln 2 / 64)^i / i!
    double p = fma(r, 5.732851688640402e-10, 2.1173137155464774e-07);
    p = fma(r, p, 5.864904955056169e-05);
    p = fma(r, p, 1.0830424696249145e-02);
    const double w = fma(t * r, p, t);                     // [2^(k / 64)] without its whole power
    const double v = __hiloint2double(__double2hiint(w) + ((k >> 6) + 42) * (1 << 20), __double2loint(w));
    return (u64)__double_as_longlong(v + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;     // 2^52 + v: v to the nearest integer
  }
};

// f * w for 0 <= f < 1, exactly: rounded down, or up
__device__ __forceinline__ u64 part_of(u64 w, float f, bool up) {
  if (!(f > 0.f)) return 0;
  int e;
  const u64 bits = (u64)ldexpf(frexpf(f, &e), 24);         // f = bits * 2^(e - 24), e <= 0
  const u64 hi = __umul64hi(w, bits), lo = w * bits;       // below 2^86
  const int down = 24 - e;                                 // at least 24
  if (down < 64) return (hi << (64 - down) | lo >> down) + (up && (lo & (((u64)1 << down) - 1)) != 0);
  const u64 whole = down < 128 ? hi >> (down - 64) : 0;    // (f below 2^-40)
  return whole + (up && (lo != 0 || (down < 128 ? whole << (down - 64) : 0) != hi));
}

__device__ __forceinline__ u64 warp_sum(u64 v) {            // in parts whose sums fit a reduction of 32 bits
  const unsigned a = __reduce_add_sync(htr::kFullWarp, (unsigned)v & 0xFFFFFFu), b = __reduce_add_sync(htr::kFullWarp, (unsigned)(v >> 24) & 0xFFFFFFu),
                 c = __reduce_add_sync(htr::kFullWarp, (unsigned)(v >> 48));
  return a + ((u64)b << 24) + ((u64)c << 48);
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(htr::kFullWarp, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <int DT>
struct Shared {
  u64 known[DT == HTR_DTYPE_BF16 ? 2 * kBins + 2 : 2];
  unsigned count[2 * kBins], lo[kBins];                    // of a range of keys: tokens, and their weight in two words (the upper from kBins on)
  u64 red[2][kWarps], ahead[2][kWarps];                    // of the warps: what each has, and what those before it have
  double table[64];
  u64 mail[2][2][kMaxCluster];                             // what the thread blocks of a cluster tell one another, in turns
  u64 border[4];                                           // what the one that holds a border tells all
  u64 told[4];                                             // what its first warp tells a thread block
  u64 won[4];                                              // what lies before the warp that holds the token, the ties left there, and its part
};

template <typename V>
__device__ __forceinline__ V remote(const V* mine, unsigned rank) {
  uint32_t at;
  V v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  if constexpr (sizeof(V) == 8) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  else asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ void remote_store(const u64* mine, unsigned rank, u64 v) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

// A cluster of thread blocks per row, each with a contiguous slice of it, which it reads from memory once, into shared memory (rows too
// long for that are read again from L2).
// What bounds it: instructions of the passes over a slice, and the exchanges between thread blocks (about 1 us each), not the bytes.  So:
//  * a border is found by histograms over ranges of keys (the bits of the logits in their order), 2048 bins at a time, then inside the bin that
//    holds the border until a bin is one value.  Counts alone are enough where bins are single values from the start (16-bit logits:
//    the upper 16 binades of bf16 and as many negative ones): a bin weighs its count times one exponential.  Other tokens need an
//    exponential each, float32 ones above all, whose first range is the 12 nats below the largest, where borders usually lie;
//  * eight logits are compared with the lower end of a range at once: most passes meet few that matter;
//  * thread blocks meet in shared memory of the cluster: bins are split among them, each tells only totals, and the first warp of each
//    does the arithmetic of an exchange for all (64-bit scans in all 32 warps had been most of a small row's instructions).
template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a, int per, int staged) {
  using L = Logit<DT>;
  constexpr int kVec = 16 / L::kBytes;
  extern __shared__ __align__(16) char smem[];
  Shared<DT>& s = *reinterpret_cast<Shared<DT>*>(smem);
  char* stage = smem + sizeof(Shared<DT>);
  static_assert(sizeof(Shared<DT>) % 16 == 0, "the row's slice behind it is read in vectors");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned rank, size;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int r = blockIdx.x / size, begin = min((int)rank * per, a.vocab), n = min(begin + per, a.vocab) - begin, vectors = (n + kVec - 1) / kVec;
  const char* src = static_cast<const char*>(a.logits) + ((size_t)r * a.row_stride + begin) * L::kBytes;
  const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  const float t = a.temperature ? a.temperature[r] : 1.f, p = a.top_p ? a.top_p[r] : 1.f, least = a.min_p ? a.min_p[r] : 0.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float u = fminf(fmaxf(a.u[r], 0.f), 0.99999994f);
  const auto barrier = [&] {
    if (size > 1) htr::cluster_sync();
    else __syncthreads();
  };
  if (size > 1) htr::cluster_arrive();                     // (waited for before anything is written to another thread block)
  // by the first warp, all lanes of which have v: to every thread block of the cluster
  int turn = 0;                                            // of s.mail: a message is written over two exchanges later, when all have read it
  const auto tell = [&](int what, u64 v) {
    if (lane < size) remote_store(&s.mail[turn][what][rank], lane, v);
  };
  // kVec logits; -infinity behind the last
  const auto from_memory = [&](int x) {
    if (aligned && (x + 1) * kVec <= n) return reinterpret_cast<const uint4*>(src)[x];
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == HTR_DTYPE_F32) {
        const int i = 4 * x + j;
        w[j] = i < n ? reinterpret_cast<const uint32_t*>(src)[i] : L::kLowest;
      } else {
        const int i = 8 * x + 2 * j;
        const uint16_t* at = reinterpret_cast<const uint16_t*>(src) + i;
        w[j] = (i < n ? at[0] : L::kLowest) | (uint32_t)(i + 1 < n ? at[1] : L::kLowest) << 16;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  const auto fetch = [&](int x) { return staged ? reinterpret_cast<const uint4*>(stage)[x] : from_memory(x); };
  // ---- the largest
  float most = -__builtin_huge_valf();
#pragma unroll 2
  for (int x = tid; x < vectors; x += kThreads) {
    const uint4 w = from_memory(x);
    if (staged) reinterpret_cast<uint4*>(stage)[x] = w;
    most = fmaxf(most, L::largest(w));
  }
  if (tid < 64) s.table[tid] = exp2(tid / 64.0);
  if (tid == 64) s.won[2] = 0;
  if (size > 1) htr::cluster_wait();
  // of all threads of the cluster: the largest of a 32-bit value
  const auto largest_of = [&](uint32_t v) {
    v = __reduce_max_sync(htr::kFullWarp, v);
    if (lane == 0) s.red[0][warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = __reduce_max_sync(htr::kFullWarp, (uint32_t)s.red[0][lane]);
      tell(0, v);
    }
    barrier();
    v = __reduce_max_sync(htr::kFullWarp, lane < size ? (uint32_t)s.mail[turn][0][lane] : 0u);
    turn ^= 1;
    return v;
  };
  const uint32_t top_key = largest_of(key_of(most));
  if (top_key == 0 || !(t > 0.f)) {                        // nothing to choose from; greedy: the first index that has it
    uint32_t at = 0xFFFFFFFFu;
    for (int x = tid; x < vectors && top_key; x += kThreads) {
      const uint4 w = fetch(x);
      if (key_of(L::largest(w)) != top_key) continue;
#pragma unroll
      for (int j = kVec - 1; j >= 0; --j)
        if (key_of(L::at(w, j)) == top_key) at = min(at, (uint32_t)(begin + x * kVec + j));
    }
    at = ~largest_of(~at);
    if (tid == 0 && rank == 0) {
      a.tokens[r] = top_key == 0 ? -1 : (long long)at;
      if (a.logprobs) a.logprobs[r] = top_key == 0 ? __int_as_float(0x7FC00000) : 0.f;
    }
    return;
  }
  Weigh weigh = {(double)logit_of(top_key), 64 * 1.4426950408889634 / (double)t, isinf(logit_of(top_key)) != 0, s.table, top_key, nullptr};
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  const u64 bound = least > 0.f ? (u64)ceil((double)fminf(least, 1.f) * kOne) : 0;
  if constexpr (DT == HTR_DTYPE_BF16) {
    if (!by_k) {                                           // all tokens will be weighed: their values are fewer
      for (int b = tid; b < 2 * kBins; b += kThreads) {
        const uint32_t from = b < kBins ? top_key : kNegative, step = (uint32_t)(b & (kBins - 1)) << 16;
        s.known[b] = from > step ? weigh.computed(from - step) : 0;
      }
      if (tid == 0) s.known[2 * kBins] = 0;
      weigh.known = s.known;
      __syncthreads();
    }
  }
  // bf16 whose values have a place in s.known by a subtraction (zero lies below the first 2048, and nothing is infinite): without a branch per logit
  const bool quick = weigh.known && !weigh.infinite && (top_key >> 16) - 0x8000u >= (uint32_t)kBins;
  const uint32_t top_half = top_key >> 16, real = top_half - 0x7Fu;       // (0x7F: of -infinity)
  const auto place_of = [&](uint32_t half, bool& odd) {    // 2 * kBins: none; odd: and it is neither NaN nor -infinity
    const uint32_t d = top_half - half, e = (kNegative >> 16) - half, at = d < (uint32_t)kBins ? d : (uint32_t)kBins + min(e, (uint32_t)kBins);
    odd = d < real && at == 2u * kBins;
    return at;
  };
  const auto half_of = [&](const uint4& w, int j) {
    const uint32_t y = L::two_keys(j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w);
    return j & 1 ? y >> 16 : y & 0xFFFFu;
  };
  // ---- the border: keys above `high` are kept, and of the `tied` tokens in [low, high], which are all equal, the first `ties`
  uint32_t low = 0, high = 0;
  unsigned ties = 0xFFFFFFFFu, tied = 0;
  // finds the border at which the tokens reach `count`, or their weight `part` of that of all that have been kept so far
  const auto find = [&](bool counts, u64 count, float part) {
    u64 above = 0, target = count;
    uint32_t hi = top_key, lo = 0;
    for (bool first = true;; first = false) {
      if (first) {                                         // 16-bit logits: as many values as there are bins
        // (what is counted is few, and lies within two binades as a rule: the more values, the more tokens to count)
        const uint32_t values = counts && L::kGap == 16 ? 255 : kBins - 1;
        lo = L::kGap ? (hi > values << L::kGap ? hi - (values << L::kGap) : 0)
                     : key_of((float)(weigh.max - 12.0 * (double)t));
        lo = max(weigh.infinite ? hi : lo, low);
      }
      const int shift = max(21 - __clz(hi - lo), 0);       // at most kBins bins
      const bool single = L::kGap && shift <= L::kGap;     // bins are single values
      const bool sums = first && !counts;                  // the weight of all is needed
      const bool below = sums && single && L::kGap == 16;           // the negative values from -2^-8 to -2^8 have bins too, behind the others
      for (int b = tid; b < kBins; b += kThreads) {
        s.count[b] = s.count[kBins + b] = 0;
        if (!single) s.lo[b] = 0;
      }
      __syncthreads();
      u64 rest = 0;                                        // the weight of tokens without a bin
      const uint32_t from_key = sums ? low : lo;
      const float from = from_key < 0x00800000u ? -3.402823466e38f : logit_of(from_key);
      for (int x = tid; x < vectors; x += kThreads) {
        const uint4 w = fetch(x);
        if (!(L::largest(w) >= from)) continue;
        if (below && quick) {
          unsigned odd = 0;                                // logits without a place
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            bool is;
            const uint32_t at = place_of(half_of(w, j), is);
            if (at < 2u * kBins) atomicAdd(&s.count[at], 1u);
            if (is) odd |= 1u << j;
          }
          for (; odd; odd &= odd - 1) rest += weigh.computed(key_of(L::at(w, __ffs(odd) - 1)));
          continue;
        }
        const auto take = [&](uint32_t key) {
          if (key > hi || key < from_key || key == 0) return;
          if (key >= lo) {
            const int b = (hi - key) >> shift;
            atomicAdd(&s.count[b], 1u);
            if (counts || single) return;
            const u64 v = weigh(key);
            const unsigned y = (unsigned)v, was = atomicAdd(&s.lo[b], y), z = (unsigned)(v >> 32) + (was + y < y);
            if (z) atomicAdd(&s.count[kBins + b], z);
          } else if (below && kNegative - key < (uint32_t)kBins << 16) {
            atomicAdd(&s.count[kBins + ((kNegative - key) >> 16)], 1u);
          } else {
            rest += weigh(key);
          }
        };
        if constexpr (L::kGap == 16) {                     // few, as a rule
          for (unsigned some = L::at_least(w, from); some; some &= some - 1) take(key_of(L::of_bit(w, __ffs(some) - 1)));
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) take(key_of(L::at(w, j)));
        }
      }
      barrier();
      // this thread block's share of the bins, over the cluster: one or two for each of its first threads
      const int share = kBins / size, each = share > kThreads ? 2 : 1, b0 = rank * share + each * tid;
      u64 value[2] = {0, 0}, end = 0;
      unsigned tokens[2] = {0, 0};
      if (warp * 32 * each < share) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j >= each) continue;
          const int b = b0 + j;
          unsigned more = 0;
          u64 mass = 0;
          // (as many as may be at once: a load under a condition waits for the one before)
          const auto gathered = [&](const unsigned* of, unsigned (&got)[kMaxCluster]) {
            const auto some = [&](auto from, auto to) {
#pragma unroll
              for (unsigned c = decltype(from)::value; c < decltype(to)::value; ++c) got[c] = remote(of, c < size ? c : rank);
            };
            some(std::integral_constant<unsigned, 0>{}, std::integral_constant<unsigned, 2>{});
            if (size > 2) some(std::integral_constant<unsigned, 2>{}, std::integral_constant<unsigned, kMaxCluster>{});
#pragma unroll
            for (unsigned c = 0; c < kMaxCluster; ++c) got[c] = c < size ? got[c] : 0;
          };
          unsigned got[kMaxCluster], low_word[kMaxCluster];
          gathered(&s.count[b], got);
#pragma unroll
          for (int c = 0; c < kMaxCluster; ++c) tokens[j] += got[c];
          if (below || !(counts || single)) gathered(&s.count[kBins + b], got);
          if (below) {
#pragma unroll
            for (int c = 0; c < kMaxCluster; ++c) more += got[c];
          } else if (!(counts || single)) {
            gathered(&s.lo[b], low_word);
#pragma unroll
            for (int c = 0; c < kMaxCluster; ++c) mass += ((u64)got[c] << 32) + low_word[c];
          }
          if (single && !counts) {
            const uint32_t top_of = hi - ((uint32_t)b << shift);
            if (tokens[j]) mass = tokens[j] * weigh(L::only(top_of - min((1u << shift) - 1, top_of), top_of));
            if (more) rest += more * weigh(kNegative - ((uint32_t)b << 16));
          }
          value[j] = counts ? tokens[j] : mass;
        }
        end = warp_scan(value[0] + value[1], lane);
      }
      if (lane == 31) s.red[0][warp] = end;
      if (sums) {
        rest = warp_sum(rest);
        if (lane == 0) s.red[1][warp] = rest;
      }
      __syncthreads();
      if (warp == 0) {
        const u64 v = s.red[0][lane], e = warp_scan(v, lane);
        s.ahead[0][lane] = e - v;
        rest = sums ? warp_sum(s.red[1][lane]) : 0;
        tell(0, __shfl_sync(htr::kFullWarp, e, 31));
        if (sums) tell(1, rest);
      }
      barrier();
      if (warp == 0) {
        const u64 v = lane < size ? s.mail[turn][0][lane] : 0, before = warp_sum(lane < rank ? v : 0), all = warp_sum(v);
        rest = sums ? warp_sum(lane < size ? s.mail[turn][1][lane] : 0) : 0;
        if (lane == 0) {
          s.told[0] = above + before;
          s.told[1] = above + all;
          s.told[2] = above + all + rest;
        }
      }
      turn ^= 1;
      __syncthreads();
      const u64 all = s.told[1];
      if (sums) {
        u64 kept = s.told[2];
        if (tied > ties) kept -= (u64)(tied - ties) * weigh(L::only(low, high));
        target = max(part_of(kept, part, true), (u64)1);
      }
      if (all < target) {                                  // the border lies below this range
        above = all;
        if (lo <= low) return;                             // (nothing is left: all that was kept is)
        hi = lo - 1;
        lo = low;
        continue;
      }
      const u64 before = s.told[0] + s.ahead[0][warp] + end - value[0] - value[1];
      if (before < target && before + value[0] + value[1] >= target) {
        const bool second = before + value[0] < target;
        const u64 message[3] = {(u64)(b0 + second), before + (second ? value[0] : 0), second ? tokens[1] : tokens[0]};
        for (unsigned c = 0; c < size; ++c)
#pragma unroll
          for (int j = 0; j < 3; ++j) remote_store(&s.border[j], c, message[j]);
      }
      barrier();
      const uint32_t in = (uint32_t)s.border[2];
      const u64 so_far = s.border[1];
      hi -= (uint32_t)s.border[0] << shift;
      if (hi - lo >> shift) lo = hi - ((1u << shift) - 1);
      if (shift <= L::kGap) {                              // one value
        const u64 one = counts ? 1 : weigh(L::only(lo, hi)), need = one ? (target - so_far + one - 1) / one : in;
        low = lo;
        high = hi;
        tied = in;
        ties = (unsigned)min(max(need, (u64)1), (u64)in);
        return;
      }
      above = so_far;
    }
  };
  if (by_k) find(true, (u64)k, 0.f);
  if (by_p) find(false, 0, p);
  // ---- the token: a warp takes consecutive tokens, a lane kVec at a time
  const float from = low < 0x00800000u ? -3.402823466e38f : logit_of(low);
  const int seg = ((vectors + kWarps - 1) / kWarps + 31) / 32 * 32, first = min(warp * seg, vectors), last = min(first + seg, vectors);
  u64 each = 0;                                            // the weight of a tie
  if (tied) {
    each = weigh(L::only(low, high));
    if (each < bound) each = 0;
  }
  // from here on what is not kept weighs nothing, and ties are counted
  const uint32_t tie = tied ? L::only(low, high) >> 16 : 0;
  if (quick && (tied || bound)) {
    __syncthreads();
    for (int b = tid; b < 2 * kBins; b += kThreads) {
      const uint32_t half = (b < kBins ? top_half : kNegative >> 16) - (b & (kBins - 1));
      if (half <= tie || s.known[b] < bound) s.known[b] = 0;
    }
    __syncthreads();
  }
  // of a lane's vector: the weight of what lies above the border, and how many ties there are
  const auto weight_of = [&](const uint4& w, unsigned& here) {
    u64 sum = 0;
    here = 0;
    if (!(L::largest(w) >= from)) return sum;
    if (quick) {
      unsigned odd = 0;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        bool is;
        sum += s.known[place_of(half_of(w, j), is)];
        if (is) odd |= 1u << j;
      }
      if (tied) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) here += half_of(w, j) == tie && !(odd >> j & 1);
      }
      for (; odd; odd &= odd - 1) {
        const uint32_t key = key_of(L::at(w, __ffs(odd) - 1));
        if (key < low) continue;
        if (key <= high) {
          ++here;
          continue;
        }
        const u64 v = weigh.computed(key);
        if (v >= bound) sum += v;
      }
      return sum;
    }
    const auto take = [&](uint32_t key) {
      if (key == 0 || key < low) return;
      if (key <= high) {
        ++here;
        return;
      }
      const u64 v = weigh(key);
      if (v >= bound) sum += v;
    };
    if constexpr (L::kGap == 16) {
      for (unsigned some = L::at_least(w, from); some; some &= some - 1) take(key_of(L::of_bit(w, __ffs(some) - 1)));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) take(key_of(L::at(w, j)));
    }
    return sum;
  };
  u64 mine = 0;
  unsigned mine_tied = 0;
  for (int x = first + lane; x < last; x += 32) {
    unsigned here;
    mine += weight_of(fetch(x), here);
    mine_tied += here;
  }
  mine = warp_sum(mine);
  mine_tied = __reduce_add_sync(htr::kFullWarp, mine_tied);
  // sums before this warp: over the thread block, then over the cluster
  if (lane == 0) {
    s.red[0][warp] = mine;
    s.red[1][warp] = mine_tied;
  }
  __syncthreads();
  if (warp == 0) {
    const u64 x = s.red[0][lane], y = s.red[1][lane], ex = warp_scan(x, lane), ey = warp_scan(y, lane);
    s.ahead[0][lane] = ex - x;
    s.ahead[1][lane] = ey - y;
    tell(0, __shfl_sync(htr::kFullWarp, ex, 31));
    tell(1, __shfl_sync(htr::kFullWarp, ey, 31));
  }
  barrier();
  if (warp == 0) {
    const u64 x = lane < size ? s.mail[turn][0][lane] : 0, y = lane < size ? s.mail[turn][1][lane] : 0;
    const u64 bx = warp_sum(lane < rank ? x : 0), by = warp_sum(lane < rank ? y : 0), all = warp_sum(x);
    if (lane == 0) {
      s.told[0] = bx;
      s.told[1] = by;
      s.told[2] = all;
    }
  }
  __syncthreads();
  const u64 ahead = s.told[1] + s.ahead[1][warp], total = s.told[2] + each * min((u64)tied, (u64)ties), target = part_of(total, u, false);
  u64 before = s.told[0] + s.ahead[0][warp] + each * min(ahead, (u64)ties);
  u64 room = ties > ahead ? ties - ahead : 0;              // ties of this warp and of later ones that are kept
  mine += each * min((u64)mine_tied, room);
  // the warp that holds the token: its part, 32 vectors at a time, by all warps (32 times at most: a thread block has 2^17 logits at most)
  if (lane == 0 && before <= target && target < before + mine) {
    s.won[0] = before;
    s.won[1] = room;
    s.won[2] = (u64)first << 32 | (unsigned)last;
  }
  __syncthreads();
  if (s.won[2]) {
    const int x = (int)(s.won[2] >> 32) + tid, end_of = (int)(unsigned)s.won[2];
    unsigned here = 0;
    uint4 w = {};
    u64 sum = 0;
    if (x < end_of) {
      w = fetch(x);
      sum = weight_of(w, here);
    }
    const unsigned passed = (unsigned)warp_scan(here, lane);
    const u64 run_of = warp_scan(sum, lane);               // (without ties)
    if (lane == 31) {
      s.red[0][warp] = run_of;
      s.red[1][warp] = passed;
    }
    __syncthreads();
    const u64 earlier = warp_sum(lane < warp ? s.red[0][lane] : 0), ties_before = warp_sum(lane < warp ? s.red[1][lane] : 0) + passed - here;
    room = s.won[1];
    const u64 mine_room = room > ties_before ? room - ties_before : 0;
    u64 run = s.won[0] + earlier + run_of - sum + each * min(ties_before, room);
    if (run <= target && target < run + sum + each * min((u64)here, mine_room)) {
      u64 tie_at = 0;
#pragma unroll 1
      for (int j = 0; j < kVec && run <= target; ++j) {
        const uint32_t key = key_of(L::at(w, j));
        if (key == 0 || key < low || (key <= high && tie_at++ >= mine_room)) continue;
        const u64 v = key <= high ? each : weigh(key);
        if (v < bound || v == 0) continue;
        run += v;
        if (run <= target) continue;
        a.tokens[r] = begin + x * kVec + j;
        if (a.logprobs) {
          const double d = (double)logit_of(key);
          a.logprobs[r] = (float)((d == weigh.max ? 0.0 : (d - weigh.max) / (double)t) - log((double)total / kOne));
        }
      }
    }
  }
}

template <int DT>
int run(const SampleArgs& a, cudaStream_t st) {
  constexpr int kStage = 160 * 1024;
  // thread blocks per row: as many as the GPU has room for at one per SM; a row in fewer is one with fewer exchanges
  const int sms = htr::current_device_sms();
  int size = 1;
  while (size < kMaxCluster && (long long)a.rows * size * 2 <= sms && a.vocab > size * 2048) size *= 2;
  while (size < kMaxCluster && (long long)a.vocab * Logit<DT>::kBytes > (long long)size * kStage) size *= 2;
  const int per = ((a.vocab + size - 1) / size + 15) / 16 * 16;
  const bool staged = (long long)per * Logit<DT>::kBytes <= kStage;
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (!e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStage + (int)sizeof(Shared<DT>));
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows * size);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared<DT>) + (staged ? (size_t)per * Logit<DT>::kBytes : 0);
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
