// What the kernels of the paged 8-bit cache share: element types, e4m3 conversions, the arguments of the attention, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/htr_b200.h"
#include "htr_common.cuh"

namespace htr {

int paged_fail(int cuda_error);                            // keeps the error for htr_paged_last_cuda_error, HTR_ERR_CUDA
int attention_withhold();                                  // what htr_paged_attention_withhold has set for this thread

template <typename Kern, typename... Args>
int paged_launch(Kern kern, dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const int e = (int)cudaLaunchKernelEx(&cfg, kern, args...);
  if (!e) return HTR_OK;
  (void)cudaGetLastError();                                // a refused launch leaves no error behind for the caller's next check
  return paged_fail(e);
}

template <typename T> struct Half;
template <> struct Half<__nv_bfloat16> {
  static constexpr int kBits = 8;                          // significant
  static __device__ __forceinline__ float2 wide(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
  static __device__ __forceinline__ uint32_t narrow(float x, float y) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <> struct Half<__half> {
  static constexpr int kBits = 11;
  static __device__ __forceinline__ float2 wide(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ uint32_t narrow(float x, float y) {
    const __half2 r = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};

// two floats as e4m3, the first in the low byte (beyond the range: the largest value; NaN stays NaN)
__device__ __forceinline__ uint32_t to_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t from_e4m3(uint32_t two) {   // two e4m3 in the low half -> two fp16
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
constexpr float kScaleLeast = 7.888609052210118e-31f, kScaleMost = 6.646139978924579e35f;          // of codes of 4 bits: 2^-100, 2^119
// a byte's two codes as fp16, each of the four
__device__ __forceinline__ void from_e2m1(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {     // 0xFF where a byte is one of e4m3's NaN
  return __vcmpeq4(v & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
}
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr float kNone = -__builtin_huge_valf();
// The sum of a row's probabilities in units of 2^7: terms of up to 2^15.5 under scales of values of 2^-100 stay finite for 2^19 of them (at 2^12, where they
// begin, for 2^23), and the inverse of the largest scale, 2^119, is a normal number.
constexpr float kSumUnit = 0.0078125f;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.b32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
  return done != 0;
}
// polls of a wait before it gives up: about two seconds of one thread (1 us each) and of a warp whose lanes all poll (4 us); and half a second
// of such a warp for what is still on its way then
constexpr unsigned kSpinLimit = 2000000u, kWarpSpinLimit = 500000u, kDrainLimit = 125000u;
// bounded: false when the limit ran out or another has given up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* fail, unsigned limit = kSpinLimit) {
  if (bar_try(bar, parity)) return true;
  for (unsigned i = 0; i < limit; ++i) {
    if (bar_try(bar, parity)) return true;
    if ((i & 255) == 255 && fail && *fail) return false;
  }
  if (fail) *fail = 1;
  return false;
}
// contiguous bytes (both addresses and the size multiples of 16) to shared memory
__device__ __forceinline__ void bulk_load(uint32_t to, const void* from, int bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

// Parts of a row's results (maximum m, sum l, four dimensions y), joined in their order: part i of `count` is at m_at(i) and so on; kBatch are
// fetched at once, and their factors do not wait for one another.
template <int kBatch, typename M, typename L, typename Y>
__device__ __forceinline__ void join_parts(int count, float& m, float& l, float4& y, M m_at, L l_at, Y y_at) {
  for (int first = 1; first < count; first += kBatch) {
    float pm[kBatch], pl[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      pm[i] = kNone;
      pl[i] = 0.f;
      v[i] = {0.f, 0.f, 0.f, 0.f};
      if (first + i >= count) continue;
      pm[i] = *m_at(first + i);
      pl[i] = *l_at(first + i);
      v[i] = *y_at(first + i);
    }
    float now = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) now = fmaxf(now, pm[i]);
    const float base = now == kNone ? 0.f : now, f = now == kNone ? 1.f : exp2_fast(m - now);
    m = now;
    l *= f;
    y.x *= f; y.y *= f; y.z *= f; y.w *= f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float by = exp2_fast(pm[i] - base);            // (0 where nothing was seen: a NaN there stays one)
      l = fmaf(pl[i], by, l);
      y.x = fmaf(v[i].x, by, y.x); y.y = fmaf(v[i].y, by, y.y); y.z = fmaf(v[i].z, by, y.z); y.w = fmaf(v[i].w, by, y.w);
    }
  }
}

struct AttentionArgs {
  const void* q;
  const int *starts, *seen, *tables;
  long long table_stride;
  int width, requests, tokens, q_heads, kv_heads, group, max_new;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int pages, shift;
  float scale;                                             // of the scores, times log2(e)
  void* out;
  int* status;
  float* parts;                                            // two per thread block: results, maxima, sums of a tile's rows
  int4* cuts;                                              // per thread block, of the tile that begins in its run and goes beyond it
  int withhold;                                            // test hook: the first keys of thread block withhold - 1 never arrive (0: none)
};

// the exponent that brings a row of queries, whose largest magnitude is `most`, to [2^top, 2^(top + 1)): any finite one for 7 <= top <= 14, but for rows
// below 2^(top - 126), which stay that much smaller (so that the power of two and its inverse are normal numbers)
__device__ __forceinline__ int query_exponent(float most, int top) {
  return most > 0.f && most <= 3.402823466e38f ? min(top - ((int)(__float_as_uint(most) >> 23) - 127), 126) : 0;
}

// attention for many rows a request, on the tensor cores (paged_attention_tc.cu)
bool attention_tc_serves(int tokens, int requests, int q_heads, int group, int max_new, long long width, int head_dim);
size_t attention_tc_workspace(int head_dim);
int attention_tc_run(const AttentionArgs& a, int dtype, int head_dim, void* workspace, cudaStream_t st);
bool attention4_tc_serves(int tokens, int requests, int q_heads, int group, int max_new, long long width, int head_dim);     // the same over the cache of 4 bits
int attention4_tc_run(const AttentionArgs& a, int dtype, int head_dim, void* workspace, cudaStream_t st);

}  // namespace htr
