// The paged cache in 4 bits: its writing side (rotary embedding, a Hadamard transform of queries and keys, e2m1 with one scale per token and key/value
// head), its pages as 16- or 32-bit values, and attention over it for few rows a request (many rows: paged_attention_tc.cuh).
//
// Layout of a layer's cache: keys and values [pages][kv_heads][page_size][head_dim / 2], two e2m1 codes in a byte, the even dimension in its low half;
// scales [pages][kv_heads][page_size] bf16, at least 2^-100 and at most 2^119.  The value of an element is its code's (0, 0.5, 1, 1.5, 2, 3, 4, 6) times the scale.
//
// Why the transform: a few channels of the keys of a trained model are many times the others, and the largest element of a token sets the step of all.  With
// q' = H q a and k' = H k / 8 (H the Hadamard matrix in Sylvester's order, a = 8 / head_dim) the product is the same, q' k' = q k, and a channel that
// stands out is spread over all of them: the error of keys whose elements are normal is 11 % of their norm, of such with one channel in 50 eight times as
// large 35 % without the transform and 11 with it.  Values have no such channels as a rule, and stay as they are.
// Why a scale per token: each token is rounded once, and for good.  Why bf16: a code has two significant bits, so that a code times its scale has ten
// and fp16 holds it exactly wherever matrix instructions want it.
#include "paged_attention.cuh"

namespace {

using namespace htr;

// Elements are rotated as 1 / 16 of what they are or less, and transformed as 1 / (16 D): a row of finite ones then stays finite under angles whose magnitude is up to 8 (a pair
// adds up to at most sqrt 2 times its length, which is sqrt 2 times the larger element, and D / 2 pairs to at most D times the largest).
constexpr float kDown = 0.0625f;                           // (besides 1 / D; of many tokens the angles are multiplied: 1 us of the 33 below)

__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// eight floats as e2m1 (to the nearest, ties to the even code, beyond 6: 6), the first in the lowest bits
__device__ __forceinline__ uint32_t to_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ float of_bf16(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// A row's D dimensions, 8 a lane, times the Hadamard matrix; by whole warps.
template <int D>
__device__ __forceinline__ void hadamard(float (&v)[8], int lane) {
#pragma unroll
  for (int h = 1; h < 8; h *= 2)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!(j & h)) {
        const float x = v[j], y = v[j + h];
        v[j] = x + y;
        v[j + h] = x - y;
      }
#pragma unroll
  for (int h = 1; h < D / 8; h *= 2) {
    const float sign = lane & h ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf(sign, v[j], __shfl_xor_sync(kFullWarp, v[j], h));
  }
}

// The same of 16 rows by one warp, as matrix products.  Of H = H_j x H_8 (d = 8 j + b) the H_j are products of 16 rows by 8 or 16 chunks j of 8 dimensions, for each
// b; and the H_8, over b, are sums within a lane.  Lane (g, c) of the products' operand has rows g and g + 8 at kChunks chunks, and of their result too:
// neighbouring ones (kChunks c + i), or every fourth (c + 4 i), whose 16-byte pieces lie side by side over the lanes.
template <int D>
constexpr int kChunks = D / 32;
__device__ __forceinline__ int chunk_of(bool side_by_side, int chunks, int c, int i) { return side_by_side ? c + 4 * i : chunks * c + i; }
// the right operand: (-1)^(bits of j_in & j_out) or, for rows that only move, j_in == j_out; `one`: 1 in the operand's type, two of them
template <int D>
struct Turn {
  uint32_t b[D / 64][D / 64];                              // pair of chunks that come in; 8 rows of chunks that go out
  __device__ __forceinline__ Turn(bool move, bool in_side, bool out_side, uint32_t one, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int p = 0; p < D / 64; ++p)
#pragma unroll
      for (int t = 0; t < D / 64; ++t) {
        const int out = chunk_of(out_side, kChunks<D>, g >> 1, 2 * t + (g & 1));
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int in = chunk_of(in_side, kChunks<D>, c, 2 * p + e);
          const uint32_t v = move ? (in == out ? one & 0xFFFFu : 0u) : (one & 0xFFFFu) ^ (__popc(in & out) & 1) << 15;
          r |= v << (16 * e);
        }
        b[p][t] = r;
      }
  }
};
// float32 as two of tf32, which have 11 significant bits and are cut off: 2^-20 of an element is left over at most (`b`: a pair of bf16, exact in tf32)
struct Tf32 {
  uint32_t high, low;
  __device__ __forceinline__ explicit Tf32(float x) {
    high = __float_as_uint(x) & 0xFFFFE000u;
    low = __float_as_uint(x - __uint_as_float(high));
  }
};
__device__ __forceinline__ void mma_1688_tf32(float (&d)[4], const Tf32& a0, const Tf32& a1, const Tf32& a2, const Tf32& a3, uint32_t b) {
  const auto part = [&](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b << 16), "r"(b & 0xFFFF0000u));
  };
  part(a0.low, a1.low, a2.low, a3.low);
  part(a0.high, a1.high, a2.high, a3.high);
}
__device__ __forceinline__ void mma_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(b));
}
// two lanes of float32 arithmetic in one instruction
__device__ __forceinline__ void turn2(float& x0, float& x1, float k0, float k1, float y0, float y1, float l0, float l1) {     // x k + y l
  asm("{\n\t.reg .b64 x, k, y, l;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 k, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 l, {%6, %7};\n\tmul.rn.f32x2 x, x, k;\n\t"
      "fma.rn.f32x2 x, y, l, x;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(x0), "+f"(x1) : "f"(k0), "f"(k1), "f"(y0), "f"(y1), "f"(l0), "f"(l1));
}
__device__ __forceinline__ float max_nan(float x, float y) {                                   // of magnitudes; a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(x)), "f"(fabsf(y)));
  return r;
}
// the H_8 part: over the first index
template <int kTiles>
__device__ __forceinline__ void across(float (&v)[8][kTiles][4]) {
#pragma unroll
  for (int h = 1; h < 8; h *= 2)
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (!(b & h))
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = v[b][t][i], y = v[b + h][t][i];
            v[b][t][i] = x + y;
            v[b + h][t][i] = x - y;
          }
}

// the low halves of the bytes of x, the high ones of y
__device__ __forceinline__ uint32_t low_of(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xE4;" : "=r"(r) : "r"(x), "r"(y), "n"(0x0F0F0F0Fu));
  return r;
}
// the codes of two words, 8 each, as fp16 pairs (x's, y's) of the same place
__device__ __forceinline__ void pairs_of(uint32_t x, uint32_t y, uint32_t (&r)[8]) {
  uint32_t even[4], odd[4];
  from_e2m1(low_of(x, y << 4), even);
  from_e2m1(low_of(x >> 4, y), odd);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[2 * j] = even[j];
    r[2 * j + 1] = odd[j];
  }
}

// a row's scale from its largest magnitude (NaN stays), and the division by it; elements come as x, and are x * by (a power of two)
struct Scale {
  float s, inv, less;
  __device__ __forceinline__ explicit Scale(float most, float by = 1.f) {
    most *= by;
    s = most != most ? most : fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(__fdiv_rn(most, 6.f))), kScaleLeast), kScaleMost);
    less = s * (1.f / by);
    inv = __fdiv_rn(by, s);
  }
  // x * by / s, to the nearest where it is one of the values between two codes: a tie stays one
  __device__ __forceinline__ float operator()(float x) const {
    const float y = x * inv;
    return fmaf(fmaf(-y, less, x), inv, y);
  }
  // there is more than the largest scale admits (an infinity, too): what an element is then taken for
  __device__ __forceinline__ bool beyond(float most, float by = 1.f) const { return most * by > 6.f * kScaleMost; }
  __device__ __forceinline__ float within(float x) const { return fminf(fmaxf(x, -6.f * less), 6.f * less); }
};

template <typename T>
__device__ __forceinline__ void widen(const uint4& raw, float (&v)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Half<T>::wide(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// ---- the cache's writing side -----------------------------------------------------------------------------------------------------

struct AppendArgs {
  const void* qkv;
  long long row_stride;                                    // elements
  const int *positions, *slots;
  int tokens;
  const float *cosv, *sinv;
  int angle_rows, half, q_heads, kv_heads;                 // half: pairs that are rotated
  uint8_t *k_cache, *v_cache;
  uint16_t *k_scale, *v_scale;
  long long slots_total;
  int shift;
  void* q_out;
  int* status;
};

constexpr int kAppendThreads = 256, kMaxPage = 128;
template <int D>
constexpr int kAppendTokens = kAppendThreads / (D / 8);    // of a thread block

// Which of the tokens t0 ... t0 + n - 1 are written: s_slot their slots (from place `page` on, and of a page before them; -1: not valid), s_bad 0 for those that are
// written, 2 for those that are not although their slot is not -1.  By all threads, which are in step after it.
template <int kThreads>
__device__ __forceinline__ void find_written(const AppendArgs& a, int t0, int n, int* s_slot, int* s_pos, int* s_bad) {
  const int tid = threadIdx.x, page = 1 << a.shift;
  for (int i = tid; i < page + n; i += kThreads) {
    const int t = t0 - page + i;
    const int slot = t >= 0 ? a.slots[t] : -1, pos = t >= 0 ? a.positions[t] : -1;
    const bool ok = slot >= 0 && slot < a.slots_total && pos >= 0 && pos < a.angle_rows;
    if (i >= page) {
      s_pos[i - page] = pos;
      s_bad[i - page] = ok ? 0 : slot == -1 ? 1 : 2;
    }
    s_slot[i] = ok ? slot : -1;
  }
  __syncthreads();
  if (t0 + n > 1)
    for (int w = tid >> 5; w < n; w += kThreads / 32) {
      const int slot = s_slot[page + w];
      bool bad = false;
      for (int i = 1 + (tid & 31); i < page; i += 32) {
        const int other = s_slot[page + w - i];
        bad |= other >= slot && other >> a.shift == slot >> a.shift;
      }
      if (__any_sync(kFullWarp, bad) && slot >= 0 && (tid & 31) == 0) s_bad[w] = 2;
    }
  __syncthreads();
  if (a.status && blockIdx.y == 0)
    for (int i = tid; i < n; i += kThreads)
      if (s_bad[i] == 2) atomicOr(a.status, 16);
}

// grid (kAppendTokens tokens each, heads of queries, keys and values as they stand in a row).  A thread holds 8 dimensions of a row, four pairs
// of neighbours; in halves a pair's other element comes from another lane.
// A token whose slot does not lie above those of its page in the page - 1 tokens before it is not written: every place has one writer, where the tokens of a
// page lie within so many.
// Bound by latency: slots -> rows and angles -> sums over lanes.  8 tokens of 32 heads of 128 on 8 in a chain of launches: 2.5 us.
template <typename T, int D, bool kHalves>
__global__ void __launch_bounds__(kAppendThreads) rope_append4_kernel(const AppendArgs a) {
  constexpr int kLanes = D / 8, kTokens = kAppendTokens<D>;
  __shared__ int s_slot[kTokens + kMaxPage], s_pos[kTokens], s_bad[kTokens];
  pdl_enter();
  const int tid = threadIdx.x, lane = tid % kLanes, row = tid / kLanes, page = 1 << a.shift;
  const int t0 = blockIdx.x * kTokens, n = min(kTokens, a.tokens - t0), h = blockIdx.y;
  find_written<kAppendThreads>(a, t0, n, s_slot, s_pos, s_bad);
  const bool first = 8 * lane < a.half, turned = 8 * lane < 2 * a.half;          // (halves) this lane's are the first of their pairs; they are rotated
  const int w = min(row, n - 1), slot = s_slot[page + w];
  const bool mine = row < n, ok = s_bad[w] == 0;
  const size_t t = t0 + w;
  const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.qkv) + t * a.row_stride + (size_t)h * D + lane * 8);
  float v[8];
  if (h < a.q_heads + a.kv_heads) {
    constexpr int kAngles = kHalves ? 8 : 4;
    float cs[kAngles], sn[kAngles];
    const int from = !turned ? 0 : kHalves ? 8 * lane - (first ? 0 : a.half) : 4 * lane;
    const size_t at = (ok ? (size_t)s_pos[w] * a.half : 0) + from;
#pragma unroll
    for (int j = 0; j < kAngles; j += 4) {
      const float4 c = *reinterpret_cast<const float4*>(a.cosv + at + j), s = *reinterpret_cast<const float4*>(a.sinv + at + j);
      cs[j] = c.x; cs[j + 1] = c.y; cs[j + 2] = c.z; cs[j + 3] = c.w;
      sn[j] = s.x; sn[j + 1] = s.y; sn[j + 2] = s.z; sn[j + 3] = s.w;
    }
    widen<T>(raw, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= kDown / D;
    if constexpr (kHalves) {
      const int other = lane + (turned ? first ? a.half / 8 : -a.half / 8 : 0);
      const float sign = first ? -1.f : 1.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __shfl_sync(kFullWarp, v[j], other, kLanes);
        if (turned) v[j] = v[j] * cs[j] + sign * p * sn[j];
      }
    } else if (turned) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = v[2 * j], y = v[2 * j + 1];
        v[2 * j] = x * cs[j] - y * sn[j];
        v[2 * j + 1] = x * sn[j] + y * cs[j];
      }
    }
    hadamard<D>(v, lane);
    const float by = (h < a.q_heads ? 8.f : D / 8.f) / kDown;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (v[j] + (v[j] - v[j])) * by;            // (an infinity here, which only an infinite element or angle can have made, becomes NaN)
  } else {
    widen<T>(raw, v);
  }
  if (h < a.q_heads) {
    uint4 r = {Half<T>::narrow(v[0], v[1]), Half<T>::narrow(v[2], v[3]), Half<T>::narrow(v[4], v[5]), Half<T>::narrow(v[6], v[7])};
    if (!ok) r = {0, 0, 0, 0};
    if (mine) *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (t * a.q_heads + h) * D + lane * 8) = r;
    return;
  }
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max_nan(most, v[j]);
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) most = max_nan(most, __shfl_xor_sync(kFullWarp, most, o));
  const Scale scale(most);                                 // (a row with a NaN: so are all of its values, by their scale)
  if (scale.beyond(most))
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = scale.within(v[j]);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = scale(v[j]);
  if (!mine || !ok) return;
  const bool values = h >= a.q_heads + a.kv_heads;
  const int head = h - a.q_heads - (values ? a.kv_heads : 0);
  const size_t place = (((size_t)(slot >> a.shift) * a.kv_heads + head) << a.shift) + (slot & (page - 1));
  *reinterpret_cast<uint32_t*>((values ? a.v_cache : a.k_cache) + place * (D / 2) + lane * 4) = to_e2m1(v);
  if (lane == 0) (values ? a.v_scale : a.k_scale)[place] = (uint16_t)(__float_as_uint(scale.s) >> 16);
}

// The same for many tokens: a warp takes 16 of them at a time, one head after the other, and transforms by matrix products.  The rotated elements enter as two
// tf32 each, which leave 2^-20 of an element at most.  (Two bf16, 2^-16, in half of the products took 28 us where this then took 30, but a code that lies next to a tie then comes
// out as its neighbour often enough to show: 5e-4 of the norm of fp16 keys, whose own rounding is 2e-4.)
// An infinity among a row's elements makes all of the row NaN.
// Sums over lanes, four shuffles an element, were what bound the form above here, then 65 us (now 53) for 4096 tokens of 32 heads of 128 on 8 (94 MB) in a chain of launches.  With products
// from registers 44, from shared memory, where all heads of 16 tokens are on their way at once, 33, and 28 with what a lane's chunks are known beforehand.
// Now 33 in either layout (2.9 TB/s; with the tf32 parts and the range of finite pairs).  What bounds it: some 1200 instructions for 16 rows, at half of the issue slots.  Of 128
// dimensions it holds 128 registers and spills 64 to 116 bytes a thread (halves, whole heads of bf16: 64 stored, 88 loaded; interleaved parts of heads: 4); of 64 none.
// The two forms are about level at 32768 rows, for heads of either size.  us, few / many, a launch of another kernel between two: 700 tokens of 48 heads of 128 11.7 / 10.6, 900 14.2 / 12.9, 500 of
// 80 13.6 / 12.9; 700 of 48 of 64 8.4 / 7.6.  In a chain of its own: 600 of 48 of 128 9.5 / 12.4, 900 13.1 / 13.4, 1200 16.5 / 13.3; of 64 700 7.2 / 7.9, 1200 11.0 / 8.6.
constexpr int kRowsThreads = 128, kRowsTokens = 16, kRowsHeads = 8, kManyRows = 32768;

// rows of tokens in shared memory, so far apart that lanes of two neighbouring tokens read different banks: elements, 64 bytes a piece; angles, 64 or (halves) 16 of 32
template <int D>
constexpr int kRowBytes = kRowsHeads * D * 2 + 64;
template <int D, bool kHalves>
constexpr int kAngleFloats = D / 2 + (kHalves ? 4 : 16);
template <int D, bool kHalves>
constexpr int kRowsSmem = kRowsTokens * (kRowBytes<D> + 8 * kAngleFloats<D, kHalves>);

// kFull: all of a head is rotated, and then a lane knows which of its chunks are the first of their pairs
template <typename T, int D, bool kHalves, bool kFull>
__global__ void __launch_bounds__(kRowsThreads, 4) rope_append4_rows_kernel(const AppendArgs a) {
  constexpr int kWarps = kRowsThreads / 32, kTiles = D / 64, kAngles = kAngleFloats<D, kHalves>;
  const int pairs = kFull ? D / 2 : a.half;
  extern __shared__ __align__(128) uint8_t rows_smem[];
  float *cos_s = reinterpret_cast<float*>(rows_smem + kRowsTokens * kRowBytes<D>), *sin_s = cos_s + kRowsTokens * kAngles;
  __shared__ int s_slot[kRowsTokens + kMaxPage], s_pos[kRowsTokens], s_bad[kRowsTokens];
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3, page = 1 << a.shift;
  const int t0 = blockIdx.x * kRowsTokens, n = min(kRowsTokens, a.tokens - t0);
  const int h0 = blockIdx.y * kRowsHeads, heads = min(kRowsHeads, a.q_heads + 2 * a.kv_heads - h0);
  {                                                        // all heads of the tokens are on their way while the slots are looked at
    const uint8_t* from = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.qkv) + (size_t)t0 * a.row_stride + (size_t)h0 * D);
    const int pieces = heads * D / 8;                      // of a token, 16 bytes each
    for (int w = warp; w < n; w += kWarps)
      for (int i = lane; i < pieces; i += 32) copy16(smem_u32(rows_smem + w * kRowBytes<D> + 16 * i), from + (size_t)w * a.row_stride * 2 + 16 * i);
  }
  find_written<kRowsThreads>(a, t0, n, s_slot, s_pos, s_bad);
  if (h0 < a.q_heads + a.kv_heads)
    for (int w = warp; w < n; w += kWarps) {
      const size_t at = s_bad[w] == 0 ? (size_t)s_pos[w] * pairs : 0;
      for (int i = lane; i < pairs / 2; i += 32) {        // cosines, then sines
        const int z = i < pairs / 4 ? i : i - pairs / 4;
        copy16(smem_u32((i < pairs / 4 ? cos_s : sin_s) + w * kAngles + 4 * z), (i < pairs / 4 ? a.cosv : a.sinv) + at + 4 * z);
      }
    }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (h0 < a.q_heads + a.kv_heads)                         // angles times kDown, by the threads that fetched them
    for (int w = warp; w < n; w += kWarps)
      for (int i = lane; i < pairs / 2; i += 32) {
        float4* const at = reinterpret_cast<float4*>((i < pairs / 4 ? cos_s : sin_s - pairs) + w * kAngles + 4 * i);
        const float4 f = *at;
        *at = make_float4(f.x * kDown, f.y * kDown, f.z * kDown, f.w * kDown);
      }
  __syncthreads();
  for (int h = h0 + warp; h < h0 + heads; h += kWarps) {
    const bool turns = h < a.q_heads + a.kv_heads, query = h < a.q_heads;
    // rows g and g + 8; those behind the last are its
    int w[2];
    const uint8_t* row[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      w[r] = min(g + 8 * r, n - 1);
      row[r] = rows_smem + w[r] * kRowBytes<D> + (h - h0) * D * 2;
    }
    float v[8][kTiles][4];                                 // of dimension b of chunk 2 t + i % 2, row g + 8 (i / 2)
    if (turns) {
      // times 1 / D, which with kDown of the angles the scale of keys makes up for; queries times 8 / D / kDown
      const Turn<D> turn(false, true, query, (D == 128 ? 0x3C003C00u : 0x3C803C80u) + (query ? 0x03800380u : 0), lane);
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int t = 0; t < kTiles; ++t) v[b][t][0] = v[b][t][1] = v[b][t][2] = v[b][t][3] = 0.f;
#pragma unroll
      for (int p = 0; p < kTiles; ++p) {
        float x[2][2][8];                                  // rows, chunks of the pair
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float *cs_at = cos_s + w[r] * kAngles, *sn_at = sin_s + w[r] * kAngles;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = 8 * chunk_of(true, kChunks<D>, c, 2 * p + e);
            widen<T>(*reinterpret_cast<const uint4*>(row[r] + 2 * at), x[r][e]);
            if (!kFull && at >= 2 * pairs) {
#pragma unroll
              for (int b = 0; b < 8; ++b) x[r][e][b] *= kDown;
              continue;
            }
            if constexpr (kHalves) {
              const bool first = kFull ? 2 * p + e < kChunks<D> / 2 : at < pairs;
              const int other = first ? at + pairs : at - pairs, angle = first ? at : other;
              const uint32_t sign = first ? 0x80008000u : 0;
              uint4 raw = *reinterpret_cast<const uint4*>(row[r] + 2 * other);
              raw.x ^= sign; raw.y ^= sign; raw.z ^= sign; raw.w ^= sign;
              float y[8];
              widen<T>(raw, y);
#pragma unroll
              for (int z = 0; z < 8; z += 4) {
                const float4 cs = *reinterpret_cast<const float4*>(cs_at + angle + z), sn = *reinterpret_cast<const float4*>(sn_at + angle + z);
                turn2(x[r][e][z], x[r][e][z + 1], cs.x, cs.y, y[z], y[z + 1], sn.x, sn.y);
                turn2(x[r][e][z + 2], x[r][e][z + 3], cs.z, cs.w, y[z + 2], y[z + 3], sn.z, sn.w);
              }
            } else {
              const float4 cs = *reinterpret_cast<const float4*>(cs_at + at / 2), sn = *reinterpret_cast<const float4*>(sn_at + at / 2);
              const float k[4] = {cs.x, cs.y, cs.z, cs.w}, l[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float y = x[r][e][2 * j], z = x[r][e][2 * j + 1];
                x[r][e][2 * j] = y * k[j] - z * l[j];
                x[r][e][2 * j + 1] = y * l[j] + z * k[j];
              }
            }
          }
        }
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const Tf32 a0(x[0][0][b]), a1(x[1][0][b]), a2(x[0][1][b]), a3(x[1][1][b]);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) mma_1688_tf32(v[b][t], a0, a1, a2, a3, turn.b[p][t]);
        }
      }
      across(v);
    } else {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int y = 0; y < kChunks<D>; ++y) {
          float x[8];
          widen<T>(*reinterpret_cast<const uint4*>(row[r] + 16 * chunk_of(false, kChunks<D>, c, y)), x);
#pragma unroll
          for (int b = 0; b < 8; ++b) v[b][y >> 1][2 * r + (y & 1)] = x[b];
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool mine = g + 8 * r < n, ok = s_bad[w[r]] == 0;
      if (query) {
        if (!ok)
#pragma unroll
          for (int b = 0; b < 8; ++b)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) v[b][t][2 * r] = v[b][t][2 * r + 1] = 0.f;
#pragma unroll
        for (int y = 0; y < kChunks<D>; ++y) {
          const int t = y >> 1, i = 2 * r + (y & 1);
          const uint4 out = {Half<T>::narrow(v[0][t][i], v[1][t][i]), Half<T>::narrow(v[2][t][i], v[3][t][i]), Half<T>::narrow(v[4][t][i], v[5][t][i]), Half<T>::narrow(v[6][t][i], v[7][t][i])};
          if (mine) *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + ((size_t)(t0 + w[r]) * a.q_heads + h) * D + 8 * chunk_of(true, kChunks<D>, c, y)) = out;
        }
        continue;
      }
      float most = 0.f;
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int y = 0; y < kChunks<D>; ++y) most = max_nan(most, v[b][y >> 1][2 * r + (y & 1)]);
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) most = max_nan(most, __shfl_xor_sync(kFullWarp, most, o));
      const float by = turns ? D / 8.f / kDown : 1.f;
      const Scale scale(most, by);
      if (scale.beyond(most, by))
#pragma unroll
        for (int b = 0; b < 8; ++b)
#pragma unroll
          for (int y = 0; y < kChunks<D>; ++y) v[b][y >> 1][2 * r + (y & 1)] = scale.within(v[b][y >> 1][2 * r + (y & 1)]);
      uint32_t codes[kChunks<D>];
#pragma unroll
      for (int y = 0; y < kChunks<D>; ++y) {
        float x[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) x[b] = scale(v[b][y >> 1][2 * r + (y & 1)]);
        codes[y] = to_e2m1(x);
      }
      if (!mine || !ok) continue;
      const int slot = s_slot[page + w[r]], head = h - a.q_heads - (turns ? 0 : a.kv_heads);
      const size_t place = (((size_t)(slot >> a.shift) * a.kv_heads + head) << a.shift) + (slot & (page - 1));
      uint8_t* to = (turns ? a.k_cache : a.v_cache) + place * (D / 2) + 4 * kChunks<D> * c;
      if constexpr (D == 128) *reinterpret_cast<uint4*>(to) = {codes[0], codes[1], codes[2], codes[3]};
      else *reinterpret_cast<uint2*>(to) = {codes[0], codes[1]};
      if (c == 0) (turns ? a.k_scale : a.v_scale)[place] = (uint16_t)(__float_as_uint(scale.s) >> 16);
    }
  }
}

// ---- pages as values --------------------------------------------------------------------------------------------------------------

struct UnpackArgs {
  const uint8_t *k_cache, *v_cache;
  const uint16_t *k_scale, *v_scale;
  const int* ids;
  int kv_heads, shift, pages;
  void *k_out, *v_out;
};

constexpr int kUnpackThreads = 64;

template <typename T>
__device__ __forceinline__ void put8(T* to, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = {Half<T>::narrow(v[0], v[1]), Half<T>::narrow(v[2], v[3]), Half<T>::narrow(v[4], v[5]), Half<T>::narrow(v[6], v[7])};
}
template <>
__device__ __forceinline__ void put8<float>(float* to, const float (&v)[8]) {
  *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// A warp takes 16 tokens of keys, which it turns back (H H = D), or of values, which pass through the same products only to lie side by side.  The sums are those of
// codes, exact; one multiplication by the scale, and one rounding.  Bound by what it writes: 901 pages of 64 tokens, 8 heads of 128 (297 MB) in 54 us in a chain of
// launches, 5.5 TB/s.  (Sums over lanes: 78.  Warps that stay and fetch ahead: 87, their registers spill.)
template <typename T, int D>
__global__ void __launch_bounds__(kUnpackThreads) unpack4_kernel(const UnpackArgs a, long long pieces) {
  constexpr int kTiles = D / 64;
  pdl_enter();
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const long long n = (long long)blockIdx.x * (kUnpackThreads / 32) + (threadIdx.x >> 5);        // piece: 16 tokens; keys and values in turns
  if (n >= pieces) return;
  const bool values = n & 1;
  const long long sixteen = n >> 1;                        // of the output
  const int unit = (int)(sixteen >> (a.shift - 4)), i = unit / a.kv_heads, head = unit - i * a.kv_heads, id = a.ids[i];
  const bool real = id >= 0 && id < a.pages;
  const size_t from = (((size_t)(real ? id : 0) * a.kv_heads + head) << a.shift) + 16 * (sixteen & ((1 << (a.shift - 4)) - 1)), to = (size_t)sixteen * 16;
  uint32_t w[2][kChunks<D>];
  float scale[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const size_t row = from + g + 8 * r;
    const uint8_t* src = (values ? a.v_cache : a.k_cache) + row * (D / 2) + 4 * kChunks<D> * c;
    if constexpr (D == 128) {
      const uint4 x = *reinterpret_cast<const uint4*>(src);
      w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(src);
      w[r][0] = x.x; w[r][1] = x.y;
    }
    scale[r] = real ? of_bf16((values ? a.v_scale : a.k_scale)[row]) * (values ? 1.f : 8.f / D) : 0.f;        // (codes are finite: zeros)
  }
  const Turn<D> turn(values, false, true, 0x3C003C00u, lane);
  float v[8][kTiles][4];
#pragma unroll
  for (int b = 0; b < 8; ++b)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) v[b][t][0] = v[b][t][1] = v[b][t][2] = v[b][t][3] = 0.f;
#pragma unroll
  for (int p = 0; p < kTiles; ++p) {
    uint32_t x[2][8];
#pragma unroll
    for (int r = 0; r < 2; ++r) pairs_of(w[r][2 * p], w[r][2 * p + 1], x[r]);
#pragma unroll
    for (int b = 0; b < 8; ++b)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) mma_1688(v[b][t], x[0][b], x[1][b], turn.b[p][t]);
  }
  if (!values) across(v);
  T* out = static_cast<T*>(values ? a.v_out : a.k_out);
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int y = 0; y < kChunks<D>; ++y) {
      float x[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) x[b] = v[b][y >> 1][2 * r + (y & 1)] * scale[r];
      put8<T>(out + (to + g + 8 * r) * D + 8 * chunk_of(true, kChunks<D>, c, y), x);
    }
}

// ---- attention over the cache, few rows a request ---------------------------------------------------------------------------------
//
// As over the 8-bit cache (paged_kernels.cu): rows are query heads times tokens, the cache is the 16-row operand of m16n8k16, a warp takes tiles of the
// cache for itself, work is cut evenly and joined.  What differs:
//  * a tile has 32 tokens, in two halves that may lie in different pages; what a tile costs besides its tokens is paid half as often;
//  * tiles come by 16-byte asynchronous copies of all lanes.  (Eight bulk copies a tile, as halves, keys, values and scales lie apart, are issued lane by lane, 100 instructions:
//    99 us where this took 86.)  No wait here depends on another thread but __syncwarp;
//  * a byte is two neighbouring dimensions of a token, which is what a register of the keys' fragment holds; for values it has to be two neighbouring
//    tokens of one dimension: two bitwise selections make such bytes of the words of two tokens;
//  * scales belong to tokens: those of keys multiply the scores, those of values enter the exponent (P' = 2^(s + log2 scale - m)) and the sum takes them out.
//    A lane makes these numbers for one token of the tile, and all fetch what they need from shared memory.
// Row i of a half is its token i ^ (i >> 1 & 1): neighbouring lanes then read rows of both parities, which lie in different banks.
//
// 64 requests of 10 to 16384 tokens, 32 heads of 128 on 8 (392 MB): 80 us in a chain of launches, 4.9 TB/s; 64 of 16383 (1.1 GB): 192 us, 5.8 TB/s.  Two steps
// of such a length differ by what their bytes take at 6.3 TB/s; the rest, some 16 us, is begin, end and join.  At the size above copies without products
// take 67 us, products without copies 71: 434 instructions a tile at half of the issue slots, the conversions (two cycles each, with all other integer
// instructions) at half of their pipe.  Tried without gain: four thread blocks on an SM (spills: 82 to 95), rings of two or four tiles, the first tiles of the next item
// requested before the results of one are joined (82).

constexpr int kTile = 32, kUnit = kAttWarps * kTile, kDepth = 3;
constexpr int kBegin = 3;                                  // what an item costs besides its units
using Work = Span<kUnit, kBegin>;
template <int D, int NT>
constexpr int kAttBlocks = D == 128 ? (NT == 1 ? 3 : 2) : (NT == 1 ? 4 : 3);
template <int D>
constexpr int kKeys = kTile * D / 2;                       // bytes of a tile's keys, and of its values
template <int D>
constexpr int kStage = 2 * kKeys<D> + 4 * kTile;           // with their scales behind them

template <int D, int NT>
struct Running : Results<D, NT> {
  using Results<D, NT>::o;
  using Results<D, NT>::m;
  using Results<D, NT>::l;
  // a tile's tokens from `at` on; `least`: tokens that every row sees; `real`: halves that have a page; `read`: called when nothing of the stage is needed any more
  template <typename R, typename F>
  __device__ __forceinline__ void add(const uint8_t* stage, float4* wide, const R& rows, int at, int least, unsigned real, int lane, F read) {
    const int g = lane >> 2, c = lane & 3, pi = g ^ (g >> 1 & 1);
    // scales of token `lane` of the tile
    const uint16_t* scales = reinterpret_cast<const uint16_t*>(stage + 2 * kKeys<D>) + lane;
    const float my_ks = of_bf16(scales[0]), vs = of_bf16(scales[kTile]);
    const float held = fminf(fmaxf(vs, kScaleLeast), kScaleMost);      // (NaN: kScaleLeast, and the logarithm becomes NaN by what is added)
    wide[lane] = make_float4(my_ks, __log2f(held) + (vs - vs), __fdividef(kSumUnit, held), 0.f);
    __syncwarp();
    float s[2][NT][4], ks[2][2], lv[2][2], inv[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < NT; ++t) s[h][t][0] = s[h][t][1] = s[h][t][2] = s[h][t][3] = 0.f;
      uint32_t k[2][D / 32];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = 16 * h + 8 * u + pi;
        if constexpr (D == 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(stage + row * 64 + 16 * c);
          k[u][0] = w.x; k[u][1] = w.y; k[u][2] = w.z; k[u][3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(stage + row * 32 + 8 * c);
          k[u][0] = w.x; k[u][1] = w.y;
        }
        const float4 f = wide[row];
        ks[h][u] = f.x;
        lv[h][u] = f.y;
        inv[h][u] = f.z;
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        uint32_t x[4], y[4];
        from_e2m1(k[0][w], x);
        from_e2m1(k[1][w], y);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_16816(s[h][t], x[0], y[0], x[1], y[1], rows.q[2 * w][t][0], rows.q[2 * w][t][1]);
          mma_16816(s[h][t], x[2], y[2], x[3], y[3], rows.q[2 * w + 1][t][0], rows.q[2 * w + 1][t][1]);
        }
      }
    }
    float top[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) top[t][0] = top[t][1] = kNone;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][t][i] = fmaf(s[h][t][i], rows.scale[t][i & 1] * ks[h][i >> 1], lv[h][i >> 1]);
    if (at + kTile > least || real != 3) {                 // tokens that some row does not see
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)                      // token pi + 8 (i / 2) of the half, row 2 c + i % 2
            if (!(real >> h & 1) || at + 16 * h + pi + 8 * (i >> 1) >= rows.end[t][i & 1]) s[h][t][i] = kNone;
    }
    bool grows = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        top[t][y] = fmaxf(fmaxf(s[0][t][y], s[0][t][2 + y]), fmaxf(s[1][t][y], s[1][t][2 + y]));
        grows |= top[t][y] > m[t][y] + 15.5f;
      }
    if (__any_sync(kFullWarp, grows)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) this->raise(t, y, top[t][y]);
    }
    uint32_t p[2][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float base[2] = {m[t][0] == kNone ? 0.f : m[t][0], m[t][1] == kNone ? 0.f : m[t][1]};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = exp2_fast(s[h][t][i] - base[i & 1]);
          l[t][i & 1] = fmaf(e[i], inv[h][i >> 1], l[t][i & 1]);
        }
        p[h][t][0] = transposed(pack_half(e[0], e[1]));
        p[h][t][1] = transposed(pack_half(e[2], e[3]));
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[4][D / 64];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = 16 * h + 8 * (x >> 1) + ((2 * c + (x & 1)) ^ (c & 1));
        if constexpr (D == 128) {
          const uint2 w = *reinterpret_cast<const uint2*>(stage + kKeys<D> + row * 64 + 8 * g);
          v[x][0] = w.x; v[x][1] = w.y;
        } else {
          v[x][0] = *reinterpret_cast<const uint32_t*>(stage + kKeys<D> + row * 32 + 4 * g);
        }
      }
      if (h == 1) read();
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {
        // bytes of two tokens' codes of one dimension: even ones, odd ones
        const auto even = [&](int x) { return low_of(v[x][w], v[x + 1][w] << 4); };
        const auto odd = [&](int x) { return low_of(v[x][w] >> 4, v[x + 1][w]); };
        uint32_t a0[4], a1[4], a2[4], a3[4];
        from_e2m1(even(0), a0);
        from_e2m1(odd(0), a1);
        from_e2m1(even(2), a2);
        from_e2m1(odd(2), a3);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(o[4 * w + j][t], a0[j], a1[j], a2[j], a3[j], p[h][t][0], p[h][t][1]);
      }
    }
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, (kAttBlocks<D, NT>)) paged4_attention_kernel(const AttentionArgs a) {
  constexpr int kRows = 8 * NT, kRing = kDepth * kStage<D>;
  static_assert(kRing >= kRows * (D + 4) * 4, "a warp's results lie where its tiles were");
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ WarpParts<kRows> parts;
  __shared__ Place place;
  __shared__ float4 s_wide[kAttWarps][kTile];
  __shared__ int s_fail;
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    a.cuts[blockIdx.x] = {0, 0, 0, 0};
    s_fail = 0;
  }
  const Begin<Work> begin(a, kRows, &place);
  if (begin.left <= 0) return;
  const long long share = begin.share;
  int r = begin.r;
  long long skip = begin.skip, left = begin.left;
  bool bad = false;
  uint8_t* const mine = ring + warp * kRing;
  // where this lane's 16 bytes of a copy come from and go: of keys and values, and of the scales (lanes 0 to 7: of keys and of values, two lanes for a half)
  const uint8_t *from_k = a.k_cache + 16 * lane, *from_v = a.v_cache + 16 * lane;
  const uint8_t* from_scale = reinterpret_cast<const uint8_t*>(lane & 4 ? a.v_scale : a.k_scale) + 16 * (lane & 1);
  for (int segment = 0; left > 0; ++segment) {
    const Work x(a, r, kRows);
    if (skip >= x.total) {
      skip -= x.total;
      ++r;
      --segment;
      continue;
    }
    const int item = (int)(skip / (x.units + kBegin)), w0 = (int)(skip % (x.units + kBegin)), w1 = (int)min((long long)x.units + kBegin, w0 + left);
    const int u0 = max(w0 - kBegin, 0), u1 = max(w1 - kBegin, 0);
    skip += w1 - w0;
    left -= w1 - w0;
    if (u1 <= u0) {                                        // (only of what an item costs besides its units)
      --segment;
      continue;
    }
    const int kvh = item % a.kv_heads, row0 = item / a.kv_heads * kRows, rows = min(x.rows - row0, kRows);
    const int last_token = (row0 + rows - 1) / a.group;
    const int least = max(x.seen - x.n + row0 / a.group + 1, 0), end = max(x.seen - x.n + last_token + 1, 0);
    if (segment) __syncthreads();                          // the results of the last tile have been read
    // ---- the tiles of this warp: kDepth are on their way.  Lane i holds the place of half i of 16 tiles, and of the 16 after them, which are fetched in time:
    // in units of 16 tokens of a head, which are 8 D bytes of keys (int32 holds those of any memory).
    const int* table = a.tables + r * a.table_stride;
    const int stop = min(u1 * kUnit, end), first_at = u0 * kUnit + warp * kTile;
    const int tiles = first_at < stop ? (stop - first_at + kUnit - 1) / kUnit : 0;
    int some, then;
    const auto places_of = [&](int tile) {                 // -1: no page, or none of this warp's tokens
      const int token = first_at + (tile + (lane >> 1)) * kUnit + 16 * (lane & 1);
      if (token >= stop) return -1;
      const int id = table[token >> a.shift];
      const bool real = id >= 0 && id < a.pages;           // no such page: its tokens are not seen
      bad |= !real;
      return real ? ((id * a.kv_heads + kvh) << (a.shift - 4)) + ((token & ((1 << a.shift) - 1)) >> 4) : -1;
    };
    // tile `tile` into the stage at `to`, by all lanes, which have read what was there.  What has no page stays what it was.
    const auto request = [&](int tile, int places, uint8_t* to) {
      const uint32_t stage = smem_u32(to) + 16 * lane;
      int at[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        at[h] = __shfl_sync(kFullWarp, places, (2 * tile + h) & 31);
        if (at[h] < 0) continue;
        const uint8_t *k = from_k + (size_t)(unsigned)at[h] * (8 * D), *v = from_v + (size_t)(unsigned)at[h] * (8 * D);
#pragma unroll
        for (int y = 0; y < D / 64; ++y) {
          copy16(stage + h * 8 * D + 512 * y, k + 512 * y);
          copy16(stage + kKeys<D> + h * 8 * D + 512 * y, v + 512 * y);
        }
      }
      const int one = lane & 2 ? at[1] : at[0];
      if (lane < 8 && one >= 0) copy16(stage + 2 * kKeys<D>, from_scale + (size_t)(unsigned)one * 32);
    };
    const auto done = [&] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    some = then = places_of(0);
    for (int i = 0; i < kDepth; ++i) {
      if (i < tiles) request(i, some, mine + i * kStage<D>);
      done();
    }
    Rows<T, D, NT, D / 4> q;
    q.load(a, x.start, x.n, x.seen, row0, kvh, lane);
    Running<D, NT> run;
    run.clear();
    uint8_t* stage = mine;
    unsigned real = 0;
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      if ((i & 15) == 0) {
        if (i) some = then;
        if (i + 16 < tiles) then = places_of(i + 16);
        real = __ballot_sync(kFullWarp, some >= 0);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      __syncwarp();
      run.add(stage, s_wide[warp], q, first_at + i * kUnit, least, real & 3, lane, [&] {
        __syncwarp();
        if (i + kDepth < tiles) request(i + kDepth, (i & 15) + kDepth < 16 ? some : then, stage);
        done();
      });
      real >>= 2;
      stage += kStage<D>;
      if (stage == mine + kRing) stage = mine;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const bool whole = u0 == 0 && u1 == x.units;
    finish<T, D, NT, kRing>(a, run, ring, &parts, &s_fail, x, kvh, row0, rows, whole, segment != 0);
    if (!whole && u0 == 0 && tid == 0) {                   // it begins here and ends elsewhere: request, item, parts, place of the first
      const long long beyond = x.units - u1;
      a.cuts[blockIdx.x] = {r, item, 1 + (int)((beyond + share - 1) / share), segment != 0};
    }
  }
  if (__any_sync(kFullWarp, bad) && a.status && lane == 0) atomicOr(a.status, 32);
}

int attention_blocks(int head_dim, int tiles) {            // what the GPU holds at a time
  return current_device_sms() * (head_dim == 128 ? (tiles == 1 ? kAttBlocks<128, 1> : kAttBlocks<128, 2>) : tiles == 1 ? kAttBlocks<64, 1> : kAttBlocks<64, 2>);
}
int attention_tiles(int group, int max_new) { return (long long)group * max_new <= 8 ? 1 : 2; }

template <typename T, int D, int NT>
int attention_run(const AttentionArgs& a, cudaStream_t st) {
  const dim3 grid(attention_blocks(D, NT)), block(kAttThreads);
  constexpr int kBytes = kAttWarps * kDepth * kStage<D>;
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (!e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(paged4_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  if (e) return paged_fail(e);
  const int rc = paged_launch(paged4_attention_kernel<T, D, NT>, grid, block, 1, kBytes, st, a);
  return rc != HTR_OK ? rc : paged_launch(paged_attention_join_kernel<T, D, NT, Work>, dim3(grid.x, kJoins<D, NT>), block, 1, 0, st, a);
}

template <typename T>
int attention_of(const AttentionArgs& a, int head_dim, int max_new, cudaStream_t st) {
  if (attention_tiles(a.group, max_new) == 1) return head_dim == 128 ? attention_run<T, 128, 1>(a, st) : attention_run<T, 64, 1>(a, st);
  return head_dim == 128 ? attention_run<T, 128, 2>(a, st) : attention_run<T, 64, 2>(a, st);
}

template <typename T, int D, bool kHalves, bool kFull>
int append_rows(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  constexpr int kBytes = kRowsSmem<D, kHalves>;
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (kBytes > 40960 && !e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(rope_append4_rows_kernel<T, D, kHalves, kFull>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  return e ? paged_fail(e) : paged_launch(rope_append4_rows_kernel<T, D, kHalves, kFull>, grid, dim3(kRowsThreads), 1, kBytes, st, a);
}

template <typename T, int D>
int append_of(const AppendArgs& a, bool halves, cudaStream_t st) {
  const int heads = a.q_heads + 2 * a.kv_heads;
  if ((int64_t)a.tokens * heads >= kManyRows) {
    const dim3 grid((a.tokens + kRowsTokens - 1) / kRowsTokens, (heads + kRowsHeads - 1) / kRowsHeads);
    if (2 * a.half == D) return halves ? append_rows<T, D, true, true>(a, grid, st) : append_rows<T, D, false, true>(a, grid, st);
    return halves ? append_rows<T, D, true, false>(a, grid, st) : append_rows<T, D, false, false>(a, grid, st);
  }
  const dim3 grid((a.tokens + kAppendTokens<D> - 1) / kAppendTokens<D>, heads);
  return halves ? paged_launch(rope_append4_kernel<T, D, true>, grid, dim3(kAppendThreads), 1, 0, st, a)
                : paged_launch(rope_append4_kernel<T, D, false>, grid, dim3(kAppendThreads), 1, 0, st, a);
}

template <typename T>
int unpack_of(const UnpackArgs& a, int head_dim, int units, cudaStream_t st) {
  const long long pieces = ((long long)units << (a.shift - 4)) * 2;
  const long long blocks = (pieces + kUnpackThreads / 32 - 1) / (kUnpackThreads / 32);
  if (blocks > 0x7FFFFFFF) return HTR_ERR_TOO_LARGE;
  const dim3 grid((unsigned)blocks);
  return head_dim == 128 ? paged_launch(unpack4_kernel<T, 128>, grid, dim3(kUnpackThreads), 1, 0, st, a, pieces)
                         : paged_launch(unpack4_kernel<T, 64>, grid, dim3(kUnpackThreads), 1, 0, st, a, pieces);
}

}  // namespace

using namespace htr;

extern "C" {

int htr_paged4_append(const void* qkv, int dtype, int64_t row_stride, const int* positions, const int* slots, int tokens, const float* cosv,
                      const float* sinv, int angle_rows, int rotary_dim, int halves, int q_heads, int kv_heads, int head_dim, void* k_cache, void* v_cache,
                      void* k_scale, void* v_scale, int pages, int page_size, void* q_out, int* status, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16) return HTR_ERR_BAD_DTYPE;
  const int shift = page_shift(page_size);
  if (tokens < 0 || (head_dim != 64 && head_dim != 128) || q_heads < 1 || kv_heads < 1 || pages < 1 || shift < 0 || angle_rows < 1 || rotary_dim < 16 ||
      rotary_dim > head_dim || rotary_dim % 16 || row_stride < (q_heads + 2 * (int64_t)kv_heads) * head_dim || row_stride % 8)
    return HTR_ERR_BAD_SHAPE;
  if (q_heads > 16384 || kv_heads > 16384 || tokens > 1 << 30 || (int64_t)pages << shift > 0x7FFFFFFF) return HTR_ERR_TOO_LARGE;
  if (tokens == 0) return HTR_OK;
  if (!qkv || !positions || !slots || !cosv || !sinv || !k_cache || !v_cache || !k_scale || !v_scale || !q_out) return HTR_ERR_NULL;
  if (!aligned16(qkv) || !aligned16(cosv) || !aligned16(sinv) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale) ||
      !aligned16(q_out))
    return HTR_ERR_ALIGNMENT;
  const AppendArgs a = {qkv, row_stride, positions, slots, tokens, cosv, sinv, angle_rows, rotary_dim / 2, q_heads, kv_heads, static_cast<uint8_t*>(k_cache),
                        static_cast<uint8_t*>(v_cache), static_cast<uint16_t*>(k_scale), static_cast<uint16_t*>(v_scale), (int64_t)pages << shift, shift, q_out, status};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == HTR_DTYPE_BF16) return head_dim == 128 ? append_of<__nv_bfloat16, 128>(a, halves != 0, st) : append_of<__nv_bfloat16, 64>(a, halves != 0, st);
  return head_dim == 128 ? append_of<__half, 128>(a, halves != 0, st) : append_of<__half, 64>(a, halves != 0, st);
}

int htr_paged4_unpack(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale, int pages, int kv_heads, int page_size, int head_dim,
                      const int* ids, int count, void* k_out, void* v_out, int dtype, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16 && dtype != HTR_DTYPE_F32) return HTR_ERR_BAD_DTYPE;
  const int shift = page_shift(page_size);
  if (count < 0 || (head_dim != 64 && head_dim != 128) || kv_heads < 1 || pages < 1 || shift < 0) return HTR_ERR_BAD_SHAPE;
  if (kv_heads > 16384 || (int64_t)pages << shift > 0x7FFFFFFF || (int64_t)count * kv_heads > 0x7FFFFFFF) return HTR_ERR_TOO_LARGE;
  if (count == 0) return HTR_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !ids || !k_out || !v_out) return HTR_ERR_NULL;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale) || !aligned16(k_out) || !aligned16(v_out)) return HTR_ERR_ALIGNMENT;
  const UnpackArgs a = {static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), static_cast<const uint16_t*>(k_scale),
                        static_cast<const uint16_t*>(v_scale), ids, kv_heads, shift, pages, k_out, v_out};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int units = count * kv_heads;
  return dtype == HTR_DTYPE_BF16 ? unpack_of<__nv_bfloat16>(a, head_dim, units, st)
         : dtype == HTR_DTYPE_F16 ? unpack_of<__half>(a, head_dim, units, st) : unpack_of<float>(a, head_dim, units, st);
}

size_t htr_paged4_attention_workspace_bytes(int tokens, int requests, int q_heads, int kv_heads, int head_dim, int max_new, int table_width, int page_size) {
  if (tokens < 1 || requests < 1 || q_heads < 1 || kv_heads < 1 || max_new < 1 || table_width < 1 || page_shift(page_size) < 0 || (head_dim != 64 && head_dim != 128)) return 0;
  if (attention4_tc_serves(tokens, requests, q_heads, q_heads / kv_heads, max_new, (long long)table_width * page_size, head_dim)) return attention_tc_workspace(head_dim);
  const int tiles = attention_tiles(q_heads / kv_heads, max_new);
  const size_t rows = 8 * tiles;
  return attention_blocks(head_dim, tiles) * (2 * rows * (head_dim + 2) * sizeof(float) + sizeof(int4));
}

int htr_paged4_attention(const void* q, int dtype, int tokens, const int* starts, const int* seen, int requests, const int* tables,
                         int64_t table_stride, int table_width, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                         int pages, int page_size, int q_heads, int kv_heads, int head_dim, int max_new, float scale, void* out, int* status,
                         void* workspace, size_t workspace_bytes, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16) return HTR_ERR_BAD_DTYPE;
  const int shift = page_shift(page_size);
  if (tokens < 0 || requests < 1 || table_width < 1 || table_stride < table_width || (head_dim != 64 && head_dim != 128) || q_heads < 1 || kv_heads < 1 ||
      q_heads % kv_heads || pages < 1 || shift < 0 || max_new < 1)
    return HTR_ERR_BAD_SHAPE;
  if (requests > 8192 || kv_heads > 16384 || q_heads > 16384 || tokens > 1 << 30 || (int64_t)max_new * (q_heads / kv_heads) > 1 << 30 ||
      (int64_t)pages << shift > 0x7FFFFFFF || (int64_t)table_width << shift > 1 << 30)
    return HTR_ERR_TOO_LARGE;
  if (tokens == 0) return HTR_OK;
  if (!q || !starts || !seen || !tables || !k_cache || !v_cache || !k_scale || !v_scale || !out) return HTR_ERR_NULL;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale) || !aligned16(out)) return HTR_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < htr_paged4_attention_workspace_bytes(tokens, requests, q_heads, kv_heads, head_dim, max_new, table_width, page_size))
    return HTR_ERR_WORKSPACE;
  if (!aligned16(workspace)) return HTR_ERR_ALIGNMENT;
  int4* cuts = static_cast<int4*>(workspace);
  AttentionArgs a = {q, starts, seen, tables, table_stride, table_width, requests, tokens, q_heads, kv_heads, q_heads / kv_heads, max_new,
                     static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), static_cast<const float*>(k_scale),
                     static_cast<const float*>(v_scale), pages, shift, scale * 1.4426950408889634f, out, status, nullptr, cuts, attention_withhold()};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (attention4_tc_serves(tokens, requests, q_heads, a.group, max_new, (long long)table_width * page_size, head_dim)) return attention4_tc_run(a, dtype, head_dim, workspace, st);
  a.parts = reinterpret_cast<float*>(cuts + attention_blocks(head_dim, attention_tiles(a.group, max_new)));
  return dtype == HTR_DTYPE_BF16 ? attention_of<__nv_bfloat16>(a, head_dim, max_new, st) : attention_of<__half>(a, head_dim, max_new, st);
}

}  // extern "C"
