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

constexpr float kScaleLeast = 7.888609052210118e-31f, kScaleMost = 6.646139978924579e35f;          // 2^-100, 2^119

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
  int shift, window;
  void* q_out;
  int* status;
};

constexpr int kAppendThreads = 256, kMaxWindow = 64, kMaxPage = 128;

// grid (windows of tokens, groups of kHeads heads of queries, keys and values as they stand in a row).  A thread holds 8 dimensions of a row, four pairs
// of neighbours; in halves a pair's other element comes from another lane.
// A token whose slot does not lie above those of its page in the page - 1 tokens before it is not written: every place has one writer.
template <typename T, int D, int kHeads, bool kHalves>
__global__ void __launch_bounds__(kAppendThreads) rope_append4_kernel(const AppendArgs a) {
  constexpr int kLanes = D / 8, kRows = kAppendThreads / kLanes, kWarps = kAppendThreads / 32;
  __shared__ int s_slot[kMaxWindow + kMaxPage], s_pos[kMaxWindow];
  __shared__ int s_bad[kMaxWindow];
  pdl_enter();
  const int tid = threadIdx.x, lane = tid % kLanes, row = tid / kLanes, page = 1 << a.shift;
  const int t0 = blockIdx.x * a.window, n = min(a.window, a.tokens - t0), h0 = blockIdx.y * kHeads;
  const T* qkv = static_cast<const T*>(a.qkv);
  // ---- which of the tokens are written: slots of the window (from place `page` on) and of a page before it
  for (int i = tid; i < page + n; i += kAppendThreads) {
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
    for (int w = tid >> 5; w < n; w += kWarps) {
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
    for (int i = tid; i < n; i += kAppendThreads)
      if (s_bad[i] == 2) atomicOr(a.status, 16);
  const bool first = 8 * lane < a.half, turned = 8 * lane < 2 * a.half;          // (halves) this lane's are the first of their pairs; they are rotated
  for (int w0 = 0; w0 < n; w0 += kRows) {
    const int w = min(w0 + row, n - 1), slot = s_slot[page + w];
    const bool mine = w0 + row < n, ok = s_bad[w] == 0;
    const size_t t = t0 + w;
    uint4 raw[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (h0 + i < a.q_heads + 2 * a.kv_heads) raw[i] = *reinterpret_cast<const uint4*>(qkv + t * a.row_stride + (size_t)(h0 + i) * D + lane * 8);
    constexpr int kAngles = kHalves ? 8 : 4;
    float cs[kAngles], sn[kAngles];
    if (h0 < a.q_heads + a.kv_heads) {
      const int from = !turned ? 0 : kHalves ? 8 * lane - (first ? 0 : a.half) : 4 * lane;
      const size_t at = (ok ? (size_t)s_pos[w] * a.half : 0) + from;
#pragma unroll
      for (int j = 0; j < kAngles; j += 4) {
        const float4 c = *reinterpret_cast<const float4*>(a.cosv + at + j), s = *reinterpret_cast<const float4*>(a.sinv + at + j);
        cs[j] = c.x; cs[j + 1] = c.y; cs[j + 2] = c.z; cs[j + 3] = c.w;
        sn[j] = s.x; sn[j + 1] = s.y; sn[j + 2] = s.z; sn[j + 3] = s.w;
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i;
      if (h >= a.q_heads + 2 * a.kv_heads) break;
      float v[8];
      widen<T>(raw[i], v);
      if (h < a.q_heads + a.kv_heads) {
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
        // (so that no finite ones add up to an infinity on the way)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= 1.f / D;
        hadamard<D>(v, lane);
        const float by = h < a.q_heads ? 8.f : D / 8.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= by;
      }
      if (h < a.q_heads) {
        uint4 r = {Half<T>::narrow(v[0], v[1]), Half<T>::narrow(v[2], v[3]), Half<T>::narrow(v[4], v[5]), Half<T>::narrow(v[6], v[7])};
        if (!ok) r = {0, 0, 0, 0};
        if (mine) *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (t * a.q_heads + h) * D + lane * 8) = r;
        continue;
      }
      float most = 0.f;
      bool nan = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        most = fmaxf(most, fabsf(v[j]));
        nan |= v[j] != v[j];
      }
      most = nan ? __int_as_float(0x7FC00000) : most;
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) {
        const float x = __shfl_xor_sync(kFullWarp, most, o);
        most = most != most || x != x ? __int_as_float(0x7FC00000) : fmaxf(most, x);
      }
      // (a row with a NaN: so are all of its values, by their scale)
      const float scale = most != most ? most : fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(__fdiv_rn(most, 6.f))), kScaleLeast), kScaleMost);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __fdiv_rn(v[j], scale);         // (divided, not by way of an inverse: a tie stays one)
      if (!mine || !ok) continue;
      const bool values = h >= a.q_heads + a.kv_heads;
      const int head = h - a.q_heads - (values ? a.kv_heads : 0);
      const size_t place = (((size_t)(slot >> a.shift) * a.kv_heads + head) << a.shift) + (slot & (page - 1));
      *reinterpret_cast<uint32_t*>((values ? a.v_cache : a.k_cache) + place * (D / 2) + lane * 4) = to_e2m1(v);
      if (lane == 0) (values ? a.v_scale : a.k_scale)[place] = (uint16_t)(__float_as_uint(scale) >> 16);
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

constexpr int kUnpackThreads = 256;

template <typename T>
__device__ __forceinline__ void put8(T* to, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = {Half<T>::narrow(v[0], v[1]), Half<T>::narrow(v[2], v[3]), Half<T>::narrow(v[4], v[5]), Half<T>::narrow(v[6], v[7])};
}
template <>
__device__ __forceinline__ void put8<float>(float* to, const float (&v)[8]) {
  *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// A thread block per page and head: its rows of keys, turned back (H H = D), and of values.  Bound by what it writes.
template <typename T, int D>
__global__ void __launch_bounds__(kUnpackThreads) unpack4_kernel(const UnpackArgs a) {
  constexpr int kLanes = D / 8, kRows = kUnpackThreads / kLanes;
  pdl_enter();
  const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes, page = 1 << a.shift;
  const int i = blockIdx.x / a.kv_heads, head = blockIdx.x - i * a.kv_heads, id = a.ids[i];
  const bool real = id >= 0 && id < a.pages;
  const size_t from = ((size_t)(real ? id : 0) * a.kv_heads + head) << a.shift, to = (size_t)blockIdx.x << a.shift;
#pragma unroll 4
  for (int x = row; x < 2 * page; x += kRows) {            // (a multiple of kRows)
    const bool values = x >= page;
    const int place = x & (page - 1);
    const uint32_t w = *reinterpret_cast<const uint32_t*>((values ? a.v_cache : a.k_cache) + (from + place) * (D / 2) + lane * 4);
    const float scale = of_bf16((values ? a.v_scale : a.k_scale)[from + place]);
    uint32_t two[4];
    from_e2m1(w, two);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = Half<__half>::wide(two[j]);
      v[2 * j] = f.x * scale;
      v[2 * j + 1] = f.y * scale;
    }
    if (!values) {                                         // (the same for a whole warp)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= 8.f / D;
      hadamard<D>(v, lane);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = real ? v[j] : 0.f;
    put8<T>(static_cast<T*>(values ? a.v_out : a.k_out) + (to + place) * D + lane * 8, v);
  }
}

// ---- attention over the cache, few rows a request ---------------------------------------------------------------------------------
//
// As over the 8-bit cache (paged_kernels.cu): rows are query heads times tokens, the cache is the 16-row operand of m16n8k16, a warp takes tiles of the
// cache for itself, work is cut evenly and joined.  What differs:
//  * a tile has 32 tokens, in two halves that may lie in different pages;
//  * a byte is two neighbouring dimensions of a token, which is what a register of the keys' fragment holds; for values it has to be two neighbouring
//    tokens of one dimension: two bitwise selections make such bytes of the words of two tokens;
//  * scales belong to tokens: those of keys multiply the scores, those of values enter the exponent (P' = 2^(s + log2 scale - m)) and the sum takes them out.
// Row i of a half is its token i ^ (i >> 1 & 1): neighbouring lanes then read rows of both parities, which lie in different banks.

constexpr int kTile = 32, kUnit = kAttWarps * kTile, kDepth = 4;
constexpr int kBegin = 2;                                  // what an item costs besides its units
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
  // a tile's tokens from `at` on; `least`: tokens that every row sees; `real`: halves that have a page
  template <typename R, typename F>
  __device__ __forceinline__ void add(const uint8_t* stage, const R& rows, int at, int least, unsigned real, int lane, F read) {
    const int g = lane >> 2, c = lane & 3, pi = g ^ (g >> 1 & 1);
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
        const uint16_t* scales = reinterpret_cast<const uint16_t*>(stage + 2 * kKeys<D>);
        ks[h][u] = of_bf16(scales[row]);
        const float vs = of_bf16(scales[kTile + row]), held = fminf(fmaxf(vs, kScaleLeast), kScaleMost);     // (NaN: kScaleLeast, and the logarithm stays NaN)
        lv[h][u] = __log2f(vs != vs ? vs : held);
        inv[h][u] = __fdividef(kSumUnit, held);
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
    uint32_t v[2][4][D / 64];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = 16 * h + 8 * (x >> 1) + ((2 * c + (x & 1)) ^ (c & 1));
        if constexpr (D == 128) {
          const uint2 w = *reinterpret_cast<const uint2*>(stage + kKeys<D> + row * 64 + 8 * g);
          v[h][x][0] = w.x; v[h][x][1] = w.y;
        } else {
          v[h][x][0] = *reinterpret_cast<const uint32_t*>(stage + kKeys<D> + row * 32 + 4 * g);
        }
      }
    read();                                                // nothing of the stage is needed any more
    const bool edge = at + kTile > least || real != 3;
    bool grows = false;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {                      // token pi + 8 (i / 2) of the half, row 2 c + i % 2
          const float x = fmaf(s[h][t][i], rows.scale[t][i & 1] * ks[h][i >> 1], lv[h][i >> 1]);
          s[h][t][i] = edge && (!(real >> h & 1) || at + 16 * h + pi + 8 * (i >> 1) >= rows.end[t][i & 1]) ? kNone : x;
          grows |= s[h][t][i] > m[t][i & 1] + 15.5f;
        }
    if (__any_sync(kFullWarp, grows)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) this->raise(t, y, fmaxf(fmaxf(s[0][t][y], s[0][t][2 + y]), fmaxf(s[1][t][y], s[1][t][2 + y])));
    }
    uint32_t p[2][NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = exp2_fast(s[h][t][i] - (m[t][i & 1] == kNone ? 0.f : m[t][i & 1]));
          l[t][i & 1] = fmaf(e[i], inv[h][i >> 1], l[t][i & 1]);
        }
        p[h][t][0] = transposed(pack_half(e[0], e[1]));
        p[h][t][1] = transposed(pack_half(e[2], e[3]));
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {
        // bytes of two tokens' codes of one dimension: even ones, odd ones
        constexpr uint32_t kLow = 0x0F0F0F0Fu;
        const auto even = [&](int x) { return (v[h][x][w] & kLow) | ((v[h][x + 1][w] << 4) & ~kLow); };
        const auto odd = [&](int x) { return ((v[h][x][w] >> 4) & kLow) | (v[h][x + 1][w] & ~kLow); };
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
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, (kAttBlocks<D, NT>)) paged4_attention_kernel(const AttentionArgs a) {
  constexpr int kRows = 8 * NT, kRing = kDepth * kStage<D>;
  static_assert(kRing >= kRows * (D + 4) * 4, "a warp's results lie where its tiles were");
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ unsigned long long s_full[kAttWarps][kDepth];
  __shared__ int s_fail;
  __shared__ WarpParts<kRows> parts;
  __shared__ Place place;
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    a.cuts[blockIdx.x] = {0, 0, 0, 0};
    s_fail = 0;
    for (int i = 0; i < kAttWarps * kDepth; ++i) bar_init(smem_u32(&s_full[0][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const Begin<Work> begin(a, kRows, &place);
  if (begin.left <= 0) return;
  const long long share = begin.share;
  int r = begin.r;
  long long skip = begin.skip, left = begin.left;
  bool bad = false, ok = true;
  int put = 0, get = 0, ahead = 0;                         // stages of this warp's ring, and how many tiles are on their way
  uint32_t phase = 0;
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
    if (segment) {                                         // the results of the last tile have been read
      __syncthreads();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    // ---- the tiles of this warp: kDepth are on their way.  Lane i holds the page of half i of 16 tiles, and of the 16 after them, which are fetched in time.
    const int* table = a.tables + r * a.table_stride;
    const int stop = min(u1 * kUnit, end), first_at = u0 * kUnit + warp * kTile;
    const int tiles = first_at < stop && ok ? (stop - first_at + kUnit - 1) / kUnit : 0;
    int some, then;
    const auto ids_of = [&](int tile) {                    // -1: no page, or none of this warp's tokens
      const int token = first_at + (tile + (lane >> 1)) * kUnit + 16 * (lane & 1);
      if (token >= stop) return -1;
      const int id = table[token >> a.shift];
      const bool real = id >= 0 && id < a.pages;           // no such page: its tokens are not seen
      bad |= !real;
      return real ? id : -1;
    };
    const auto request = [&](int tile, int ids, int first, bool held) {        // by all lanes, of a stage that they have read; ids: of the tiles from `first` on
      const int half = lane >> 2 & 1, kind = lane & 3, id = __shfl_sync(kFullWarp, ids, 2 * (tile - first) + half);
      const unsigned real = __ballot_sync(kFullWarp, id >= 0);
      const int halves = (real & 1) + (real >> 4 & 1);
      if (!held) {
        const uint32_t bar = smem_u32(&s_full[warp][put]), to = smem_u32(ring + warp * kRing + put * kStage<D>);
        if (lane == 0) {
          if (halves) bar_expect(bar, halves * (16 * D + 64));
          else bar_arrive(bar);
        }
        __syncwarp();
        if (lane < 8 && id >= 0) {                         // keys, values and their scales of both halves
          const size_t at = (((size_t)id * a.kv_heads + kvh) << a.shift) + ((first_at + tile * kUnit + 16 * half) & ((1 << a.shift) - 1));
          if (kind < 2) bulk_load(to + kind * kKeys<D> + half * 8 * D, (kind ? a.v_cache : a.k_cache) + at * (D / 2), 8 * D, bar);
          else bulk_load(to + 2 * kKeys<D> + (kind - 2) * 2 * kTile + half * 32, reinterpret_cast<const uint16_t*>(kind == 2 ? a.k_scale : a.v_scale) + at, 32, bar);
        }
      }
      if (++put == kDepth) put = 0;
      ++ahead;
    };
    some = then = ids_of(0);
    for (int i = 0; i < min(kDepth, tiles); ++i) request(i, some, 0, i == 0 && segment == 0 && warp == 0 && a.withhold == (int)blockIdx.x + 1);
    Rows<T, D, NT, D / 4> q;
    q.load(a, x.start, x.n, x.seen, row0, kvh, lane);
    Running<D, NT> run;
    run.clear();
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      const int j = i & 15;
      if (j == 0 && i) some = then;
      if (j == 0 && i + 16 < tiles) then = ids_of(i + 16);
      ok = __all_sync(kFullWarp, bar_wait(smem_u32(&s_full[warp][get]), phase, &s_fail, kWarpSpinLimit));
      if (!ok) break;
      const unsigned real = __ballot_sync(kFullWarp, some >= 0) >> (2 * j) & 3;
      const int at = first_at + i * kUnit;
      run.add(ring + warp * kRing + get * kStage<D>, q, at, least, real, lane, [&] {
        __syncwarp();
        --ahead;
        if (++get == kDepth) {
          get = 0;
          phase ^= 1;
        }
        if (i + kDepth < tiles) request(i + kDepth, j + kDepth < 16 ? some : then, i - j + (j + kDepth < 16 ? 0 : 16), false);
      });
    }
    const bool whole = u0 == 0 && u1 == x.units;
    finish<T, D, NT, kRing>(a, run, ring, &parts, &s_fail, x, kvh, row0, rows, whole, segment != 0);
    if (!whole && u0 == 0 && tid == 0) {                   // it begins here and ends elsewhere: request, item, parts, place of the first
      const long long beyond = x.units - u1;
      a.cuts[blockIdx.x] = {r, item, 1 + (int)((beyond + share - 1) / share), segment != 0};
    }
  }
  if (!ok) {                                               // a wait ran out: what is on its way arrives before the memory goes back
    for (; ahead > 0; --ahead) {
      bar_wait(smem_u32(&s_full[warp][get]), phase, nullptr, kDrainLimit);
      if (++get == kDepth) {
        get = 0;
        phase ^= 1;
      }
    }
    if (a.status && lane == 0) atomicOr(a.status, 64);
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

template <typename T, int D>
int append_of(const AppendArgs& a, bool halves, cudaStream_t st) {
  const int heads = a.q_heads + 2 * a.kv_heads, windows = (a.tokens + a.window - 1) / a.window;
  const dim3 block(kAppendThreads);
  // few rows: a thread block for each head
  if ((int64_t)windows * heads <= 4 * (int64_t)current_device_sms())
    return halves ? paged_launch(rope_append4_kernel<T, D, 1, true>, dim3(windows, heads), block, 1, 0, st, a)
                  : paged_launch(rope_append4_kernel<T, D, 1, false>, dim3(windows, heads), block, 1, 0, st, a);
  return halves ? paged_launch(rope_append4_kernel<T, D, 4, true>, dim3(windows, (heads + 3) / 4), block, 1, 0, st, a)
                : paged_launch(rope_append4_kernel<T, D, 4, false>, dim3(windows, (heads + 3) / 4), block, 1, 0, st, a);
}

template <typename T>
int unpack_of(const UnpackArgs& a, int head_dim, int units, cudaStream_t st) {
  return head_dim == 128 ? paged_launch(unpack4_kernel<T, 128>, dim3(units), dim3(kUnpackThreads), 1, 0, st, a)
                         : paged_launch(unpack4_kernel<T, 64>, dim3(units), dim3(kUnpackThreads), 1, 0, st, a);
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
  // tokens of a thread block: those that its rows hold at a time, and more where there are thread blocks enough
  const int heads = q_heads + 2 * kv_heads, rows = kAppendThreads / (head_dim / 8);
  int window = rows;
  while (window < kMaxWindow && (int64_t)tokens * heads > (int64_t)window * current_device_sms() * 64) window *= 2;
  const AppendArgs a = {qkv, row_stride, positions, slots, tokens, cosv, sinv, angle_rows, rotary_dim / 2, q_heads, kv_heads, static_cast<uint8_t*>(k_cache),
                        static_cast<uint8_t*>(v_cache), static_cast<uint16_t*>(k_scale), static_cast<uint16_t*>(v_scale), (int64_t)pages << shift, shift, window,
                        q_out, status};
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
