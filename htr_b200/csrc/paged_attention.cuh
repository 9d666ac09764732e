// What the attention kernels over the paged caches share: the cut of the work into even runs over the thread blocks, queries as an operand of warp-level
// matrix instructions, and the join of the parts of what was cut.  The reasons stand in paged_kernels.cu.
#pragma once
#include "paged_common.cuh"

namespace htr {

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // an 8x8 matrix of fp16, a row per four lanes
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
constexpr int kAttWarps = 4, kAttThreads = kAttWarps * 32;

// a row of queries as the right operand: fragments of rows g + 8 * tile, their scale (times that of the scores), for this lane's rows 2 c, 2 c + 1
// kAcross: dimensions of a row of keys that a lane has one after the other
template <typename T, int D, int NT, int kAcross>
struct Rows {
  uint32_t q[D / 16][NT][2];
  float scale[NT][2];
  int end[NT][2];                                          // tokens that a row sees
  __device__ __forceinline__ void load(const AttentionArgs& a, int start, int n, int seen, int row0, int kvh, int lane) {
    const int g = lane >> 2, c = lane & 3, rows = n * a.group;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = row0 + 8 * t + g, i = row / a.group;
      const bool ok = row < rows;
      const T* src = static_cast<const T*>(a.q) + ((size_t)(start + i) * a.q_heads + (size_t)kvh * a.group + (row - i * a.group)) * D;
      float v[D / 16][4], most = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {                   // step k: its 4 (k % (kAcross / 4)) ... of those that begin at 4 kAcross (4 k / kAcross) + kAcross c
        uint2 raw = {0, 0};
        if (ok) raw = *reinterpret_cast<const uint2*>(src + 4 * kAcross * (4 * k / kAcross) + kAcross * c + 4 * k % kAcross);
        const float2 lo = Half<T>::wide(raw.x), hi = Half<T>::wide(raw.y);
        v[k][0] = lo.x; v[k][1] = lo.y; v[k][2] = hi.x; v[k][3] = hi.y;
#pragma unroll
        for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(v[k][j]));
      }
      most = fmaxf(most, __shfl_xor_sync(kFullWarp, most, 1));
      most = fmaxf(most, __shfl_xor_sync(kFullWarp, most, 2));
      const int e = query_exponent(most, 14);
      const float up = exp2i(e);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][t][0] = pack_half(v[k][0] * up, v[k][1] * up);
        q[k][t][1] = pack_half(v[k][2] * up, v[k][3] * up);
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {                        // of the rows in which this lane holds scores
        const int mine = 2 * c + y;
        scale[t][y] = exp2i(-__shfl_sync(kFullWarp, e, 4 * mine)) * a.scale;
        const int at = row0 + 8 * t + mine;
        end[t][y] = at < rows ? seen - n + at / a.group + 1 : 0;
      }
    }
  }
};

// units of kUnit tokens of a request, and kBegin for what an item costs besides: every row tile and key/value head has as many as its tokens fill, at least one (which writes the zeros)
template <int kUnit, int kBegin>
struct Span {
  int start, n, seen, rows, units;
  long long total;
  Span() = default;
  __device__ __forceinline__ Span(const AttentionArgs& a, int r, int tile_rows) {
    start = max(a.starts[r], 0);
    n = max(min(a.starts[r + 1], a.tokens) - start, 0);
    seen = min(max(a.seen[r], 0), a.width << a.shift);
    rows = min(n, a.max_new) * a.group;
    units = max((seen + kUnit - 1) / kUnit, 1);
    total = (long long)((rows + tile_rows - 1) / tile_rows) * (units + kBegin) * a.kv_heads;
  }
};

struct Place {                                             // of a thread block's run, in shared memory
  long long sum[kAttWarps], at;
  int r;
};
// where a thread block's run begins (unit `skip` of request r), and how long it and those of the others are; by all threads, which are in step after it
template <typename W>
struct Begin {
  int r = 0;
  long long share, skip = 0, left;
  __device__ __forceinline__ Begin(const AttentionArgs& a, int tile_rows, Place* place) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int each = (a.requests + kAttThreads - 1) / kAttThreads, first = min(tid * each, a.requests), last = min(first + each, a.requests);
    long long mine = 0;
    for (int i = first; i < last; ++i) mine += W(a, i, tile_rows).total;
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(kFullWarp, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) place->sum[warp] = sum;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) {
      if (w < warp) sum += place->sum[w];
      total += place->sum[w];
    }
    share = max((total + gridDim.x - 1) / gridDim.x, 1LL);
    const long long from = blockIdx.x * share;
    left = min(from + share, total) - from;
    if (left <= 0) return;
    sum -= mine;
    if (sum <= from && from < sum + mine) {
      int i = first;
      for (;; ++i) {
        const long long x = W(a, i, tile_rows).total;
        if (from < sum + x) break;
        sum += x;
      }
      place->r = i;
      place->at = from - sum;
    }
    __syncthreads();
    r = place->r;
    skip = place->at;
  }
};

// running softmax of a warp: results O^T (dimension D/8 g + 2 j + i / 2, rows 2 c + i % 2), maximum and sum of this lane's rows
template <int D, int NT>
struct Results {
  float o[D / 16][NT][4], m[NT][2], l[NT][2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[j][t][0] = o[j][t][1] = o[j][t][2] = o[j][t][3] = 0.f;
      m[t][0] = m[t][1] = kNone;
      l[t][0] = l[t][1] = 0.f;
    }
  }
  // a new reference of row 2 c + y, 2^12 under `most` of all lanes, which is larger than the old one allows; what there is follows
  __device__ __forceinline__ void raise(int t, int y, float most) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(kFullWarp, most, d));
    const float now = fmaxf(m[t][y], most - 12.f);
    const float keep = now == kNone ? 1.f : exp2_fast(m[t][y] - now);
    m[t][y] = now;
    l[t][y] *= keep;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      o[j][t][y] *= keep;
      o[j][t][2 + y] *= keep;
    }
  }
};

template <int kRows>
struct WarpParts {
  float m[kAttWarps][kRows], l[kAttWarps][kRows];
};
// The warps' results joined, by all threads: a tile that was not cut (`whole`) is finished; of one that was, the part goes to the workspace, to the second
// place of the thread block where it is not the run's first (`tail`).  A warp's results pass through the kRing bytes of its ring.
template <typename T, int D, int NT, int kRing, typename W>
__device__ __forceinline__ void finish(const AttentionArgs& a, const Results<D, NT>& run, uint8_t* ring, WarpParts<8 * NT>* parts, int* s_fail, const W& x, int kvh,
                                       int row0, int rows, bool whole, bool tail) {
  constexpr int kRows = 8 * NT, kPart = kRows * (D + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const auto results = [&](int w, int row) { return reinterpret_cast<float*>(ring + w * kRing) + row * (D + 4); };
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float l = run.l[t][y];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(kFullWarp, l, o);
      const int row = 8 * t + 2 * c + y;
      if (g == 0) {
        parts->m[warp][row] = run.m[t][y];
        parts->l[warp][row] = l;
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
        *reinterpret_cast<float2*>(results(warp, row) + D / 8 * g + 2 * j) = make_float2(run.o[j][t][y], run.o[j][t][2 + y]);
    }
  __syncthreads();
  const bool lost = *(volatile int*)s_fail != 0;        // a wait ran out: this tile and those behind it in this run become NaN, by way of the sum
  float* part = a.parts + ((size_t)blockIdx.x * 2 + tail) * kPart;
  for (int z = tid; z < kRows * (D / 4); z += kAttThreads) {
    const int row = z / (D / 4), d = z % (D / 4) * 4;
    if (row >= rows) continue;
    float most = kNone;
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) most = fmaxf(most, parts->m[w][row]);
    float l = 0.f;
    float4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) {
      const float f = most == kNone ? 1.f : exp2_fast(parts->m[w][row] - most);
      const float4 v = *reinterpret_cast<const float4*>(results(w, row) + d);
      l = fmaf(f, parts->l[w][row], l);
      y.x = fmaf(f, v.x, y.x); y.y = fmaf(f, v.y, y.y); y.z = fmaf(f, v.z, y.z); y.w = fmaf(f, v.w, y.w);
    }
    if (lost) l = __int_as_float(0x7FC00000);
    if (whole) {
      const float by = l == 0.f ? 0.f : kSumUnit / l;    // a row that sees nothing: zeros
      const int i = (row0 + row) / a.group, h = row0 + row - i * a.group;
      T* dst = static_cast<T*>(a.out) + ((size_t)(x.start + i) * a.q_heads + (size_t)kvh * a.group + h) * D + d;
      *reinterpret_cast<uint2*>(dst) = {Half<T>::narrow(y.x * by, y.y * by), Half<T>::narrow(y.z * by, y.w * by)};
    } else {
      *reinterpret_cast<float4*>(part + row * D + d) = y;
      if (d == 0) {
        part[kRows * D + row] = most;
        part[kRows * D + kRows + row] = l;
      }
    }
  }
}

// Joins the parts of the tiles that were cut: kJoins thread blocks per run of the launch before, a thread per row and four dimensions, eight parts on their way.
template <int D, int NT>
constexpr int kJoins = 8 * NT * (D / 4) / kAttThreads;
template <typename T, int D, int NT, typename W>
__global__ void __launch_bounds__(kAttThreads) paged_attention_join_kernel(const AttentionArgs a) {
  constexpr int kRows = 8 * NT, kPart = kRows * (D + 2);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (not before the wait: thread blocks of a next step's attention that found a place while this one's still ran cost it 35 us of 128)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.z == 0) return;
  const W x(a, cut.x, kRows);
  const int kvh = cut.y % a.kv_heads, row0 = cut.y / a.kv_heads * kRows, rows = min(x.rows - row0, kRows);
  const float *head = a.parts + ((size_t)blockIdx.x * 2 + cut.w) * kPart, *tail = a.parts + (size_t)blockIdx.x * 2 * kPart;
  for (int z = blockIdx.y * kAttThreads + threadIdx.x; z < rows * (D / 4); z += kJoins<D, NT> * kAttThreads) {
    const int row = z / (D / 4), d = z % (D / 4) * 4;
    float m = head[kRows * D + row], l = head[kRows * D + kRows + row];
    float4 y = *reinterpret_cast<const float4*>(head + row * D + d);
    const auto part = [&](int i) { return tail + (size_t)i * 2 * kPart; };
    join_parts<8>(cut.z, m, l, y, [&](int i) { return part(i) + kRows * D + row; }, [&](int i) { return part(i) + kRows * D + kRows + row; },
               [&](int i) { return reinterpret_cast<const float4*>(part(i) + row * D + d); });
    const float by = l == 0.f ? 0.f : kSumUnit / l;
    const int i = (row0 + row) / a.group, h = row0 + row - i * a.group;
    T* dst = static_cast<T*>(a.out) + ((size_t)(x.start + i) * a.q_heads + (size_t)kvh * a.group + h) * D + d;
    *reinterpret_cast<uint2*>(dst) = {Half<T>::narrow(y.x * by, y.y * by), Half<T>::narrow(y.z * by, y.w * by)};
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// log2 of a page size that the kernels take, else -1
inline int page_shift(int page_size) {
  for (int s = 4; s <= 7; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

}  // namespace htr
