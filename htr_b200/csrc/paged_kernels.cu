// Serving many sequences from a paged 8-bit cache: the plan of a step (page tables, positions, slots), the cache's writing side
// (rotary embedding, e4m3 with one power-of-two scale per page and key/value head), and attention over the cache.
//
// Layout of a layer's cache: keys and values [pages][kv_heads][page_size][head_dim] e4m3, scales [pages][kv_heads] float32.  A page
// of one head is contiguous (page_size * head_dim bytes), which is what one thread block of the attention reads at a time.
//
// Why e4m3 under powers of two: a page fills token by token, and a later token may be larger than what its scale admits.  The scale
// then grows and the older tokens are rescaled by a power of two, which keeps their three mantissa bits (only values that fall among
// the subnormals, 2^-15 of the page's largest and less, are rounded again); 8-bit integers would be rounded anew every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/htr_b200.h"
#include "htr_common.cuh"

namespace {

constexpr int kScaleFloor = -100;                          // smallest exponent of a scale: products of two scales stay normal floats

__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

thread_local int t_last_cuda = 0;

template <typename Kern, typename... Args>
int launch(Kern kern, dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t st, Args... args) {
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
  if (e) {
    t_last_cuda = e;
    (void)cudaGetLastError();                              // a refused launch leaves no error behind for the caller's next check
    return HTR_ERR_CUDA;
  }
  return HTR_OK;
}

// ---- the plan of a step -----------------------------------------------------------------------------------------------------------
//
// What bounds it: nothing but latency (a few KB for a decode step), so it is one launch.  Every thread block scans all requests by
// itself (at most 8192 of them, in shared memory) and then fills its share of the tokens by binary search: 20 times the additions of a
// scan across thread blocks, and no waiting for one another.  The outputs may be the inputs' own buffers (lengths, count): the thread
// blocks are one cluster, and nothing is written over before all of them have read.
constexpr int kPlanThreads = 512, kPlanMaxRequests = 8192, kPlanMaxCluster = 8;

struct PlanArgs {
  const int *lengths, *added;
  int requests;
  int* tables;
  long long table_stride;
  int width;
  int* free_pages;
  int pages;
  const int* count;
  int shift, max_tokens;
  int *starts, *positions, *slots, *seen, *lengths_out, *count_out, *status;
};

// inclusive scan of a pair over the block; totals come back in `total`
__device__ __forceinline__ longlong2 block_scan(longlong2 v, longlong2* part, longlong2* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(htr::kFullWarp, v.x, o), y = __shfl_up_sync(htr::kFullWarp, v.y, o);
    if (lane >= o) {
      v.x += x;
      v.y += y;
    }
  }
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  longlong2 sum = {0, 0};
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w == warp) {
      v.x += sum.x;
      v.y += sum.y;
    }
    sum.x += part[w].x;
    sum.y += part[w].y;
  }
  *total = sum;
  return v;
}

// first index of the nondecreasing list a[0..n) whose value is above x; n where there is none
__device__ __forceinline__ int above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanArgs a) {
  extern __shared__ int plan_smem[];
  int *ends = plan_smem, *need_end = ends + a.requests, *back_end = need_end + a.requests, *held = back_end + a.requests;
  __shared__ longlong2 part[kPlanThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, R = a.requests, page = 1 << a.shift;
  const int blocks = gridDim.x, block = blockIdx.x;
  const long long capacity = (long long)a.width << a.shift;
  const int count = min(max(*a.count, 0), a.pages);
  const int each = (R + kPlanThreads - 1) / kPlanThreads, first = min(tid * each, R), last = min(first + each, R);
  int bad = 0;
  // ---- tokens before every request, and pages that those which are over give back
  longlong2 mine = {0, 0}, total, run;
  for (int r = first; r < last; ++r) {
    const int len = a.lengths[r], add = a.added[r];
    if (len < 0 || len > capacity) bad |= 4;
    const int pages = len < 0 || len > capacity ? 0 : (int)(((long long)len + page - 1) >> a.shift);
    mine.x += max(add, 0);
    mine.y += add < 0 ? pages : 0;
  }
  run = block_scan(mine, part, &total);
  const int tokens = (int)min(total.x, (long long)a.max_tokens), back = (int)min(total.y, (long long)a.pages);
  if (total.x > a.max_tokens) bad |= 8;
  run.x -= mine.x;
  run.y -= mine.y;
  mine = {0, 0};
  for (int r = first; r < last; ++r) {
    const int len = a.lengths[r], add = a.added[r];
    const bool valid = len >= 0 && len <= capacity;
    const int pages = valid ? (int)(((long long)len + page - 1) >> a.shift) : 0;
    run.x += max(add, 0);
    run.y += add < 0 ? pages : 0;
    ends[r] = (int)min(run.x, (long long)a.max_tokens);
    back_end[r] = (int)min(run.y, (long long)a.pages);
    int need = -1;                                           // not served
    if (add > 0 && valid && run.x <= a.max_tokens) {
      const long long now = (long long)len + add;
      if (now <= capacity) need = (int)((now + page - 1) >> a.shift) - pages;
      else bad |= 2;
    }
    held[r] = need < 0 ? -1 : len;
    need_end[r] = need;
    mine.x += max(need, 0);
  }
  run = block_scan(mine, part, &total);
  run.x -= mine.x;
  const long long supply = (long long)count + back;
  longlong2 granted = {0, 0};
  for (int r = first; r < last; ++r) {
    const int need = need_end[r];
    run.x += max(need, 0);
    need_end[r] = (int)min(run.x, (long long)0x7FFFFFFF);
    if (need > 0 && run.x > supply) {
      held[r] = -1;
      bad |= 1;
    } else if (need > 0) {
      granted.x += need;
    }
  }
  block_scan(granted, part, &total);
  const int taken = (int)total.x;
  if (bad && a.status && block == 0) atomicOr(a.status, bad);
  __syncthreads();
  // page i of what this step takes: first those that came back, then the top of the free pages
  const auto returned = [&](int i) {
    const int r = above(back_end, R, i);
    return r < R ? a.tables[r * a.table_stride + i - (r ? back_end[r - 1] : 0)] : -1;
  };
  const auto supplied = [&](int i) {
    if (i < back) return returned(i);
    const int at = count - 1 - (i - back);
    return at >= 0 ? a.free_pages[at] : -1;
  };
  const int stride = blocks * kPlanThreads, me = block * kPlanThreads + tid;
  for (int t = me; t < a.max_tokens; t += stride) {
    int pos = -1, slot = -1;
    if (t < tokens) {
      const int r = above(ends, R, t);
      if (r < R && held[r] >= 0) {
        pos = held[r] + t - (r ? ends[r - 1] : 0);
        const int at = pos >> a.shift, have = (int)(((long long)held[r] + page - 1) >> a.shift);
        const int id = at < have ? a.tables[r * a.table_stride + at] : supplied((r ? need_end[r - 1] : 0) + at - have);
        slot = id >= 0 && id < a.pages ? (id << a.shift) + (pos & (page - 1)) : -1;
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  for (int i = me; i < taken; i += stride) {                 // the new pages enter the tables
    const int r = above(need_end, R, i);
    if (r >= R || held[r] < 0) continue;
    const int have = (int)(((long long)held[r] + page - 1) >> a.shift);
    a.tables[r * a.table_stride + have + i - (r ? need_end[r - 1] : 0)] = supplied(i);
  }
  for (int i = me; i < back - taken; i += stride)            // what came back and was not taken lies on top of the free pages
    if (count + i < a.pages) a.free_pages[count + i] = returned(taken + i);
  if (blocks > 1) htr::cluster_sync();
  else __syncthreads();
  for (int r = me; r < R; r += stride) {
    const int len = a.lengths[r], add = a.added[r];
    const bool served = held[r] >= 0;
    a.starts[r + 1] = ends[r];
    a.seen[r] = served ? len + add : 0;
    a.lengths_out[r] = add < 0 ? 0 : served ? len + add : len;
  }
  if (me == 0) {
    a.starts[0] = 0;
    *a.count_out = min(count + back - taken, a.pages);
  }
}

// ---- the cache's writing side -----------------------------------------------------------------------------------------------------

template <typename T> struct Half;
template <> struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ float2 wide(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
  static __device__ __forceinline__ uint32_t narrow(float x, float y) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <> struct Half<__half> {
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
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

// the exponent of the smallest power of two under which `most` (finite, not negative) lies within e4m3
__device__ __forceinline__ int scale_exponent(float most) {
  if (most == 0.f) return kScaleFloor;
  int e;
  const float m = frexpf(most, &e);
  return max(m <= 0.875f ? e - 9 : e - 8, kScaleFloor);
}

struct AppendArgs {
  const void* qkv;
  long long row_stride;                                    // elements
  const int *positions, *slots;
  int tokens;
  const float *cosv, *sinv;
  int angle_rows, q_heads, kv_heads;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  long long slots_total;
  int shift, window;
  void* q_out;
  int* status;
};

// A thread holds 8 consecutive dimensions of a row, four pairs of the rotation.
template <typename T, int D>
struct Row {
  static constexpr int kLanes = D / 8;
  static __device__ __forceinline__ void load(const T* row, int lane, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(row + lane * 8);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Half<T>::wide(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void rotate(float (&v)[8], const float4 c, const float4 s) {
    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = v[2 * i], y = v[2 * i + 1];
      v[2 * i] = x * cs[i] - y * sn[i];
      v[2 * i + 1] = x * sn[i] + y * cs[i];
    }
  }
};

constexpr int kAppendThreads = 128;

// grid (windows of tokens, 2 * kv_heads + 1): y < 2 * kv_heads: the keys (even) or values (odd) of one head; the last: the queries.
// A run = the tokens of this step that lie in one page; the block of the window in which a run begins writes it whole, so that one
// block alone reads and writes the page's scale.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) rope_append_kernel(const AppendArgs a) {
  using R = Row<T, D>;
  constexpr int kRows = kAppendThreads / R::kLanes;        // rows of a pass
  __shared__ float red[kAppendThreads / 32];
  __shared__ int s_run;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid % R::kLanes, row = tid / R::kLanes, page = 1 << a.shift;
  const T* qkv = static_cast<const T*>(a.qkv);
  const auto slot_of = [&](int t) {                        // -1: the token is not written
    const int slot = a.slots[t], pos = a.positions[t];
    return slot >= 0 && slot < a.slots_total && pos >= 0 && pos < a.angle_rows ? slot : -1;
  };
  const int t0 = blockIdx.x * a.window, t1 = min(t0 + a.window, a.tokens);
  if (blockIdx.y == 2 * a.kv_heads) {                      // queries: the angles of a row serve all of its heads
    for (int t = t0 + row; t < t1; t += kRows) {
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (size_t)t * a.q_heads * D + lane * 8);
      const T* in = qkv + (size_t)t * a.row_stride;
      const bool ok = slot_of(t) >= 0;
      if (!ok && a.status && lane == 0 && a.slots[t] != -1) atomicOr(a.status, 16);
      const size_t at = ok ? (size_t)a.positions[t] * (D / 2) + lane * 4 : 0;
      const float4 c = ok ? *reinterpret_cast<const float4*>(a.cosv + at) : make_float4(0, 0, 0, 0);
      const float4 s = ok ? *reinterpret_cast<const float4*>(a.sinv + at) : make_float4(0, 0, 0, 0);
      for (int h = 0; h < a.q_heads; ++h) {
        float v[8];
        R::load(in + (size_t)h * D, lane, v);
        R::rotate(v, c, s);
        uint4 r = {Half<T>::narrow(v[0], v[1]), Half<T>::narrow(v[2], v[3]), Half<T>::narrow(v[4], v[5]), Half<T>::narrow(v[6], v[7])};
        if (!ok) r = {0, 0, 0, 0};
        out[(size_t)h * R::kLanes] = r;
      }
    }
    return;
  }
  const int head = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  uint8_t* cache = values ? a.v_cache : a.k_cache;
  float* scales = values ? a.v_scale : a.k_scale;
  const T* in = qkv + (size_t)(a.q_heads + (values ? a.kv_heads : 0) + head) * D;
  for (int t = t0; t < t1; ++t) {
    const int slot = slot_of(t), off = slot & (page - 1);
    if (slot < 0 || (off != 0 && t > 0 && slot_of(t - 1) == slot - 1)) continue;     // (the whole block)
    if (tid == 0) s_run = page - off;
    __syncthreads();
    for (int i = tid; i < page - off; i += kAppendThreads)
      if (t + i >= a.tokens || slot_of(t + i) != slot + i) atomicMin(&s_run, i);
    __syncthreads();
    const int run = s_run;
    const auto fetch = [&](int i, float (&v)[8]) {
      R::load(in + (size_t)(t + i) * a.row_stride, lane, v);
      if (!values) {
        const size_t at = (size_t)a.positions[t + i] * (D / 2) + lane * 4;
        R::rotate(v, *reinterpret_cast<const float4*>(a.cosv + at), *reinterpret_cast<const float4*>(a.sinv + at));
      }
    };
    float most = 0.f;
    for (int i = row; i < run; i += kRows) {
      float v[8];
      fetch(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float m = fabsf(v[j]);
        if (m <= 3.402823466e38f) most = fmaxf(most, m);   // infinities saturate and NaN stays: neither sets the scale
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(htr::kFullWarp, most, o));
    if ((tid & 31) == 0) red[tid >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) most = fmaxf(most, red[w]);
    const size_t unit = (size_t)(slot >> a.shift) * a.kv_heads + head;
    uint8_t* at = cache + (unit << a.shift) * D;
    int e = scale_exponent(most);
    if (off) {                                             // older tokens: their scale never shrinks, and they follow where it grows
      const int old = max((int)((__float_as_uint(scales[unit]) >> 23) & 255) - 127, kScaleFloor);
      if (old >= e) {
        e = old;
      } else {
        const float down = exp2i(max(old - e, -126));
        for (int x = tid; x < off * D / 4; x += kAppendThreads) {
          uint32_t* p = reinterpret_cast<uint32_t*>(at) + x;
          const uint32_t lo = from_e4m3(*p & 0xFFFFu), hi = from_e4m3(*p >> 16);
          const float2 f = Half<__half>::wide(lo), g = Half<__half>::wide(hi);
          *p = to_e4m3(f.x * down, f.y * down) | to_e4m3(g.x * down, g.y * down) << 16;
        }
      }
    }
    const float up = exp2i(-e);
    for (int i = row; i < run; i += kRows) {
      float v[8];
      fetch(i, v);
      const uint2 r = {to_e4m3(v[0] * up, v[1] * up) | to_e4m3(v[2] * up, v[3] * up) << 16,
                       to_e4m3(v[4] * up, v[5] * up) | to_e4m3(v[6] * up, v[7] * up) << 16};
      *reinterpret_cast<uint2*>(at + (size_t)(off + i) * D + lane * 8) = r;
    }
    __syncthreads();                                       // the old scale has been read by all
    if (tid == 0) scales[unit] = exp2i(e);
  }
}

// ---- attention over the cache -----------------------------------------------------------------------------------------------------
//
// The query heads of one key/value head and a request's tokens of this step are rows of one product, 16 at a time (row = token * group
// + head), on warp-level matrix instructions m16n8k16.  A warp takes 16 cached tokens at a time, for itself alone: the dimensions that
// a product sums over and the columns of a result may be taken in any order, so that every lane loads whole 16-byte pieces of the
// cache's rows straight into the fragments of K^T (lane g, c: token g, dimensions 16 c ...) and of V (tokens 2 c, 2 c + 1, ...,
// dimensions 16 g ...), and e4m3 becomes fp16, which holds it exactly, in registers.
// Queries are fp16 under a power of two per row (bf16 keeps all its bits: 29 binades of normal fp16 below the row's largest element).
// Probabilities are rounded to fp16, relative to the contribution that they make: the scale of the values' page is part of the exponent
// (P' = 2^(s + log2 scale - m)), and the sum of the probabilities takes it out again.  2^-12 each, averaged over the tokens: below the
// rounding of the output.  Maxima, sums and results are float32.

struct AttentionArgs {
  const void* q;
  const int *starts, *seen, *tables;
  long long table_stride;
  int width, requests, tokens, q_heads, kv_heads, group;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int pages, shift;
  float scale;                                             // of the scores, times log2(e)
  void* out;
  int* status;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

constexpr int kAttWarps = 4;
constexpr float kNone = -__builtin_huge_valf();

template <typename T, int D>
__global__ void __launch_bounds__(kAttWarps * 32) paged_attention_kernel(const AttentionArgs a) {
  constexpr int kSteps = D / 16, kCols = D / 8;            // k-steps of a score; 8-column tiles of the result = dimensions of a lane
  __shared__ float s_o[kAttWarps][16][D + 1];
  __shared__ float s_m[kAttWarps][16], s_l[kAttWarps][16];
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int r = blockIdx.z, kvh = blockIdx.y;
  const int start = a.starts[r], n = min(a.starts[r + 1], a.tokens) - start, seen = a.seen[r];
  const int row0 = blockIdx.x * 16, rows = n * a.group;
  if (start < 0 || row0 >= rows) return;
  const int last = min(row0 + 15, rows - 1) / a.group;     // of the tile's tokens: it sees the most
  const int end = min(max(seen - n + last + 1, 0), (int)min((long long)a.width << a.shift, 0x7FFFFFFFLL));
  // queries
  uint32_t qf[kSteps][4];
  float row_scale[2];
  int row_end[2];                                          // tokens that a row sees
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = row0 + g + 8 * x, i = row / a.group;
    const bool ok = row < rows;
    row_end[x] = ok ? seen - n + i + 1 : 0;
    const T* src = static_cast<const T*>(a.q) + ((size_t)(start + i) * a.q_heads + (size_t)kvh * a.group + (row - i * a.group)) * D;
    float v[kSteps][4];
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {                     // step k: dimensions 64 (k / 4) + 16 c + 4 (k % 4) ...
      uint2 raw = {0, 0};
      if (ok) raw = *reinterpret_cast<const uint2*>(src + 64 * (k >> 2) + 16 * c + 4 * (k & 3));
      const float2 lo = Half<T>::wide(raw.x), hi = Half<T>::wide(raw.y);
      v[k][0] = lo.x; v[k][1] = lo.y; v[k][2] = hi.x; v[k][3] = hi.y;
#pragma unroll
      for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(v[k][j]));
    }
    most = fmaxf(most, __shfl_xor_sync(htr::kFullWarp, most, 1));
    most = fmaxf(most, __shfl_xor_sync(htr::kFullWarp, most, 2));
    int e = 0;
    if (sizeof(T) == 2 && most > 0.f && most <= 3.402823466e38f) e = min(max(14 - ((int)(__float_as_uint(most) >> 23) - 127), -100), 100);
    const float up = exp2i(e);
    row_scale[x] = exp2i(-e) * a.scale;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      qf[k][x] = pack_half(v[k][0] * up, v[k][1] * up);
      qf[k][2 + x] = pack_half(v[k][2] * up, v[k][3] * up);
    }
  }
  float o[kCols][4];
#pragma unroll
  for (int j = 0; j < kCols; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[2] = {kNone, kNone}, l[2] = {0.f, 0.f};
  const int* table = a.tables + r * a.table_stride;
  bool bad = false;
  for (int at = warp * 16; at < end; at += kAttWarps * 16) {
    const int id = table[at >> a.shift];
    if (id < 0 || id >= a.pages) {                         // no such page: its tokens are not seen
      bad = true;
      continue;
    }
    const size_t unit = (size_t)id * a.kv_heads + kvh;
    const size_t base = ((unit << a.shift) + (at & ((1 << a.shift) - 1))) * D;
    const float ks = a.k_scale[unit], vs = a.v_scale[unit];
    const float lv = log2f(vs), inv = 1.f / vs;
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint4 raw = *reinterpret_cast<const uint4*>(a.k_cache + base + (size_t)(8 * t + g) * D + 64 * i + 16 * c);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_16816(s[t], qf[4 * i + j], from_e4m3(w[j] & 0xFFFFu), from_e4m3(w[j] >> 16));
      }
    }
    float p[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float most = kNone;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float& v = s[t][2 * x + y];
          v = at + 8 * t + 2 * c + y < row_end[x] ? v * (row_scale[x] * ks) + lv : kNone;
          most = fmaxf(most, v);
        }
      most = fmaxf(most, __shfl_xor_sync(htr::kFullWarp, most, 1));
      most = fmaxf(most, __shfl_xor_sync(htr::kFullWarp, most, 2));
      const float now = fmaxf(m[x], most), from = now == kNone ? 0.f : now;
      const float keep = exp2_fast(m[x] - from);
      m[x] = now;
      l[x] *= keep;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        o[j][2 * x] *= keep;
        o[j][2 * x + 1] *= keep;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float e = exp2_fast(s[t][2 * x + y] - from);
          p[t][2 * x + y] = e;
          l[x] += e * inv;
        }
    }
    const uint32_t pf[4] = {pack_half(p[0][0], p[0][1]), pack_half(p[0][2], p[0][3]), pack_half(p[1][0], p[1][1]), pack_half(p[1][2], p[1][3])};
    uint32_t v[4][kCols / 4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int token = 2 * c + (x & 1) + 8 * (x >> 1);
      const uint8_t* src = a.v_cache + base + (size_t)token * D + kCols * g;
      const bool real = at + token < end;                  // behind the request's tokens lies what an earlier one left
      if constexpr (D == 128) {
        const uint4 raw = *reinterpret_cast<const uint4*>(src);
        v[x][0] = raw.x; v[x][1] = raw.y; v[x][2] = raw.z; v[x][3] = raw.w;
      } else {
        const uint2 raw = *reinterpret_cast<const uint2*>(src);
        v[x][0] = raw.x; v[x][1] = raw.y;
      }
#pragma unroll
      for (int j = 0; j < kCols / 4; ++j)
        if (!real) v[x][j] = 0;
    }
#pragma unroll
    for (int j = 0; j < kCols / 4; ++j) {
      const uint32_t a0 = __byte_perm(v[0][j], v[1][j], 0x5140), a1 = __byte_perm(v[0][j], v[1][j], 0x7362);
      const uint32_t b0 = __byte_perm(v[2][j], v[3][j], 0x5140), b1 = __byte_perm(v[2][j], v[3][j], 0x7362);
      mma_16816(o[4 * j], pf, from_e4m3(a0 & 0xFFFFu), from_e4m3(b0 & 0xFFFFu));
      mma_16816(o[4 * j + 1], pf, from_e4m3(a0 >> 16), from_e4m3(b0 >> 16));
      mma_16816(o[4 * j + 2], pf, from_e4m3(a1 & 0xFFFFu), from_e4m3(b1 & 0xFFFFu));
      mma_16816(o[4 * j + 3], pf, from_e4m3(a1 >> 16), from_e4m3(b1 >> 16));
    }
  }
  if (bad && a.status && lane == 0) atomicOr(a.status, 32);
  // ---- the warps' parts
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(htr::kFullWarp, l[x], 1);
    l[x] += __shfl_xor_sync(htr::kFullWarp, l[x], 2);
    if (c == 0) {
      s_m[warp][g + 8 * x] = m[x];
      s_l[warp][g + 8 * x] = l[x];
    }
#pragma unroll
    for (int j = 0; j < kCols; ++j) {                      // column 2 c + y of tile j: dimension kCols (2 c + y) + j
      s_o[warp][g + 8 * x][kCols * (2 * c) + j] = o[j][2 * x];
      s_o[warp][g + 8 * x][kCols * (2 * c + 1) + j] = o[j][2 * x + 1];
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * (D / 2); x += kAttWarps * 32) {
    const int row = x / (D / 2), d = x % (D / 2) * 2;
    if (row0 + row >= rows) continue;
    float most = kNone;
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) most = fmaxf(most, s_m[w][row]);
    const float from = most == kNone ? 0.f : most;
    float sum = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) {
      const float f = exp2_fast(s_m[w][row] - from);
      sum += f * s_l[w][row];
      y0 += f * s_o[w][row][d];
      y1 += f * s_o[w][row][d + 1];
    }
    const float by = sum == 0.f ? 0.f : 1.f / sum;         // a row that sees nothing: zeros
    const int i = (row0 + row) / a.group, h = row0 + row - i * a.group;
    T* dst = static_cast<T*>(a.out) + ((size_t)(start + i) * a.q_heads + (size_t)kvh * a.group + h) * D + d;
    *reinterpret_cast<uint32_t*>(dst) = Half<T>::narrow(y0 * by, y1 * by);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// log2 of a page size that the kernels take, else -1
int page_shift(int page_size) {
  for (int s = 4; s <= 7; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

template <typename T>
int attention_of(const AttentionArgs& a, int head_dim, int max_new, cudaStream_t st) {
  const dim3 grid((unsigned)(((long long)max_new * a.group + 15) / 16), a.kv_heads, a.requests);
  return head_dim == 128 ? launch(paged_attention_kernel<T, 128>, grid, dim3(kAttWarps * 32), 1, 0, st, a)
                         : launch(paged_attention_kernel<T, 64>, grid, dim3(kAttWarps * 32), 1, 0, st, a);
}

template <typename T>
int append_of(const AppendArgs& a, int head_dim, dim3 grid, cudaStream_t st) {
  return head_dim == 128 ? launch(rope_append_kernel<T, 128>, grid, dim3(kAppendThreads), 1, 0, st, a)
                         : launch(rope_append_kernel<T, 64>, grid, dim3(kAppendThreads), 1, 0, st, a);
}

}  // namespace

extern "C" {

int htr_paged_last_cuda_error(void) { return t_last_cuda; }

int htr_page_plan(const int* lengths, const int* added, int requests, int* tables, int64_t table_stride, int table_width, int* free_pages, int pages,
                  const int* count, int page_size, int max_tokens, int* starts, int* positions, int* slots, int* seen, int* lengths_out,
                  int* count_out, int* status, htr_stream_t stream) {
  const int shift = page_shift(page_size);
  if (requests < 1 || table_width < 1 || table_stride < table_width || pages < 1 || shift < 0 || max_tokens < 0) return HTR_ERR_BAD_SHAPE;
  if (requests > kPlanMaxRequests || max_tokens > 1 << 30 || (int64_t)pages << shift > 0x7FFFFFFF || (int64_t)table_width << shift > 0x7FFFFFFF)
    return HTR_ERR_TOO_LARGE;
  if (!lengths || !added || !tables || !free_pages || !count || !starts || (max_tokens && (!positions || !slots)) || !seen || !lengths_out || !count_out)
    return HTR_ERR_NULL;
  const PlanArgs a = {lengths, added, requests, tables, table_stride, table_width, free_pages, pages, count, shift, max_tokens,
                      starts, positions, slots, seen, lengths_out, count_out, status};
  const size_t smem = 4 * sizeof(int) * (size_t)requests;
  if (smem > 40960) {
    const int e = (int)cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * sizeof(int) * kPlanMaxRequests);
    if (e) {
      t_last_cuda = e;
      return HTR_ERR_CUDA;
    }
  }
  const int work = max_tokens > requests ? max_tokens : requests;
  const int blocks = work <= 2 * kPlanThreads ? 1 : kPlanMaxCluster;
  return launch(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), blocks, smem, static_cast<cudaStream_t>(stream), a);
}

int htr_paged_append(const void* qkv, int dtype, int64_t row_stride, const int* positions, const int* slots, int tokens, const float* cosv,
                     const float* sinv, int angle_rows, int q_heads, int kv_heads, int head_dim, void* k_cache, void* v_cache, float* k_scale,
                     float* v_scale, int pages, int page_size, void* q_out, int* status, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16) return HTR_ERR_BAD_DTYPE;
  const int shift = page_shift(page_size);
  if (tokens < 0 || (head_dim != 64 && head_dim != 128) || q_heads < 1 || kv_heads < 1 || pages < 1 || shift < 0 || angle_rows < 1 ||
      row_stride < (int64_t)(q_heads + 2 * (int64_t)kv_heads) * head_dim || row_stride % 8)
    return HTR_ERR_BAD_SHAPE;
  if (q_heads > 16384 || kv_heads > 16384 || tokens > 1 << 30 || (int64_t)pages << shift > 0x7FFFFFFF) return HTR_ERR_TOO_LARGE;
  if (tokens == 0) return HTR_OK;
  if (!qkv || !positions || !slots || !cosv || !sinv || !k_cache || !v_cache || !k_scale || !v_scale || !q_out) return HTR_ERR_NULL;
  if (!aligned16(qkv) || !aligned16(cosv) || !aligned16(sinv) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(q_out)) return HTR_ERR_ALIGNMENT;
  const int units = 2 * kv_heads + 1;
  int window = 1;                                          // tokens of a thread block: few where there is little to share out
  while (window < page_size && (int64_t)tokens * units > (int64_t)window * 148 * 16) window *= 2;
  const AppendArgs a = {qkv, row_stride, positions, slots, tokens, cosv, sinv, angle_rows, q_heads, kv_heads, static_cast<uint8_t*>(k_cache),
                        static_cast<uint8_t*>(v_cache), k_scale, v_scale, (int64_t)pages << shift, shift, window, q_out, status};
  const dim3 grid((unsigned)((tokens + window - 1) / window), units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == HTR_DTYPE_BF16 ? append_of<__nv_bfloat16>(a, head_dim, grid, st) : append_of<__half>(a, head_dim, grid, st);
}

size_t htr_paged_attention_workspace_bytes(int tokens, int requests, int q_heads, int kv_heads, int head_dim, int max_new) { return 0; }

int htr_paged_attention(const void* q, int dtype, int tokens, const int* starts, const int* seen, int requests, const int* tables,
                        int64_t table_stride, int table_width, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                        int pages, int page_size, int q_heads, int kv_heads, int head_dim, int max_new, float scale, void* out, int* status,
                        void* workspace, size_t workspace_bytes, htr_stream_t stream) {
  if (dtype != HTR_DTYPE_BF16 && dtype != HTR_DTYPE_F16) return HTR_ERR_BAD_DTYPE;
  const int shift = page_shift(page_size);
  if (tokens < 0 || requests < 1 || table_width < 1 || table_stride < table_width || (head_dim != 64 && head_dim != 128) || q_heads < 1 || kv_heads < 1 ||
      q_heads % kv_heads || pages < 1 || shift < 0 || max_new < 1)
    return HTR_ERR_BAD_SHAPE;
  if (requests > 8192 || kv_heads > 16384 || q_heads > 16384 || tokens > 1 << 30 || (int64_t)max_new * (q_heads / kv_heads) > 1 << 30 ||
      (int64_t)pages << shift > 0x7FFFFFFF || (int64_t)table_width << shift > 0x7FFFFFFF)
    return HTR_ERR_TOO_LARGE;
  if (tokens == 0) return HTR_OK;
  if (!q || !starts || !seen || !tables || !k_cache || !v_cache || !k_scale || !v_scale || !out) return HTR_ERR_NULL;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return HTR_ERR_ALIGNMENT;
  const AttentionArgs a = {q, starts, seen, tables, table_stride, table_width, requests, tokens, q_heads, kv_heads, q_heads / kv_heads,
                           static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale, pages, shift,
                           scale * 1.4426950408889634f, out, status};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == HTR_DTYPE_BF16 ? attention_of<__nv_bfloat16>(a, head_dim, max_new, st) : attention_of<__half>(a, head_dim, max_new, st);
}

}  // extern "C"
