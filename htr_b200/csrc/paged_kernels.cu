// Serving many sequences from a paged 8-bit cache: the plan of a step (page tables, positions, slots), the cache's writing side
// (rotary embedding, e4m3 with one power-of-two scale per page and key/value head), and attention over the cache.
//
// Layout of a layer's cache: keys and values [pages][kv_heads][page_size][head_dim] e4m3, scales [pages][kv_heads] float32.  A page
// of one head is contiguous (page_size * head_dim bytes), which is what one thread block of the attention reads at a time.
//
// Why e4m3 under powers of two: a page fills token by token, and a later token may be larger than what its scale admits.  The scale
// then grows and the older tokens are rescaled by a power of two, which keeps their three mantissa bits (only values that fall among
// the subnormals, 2^-15 of the page's largest and less, are rounded again); 8-bit integers would be rounded anew every time.
#include "paged_attention.cuh"

namespace {

using namespace htr;

constexpr int kScaleFloor = -100;                          // smallest exponent of a scale, which a page of zeros has: it and its inverse are normal floats

__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

thread_local int t_last_cuda = 0;
thread_local int t_withhold = 0;                           // (htr_paged_attention_withhold)

// ---- the plan of a step -----------------------------------------------------------------------------------------------------------
//
// What bounds it: latency (a few KB for a decode step), so it is one launch: 4.5 us in a chain of launches for 32
// requests of one token, and 13 us, most of it the scans below, for 1024 that add up to 200 each.  Every thread block scans all requests by
// itself (at most 8192 of them, in shared memory) and then fills its share of the tokens by binary search: 20 times the additions of a
// scan across thread blocks, and no waiting for one another.  The outputs may be the inputs' own buffers (lengths, count): the thread
// blocks are one cluster, and nothing is written over before all of them have read.
constexpr int kPlanThreads = 1024, kPlanMaxRequests = 8192, kPlanMaxCluster = 8;

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
  const auto scan = [lane](longlong2 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(htr::kFullWarp, v.x, o), y = __shfl_up_sync(htr::kFullWarp, v.y, o);
      if (lane >= o) {
        v.x += x;
        v.y += y;
      }
    }
    return v;
  };
  v = scan(v);
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  const longlong2 w = lane < kPlanThreads / 32 ? part[lane] : longlong2{0, 0}, e = scan(w);
  v.x += __shfl_sync(htr::kFullWarp, e.x - w.x, warp);
  v.y += __shfl_sync(htr::kFullWarp, e.y - w.y, warp);
  total->x = __shfl_sync(htr::kFullWarp, e.x, 31);
  total->y = __shfl_sync(htr::kFullWarp, e.y, 31);
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
  __shared__ int s_taken[kPlanThreads / 32];
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
  int granted = 0;                                         // the requests that are served and need pages come first of all that need some
  for (int r = first; r < last; ++r) {
    const int need = need_end[r];
    run.x += max(need, 0);
    need_end[r] = (int)min(run.x, (long long)0x7FFFFFFF);
    if (need > 0 && run.x > supply) {
      held[r] = -1;
      bad |= 1;
    } else if (need > 0) {
      granted = (int)run.x;
    }
  }
  granted = __reduce_max_sync(htr::kFullWarp, granted);
  __syncthreads();
  if ((tid & 31) == 0) s_taken[tid >> 5] = granted;
  __syncthreads();
  const int taken = __reduce_max_sync(htr::kFullWarp, s_taken[tid & 31]);
  if (bad && a.status && block == 0) atomicOr(a.status, bad);
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
  // a thread takes four tokens in a row where there are many: they mostly share their request and its page
  const int row = a.max_tokens > stride ? 4 : 1;
  for (int t0 = me * row; t0 < a.max_tokens; t0 += stride * row) {
    int r = above(ends, R, t0), at = -1, id = -1;
    for (int t = t0; t < min(t0 + row, a.max_tokens); ++t) {
      int pos = -1, slot = -1;
      if (t < tokens) {
        while (r < R && ends[r] <= t) {
          ++r;
          at = -1;
        }
        if (r < R && held[r] >= 0) {
          pos = held[r] + t - (r ? ends[r - 1] : 0);
          if (at != pos >> a.shift) {
            at = pos >> a.shift;
            const int have = (int)(((long long)held[r] + page - 1) >> a.shift);
            id = at < have ? a.tables[r * a.table_stride + at] : supplied((r ? need_end[r - 1] : 0) + at - have);
          }
          slot = id >= 0 && id < a.pages ? (id << a.shift) + (pos & (page - 1)) : -1;
        }
      }
      a.positions[t] = pos;
      a.slots[t] = slot;
    }
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
  static __device__ __forceinline__ void widen(const uint4& raw, float (&v)[8]) {
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

constexpr int kAppendThreads = 256, kQueryHeads = 4;

// grid (windows of tokens, 2 * kv_heads + groups of query heads): y < 2 * kv_heads: the keys (even) or values (odd) of one head; then the queries.
// A run = the tokens of this step that lie in one page; the block of the window in which a run begins writes it whole, so that one
// block alone reads and writes the page's scale.  Tokens that are not written do not end a run (the block of the next one would be another): a token
// begins one where the written token before it, up to a page back, is not of its page, and a slot that does not rise closes its page.  A prompt is bound by its bytes: a run stays in registers between the search for
// its largest element and the rounding, and query rows are read four heads at a time, whose angles are the same.  A few tokens are
// bound by latency: slots and positions, then rows, angles and the old scale at once, then the maximum.
// What holds a prompt back is the registers of a run, which for pages of 128 leave two thread blocks on an SM; for up to 64, half of them, four.
// 4096 tokens of 32 heads of 128 on 8 (94 MB), in a chain of launches: 15.8 us in pages of 64, 6.0 TB/s, and 18.7 in pages of 128.  8 tokens: 3.6 and 3.8 us.
template <typename T, int D, int kMaxPage>
__global__ void __launch_bounds__(kAppendThreads, kMaxPage == 64 ? 4 : 2) rope_append_kernel(const AppendArgs a) {
  using R = Row<T, D>;
  constexpr int kRows = kAppendThreads / R::kLanes, kPasses = kMaxPage / kRows, kAtOnce = kPasses < 4 ? kPasses : 4, kWarps = kAppendThreads / 32;   // rows of a pass; passes of a page
  __shared__ float red[kWarps];
  __shared__ int s_slot[3 * kMaxPage], s_pos[3 * kMaxPage];
  __shared__ unsigned s_begins[kMaxPage / 32], s_ends[kMaxPage / 32], s_real[3 * kMaxPage / 32];
  static_assert(3 * kMaxPage % 32 == 0 && kAppendThreads % 32 == 0, "a warp has the 32 places of a word");
  pdl_enter();
  const int tid = threadIdx.x, lane = tid % R::kLanes, row = tid / R::kLanes, page = 1 << a.shift;
  const T* qkv = static_cast<const T*>(a.qkv);
  const int t0 = blockIdx.x * a.window, t1 = min(t0 + a.window, a.tokens);
  const auto valid = [&](int slot, int pos) { return slot >= 0 && slot < a.slots_total && pos >= 0 && pos < a.angle_rows; };
  if (blockIdx.y >= 2 * a.kv_heads) {                      // queries
    const int h0 = (blockIdx.y - 2 * a.kv_heads) * kQueryHeads, heads = min(kQueryHeads, a.q_heads - h0);
    for (int first = t0 + row; first < t1; first += 2 * kRows) {       // two tokens at once
      uint4 raw[2][kQueryHeads];
      float4 c[2], sn[2];
      bool ok[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int t = first + y * kRows;
        if (t >= t1) continue;
        const int slot = a.slots[t], pos = a.positions[t];
        const T* in = qkv + (size_t)t * a.row_stride + (size_t)h0 * D + lane * 8;
#pragma unroll
        for (int h = 0; h < kQueryHeads; ++h)
          if (h < heads) raw[y][h] = *reinterpret_cast<const uint4*>(in + h * D);
        ok[y] = valid(slot, pos);
        if (!ok[y] && a.status && lane == 0 && h0 == 0 && slot != -1) atomicOr(a.status, 16);
        const size_t at = ok[y] ? (size_t)pos * (D / 2) + lane * 4 : 0;
        c[y] = *reinterpret_cast<const float4*>(a.cosv + at);
        sn[y] = *reinterpret_cast<const float4*>(a.sinv + at);
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int t = first + y * kRows;
        if (t >= t1) continue;
        uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + ((size_t)t * a.q_heads + h0) * D + lane * 8);
#pragma unroll
        for (int h = 0; h < kQueryHeads; ++h) {
          if (h >= heads) continue;
          float v[8];
          R::widen(raw[y][h], v);
          R::rotate(v, c[y], sn[y]);
          uint4 r = {Half<T>::narrow(v[0], v[1]), Half<T>::narrow(v[2], v[3]), Half<T>::narrow(v[4], v[5]), Half<T>::narrow(v[6], v[7])};
          if (!ok[y]) r = {0, 0, 0, 0};
          out[(size_t)h * R::kLanes] = r;
        }
      }
    }
    return;
  }
  const int head = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  uint8_t* cache = values ? a.v_cache : a.k_cache;
  float* scales = values ? a.v_scale : a.k_scale;
  const T* in = qkv + (size_t)(a.q_heads + (values ? a.kv_heads : 0) + head) * D;
  // slots of the window (from place `page` on) and of a page before and behind it; negative: the token is not written
  for (int i = tid; i < 3 * kMaxPage; i += kAppendThreads) {
    const int t = t0 - page + i;
    int slot = -2, pos = 0;
    if (t >= 0 && t < a.tokens && i < a.window + 2 * page) {
      slot = a.slots[t];
      pos = a.positions[t];
      if (!valid(slot, pos)) slot = -2, pos = 0;
    }
    s_slot[i] = slot;
    s_pos[i] = pos;
    const unsigned real = __ballot_sync(htr::kFullWarp, slot >= 0);
    if ((tid & 31) == 0) s_real[i >> 5] = real;
  }
  __syncthreads();
  const auto last_of = [&](int i, int n) {                 // the last written token's place among the n before place i; -1: none
    int w = (i - 1) >> 5;
    unsigned m = s_real[w] & 0xFFFFFFFFu >> (31 - ((i - 1) & 31));
    while (m == 0 && 32 * w > i - n) m = s_real[--w];
    const int j = 32 * w + 31 - __clz(m);
    return m && j >= i - n ? j : -1;
  };
  const auto before = [&](int i) {                         // the slot of the written token before place i, fewer than `page` tokens back; negative: none
    const int slot = s_slot[i - 1];
    if (slot >= 0) return slot;
    const int j = last_of(i, page - 1);
    return j < 0 ? -2 : s_slot[j];
  };
  if (tid < kMaxPage) {                                    // where runs begin
    const int slot = tid < t1 - t0 ? s_slot[page + tid] : -2;
    const bool is = slot >= 0 && before(page + tid) >> a.shift != slot >> a.shift;
    const unsigned begins = __ballot_sync(htr::kFullWarp, is);
    if ((tid & 31) == 0) s_begins[tid >> 5] = begins;
  }
  __syncthreads();
  unsigned begins = s_begins[0];
  for (int word = 0;;) {
    while (begins == 0 && ++word < kMaxPage / 32) begins = s_begins[word];
    if (begins == 0) break;
    const int t = t0 + 32 * word + __ffs(begins) - 1;
    begins &= begins - 1;
    const int at_run = page + t - t0, slot = s_slot[at_run], off = slot & (page - 1);
    const size_t unit = (size_t)(slot >> a.shift) * a.kv_heads + head;
    const float old_scale = off ? scales[unit] : 0.f;
    // its run: up to the first token of another page or whose slot does not rise, without what is not written at the end
    if (tid < kMaxPage) {
      const int mine = tid < page ? s_slot[at_run + tid] : 0;
      const bool is = tid >= page || (tid && mine >= 0 && (mine >> a.shift != slot >> a.shift || mine <= before(at_run + tid)));
      const unsigned ends = __ballot_sync(htr::kFullWarp, is);
      if ((tid & 31) == 0) s_ends[tid >> 5] = ends;
    }
    __syncthreads();
    int end = page;
#pragma unroll
    for (int w = kMaxPage / 32 - 1; w >= 0; --w)
      if (s_ends[w]) end = 32 * w + __ffs(s_ends[w]) - 1;
    const int run = s_slot[at_run + end - 1] >= 0 ? end : last_of(at_run + end, end) + 1 - at_run;     // (the first is written)
    if (tid == 0 && end < page && s_slot[at_run + end] >> a.shift == slot >> a.shift && blockIdx.y == 0 && a.status) atomicOr(a.status, 16);
    int place[kPasses];                                    // of this thread's rows; negative: not written
#pragma unroll
    for (int x = 0; x < kPasses; ++x) place[x] = x * kRows + row < run ? s_slot[at_run + x * kRows + row] : -1;
    float v[kPasses][8];
    uint4 raw[kPasses];                                    // all loads before the first use
#pragma unroll
    for (int x = 0; x < kPasses; ++x) raw[x] = place[x] >= 0 ? *reinterpret_cast<const uint4*>(in + (size_t)(t + x * kRows + row) * a.row_stride + lane * 8) : uint4{0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < kPasses; ++x) R::widen(raw[x], v[x]);
    if (!values) {
#pragma unroll
      for (int x0 = 0; x0 < kPasses; x0 += kAtOnce) {
        float4 c[kAtOnce], s[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const size_t from = (size_t)s_pos[at_run + min((x0 + x) * kRows + row, run - 1)] * (D / 2) + lane * 4;
          c[x] = *reinterpret_cast<const float4*>(a.cosv + from);
          s[x] = *reinterpret_cast<const float4*>(a.sinv + from);
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) R::rotate(v[x0 + x], c[x], s[x]);
        if ((x0 + kAtOnce) * kRows >= run) break;
      }
    }
    // the largest of the run, NaN left aside; infinities saturate and do not set the scale either: where there is one, once more without
    const auto largest = [&](float limit) {
      float most = 0.f;
#pragma unroll
      for (int x = 0; x < kPasses; ++x)
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, limit > 0.f && fabsf(v[x][j]) > limit ? 0.f : fabsf(v[x][j]));
#pragma unroll
      for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(htr::kFullWarp, most, o));
      if ((tid & 31) == 0) red[tid >> 5] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) most = fmaxf(most, red[w]);
      return most;
    };
    float most = largest(0.f);
    if (most > 3.402823466e38f) {
      __syncthreads();
      most = largest(3.402823466e38f);
    }
    uint8_t* at = cache + (unit << a.shift) * D;
    int e = scale_exponent(most);
    if (off) {                                             // older tokens: their scale never shrinks, and they follow where it grows
      const int old = max((int)((__float_as_uint(old_scale) >> 23) & 255) - 127, kScaleFloor);
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
#pragma unroll
    for (int x = 0; x < kPasses; ++x) {
      if (place[x] < 0) continue;
      const uint2 r = {to_e4m3(v[x][0] * up, v[x][1] * up) | to_e4m3(v[x][2] * up, v[x][3] * up) << 16,
                       to_e4m3(v[x][4] * up, v[x][5] * up) | to_e4m3(v[x][6] * up, v[x][7] * up) << 16};
      *reinterpret_cast<uint2*>(at + (size_t)(place[x] & (page - 1)) * D + lane * 8) = r;
    }
    if (tid == 0) scales[unit] = exp2i(e);                 // (the old one was read by all before the last barrier)
    __syncthreads();                                       // s_ends and red have been read
  }
}

// ---- attention over the cache -----------------------------------------------------------------------------------------------------
//
// What bounds it for single tokens: the cache's bytes.  The query heads of one key/value head and a request's tokens of this step are the
// rows of one product, 8 or 16 at a time (row = token * group + head), on warp-level matrix instructions m16n8k16 with the cache as the
// 16-row operand (S^T = K Q^T, O^T = V^T P^T), so that 8 rows fill a tile.  A warp takes 16 cached tokens at a time for itself alone.  The dimensions that a product sums over and the rows of a result may be taken in any order, so
// every lane (g = lane / 4, c = lane % 4) reads whole 16-byte pieces of the cache's rows straight into fragments: of K those of the tokens g
// and g + 8 at dimensions 16 c ..., of V those of the tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9 at dimensions 16 g ...; e4m3 becomes fp16, which
// holds it exactly, on the way.  The tiles come through a ring of four per warp in shared memory, two bulk copies each, so that up to 190 KB
// are on their way to an SM; no barrier until a warp's tokens are through.
//
// The work is cut evenly, whatever the requests' lengths: a flat list of units of 64 tokens (of every request, row tile and key/value
// head, each with kBegin units more for what its beginning and end cost) in equal runs over the thread blocks.  A tile that lies in one run is finished
// there; of a tile that is cut every thread block leaves its part (maximum, sum, result) in the workspace, and a second launch joins them in the
// order of the tokens.
//
// 64 requests of 10 to 16384 tokens, 32 heads of 128 on 8 (759 MB): 128 us in a chain of launches, 5.9 TB/s (a call by itself 132 to 144).  Where it was tried, with
// tiles in registers 172; with bank conflicts among the pieces of V 162; in runs that count units alone 171; rows of V apart, by a copy for every two, 165.
//
// Queries are fp16 under a power of two per row (bf16 keeps all its bits: 29 binades of normal fp16 below the row's largest element).
// Probabilities are rounded to fp16, relative to the contribution that they make: the scale of the values' page is part of the exponent
// (P' = 2^(s + log2 scale - m)), and the sum of the probabilities, in float32 and of what they were before, takes it out again.  m lies 2^12
// below the largest P' when it moves, and it moves when one grows beyond 2^15.5, so that P' of 2^-26 of the largest and more are normal
// numbers: 2^-11 each at most, half of bf16's rounding of the output and a quarter of it, but as much as fp16's; smaller ones are off by up to 2^-37 of the largest.
// (A token that takes nearly everything and whose values are zero leaves the result to terms that small: 2^-26 is 18 nats.)

constexpr int kUnit = kAttWarps * 16;                      // tokens of a unit
// thread blocks per SM, by the registers that results and a tile need without spills and by the rings (of 128 dimensions 64 KB: three at most)
template <int D, int NT>
constexpr int kAttBlocks = D == 128 ? (NT == 1 ? 3 : 2) : (NT == 1 ? 4 : 3);
constexpr int kDepth = 4;                                  // stages of a warp's ring
template <int D>
constexpr int kRingBytes = kDepth * 32 * D;                // of a warp

// 16 tokens of keys and values of one page
template <int D>
struct Tile {
  uint4 k[2][D / 64];
  uint32_t v[4][D / 32];
  float ks, vs;
  __device__ __forceinline__ void read(const uint8_t* stage, int lane) {
    const int g = lane >> 2, c = lane & 3;
    const uint8_t *kp = stage + g * D + 16 * c, *vp = stage + 16 * D + 2 * c * D + D / 8 * g;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) k[t][i] = *reinterpret_cast<const uint4*>(kp + 8 * t * D + 64 * (D == 128 ? i ^ (g & 1) : i));
    // (rows of 128 bytes lie in the same banks: odd ones begin with their other half, and lanes with odd c with the other half of a piece of V)
    if (D == 128 && (g & 1))
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint4 y = k[t][0];
        k[t][0] = k[t][D / 64 - 1];
        k[t][D / 64 - 1] = y;
      }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint8_t* src = vp + ((x & 1) + 8 * (x >> 1)) * D;
      if constexpr (D == 128) {
        const uint2 one = *reinterpret_cast<const uint2*>(src + 8 * (c & 1)), two = *reinterpret_cast<const uint2*>(src + 8 * (~c & 1));
        v[x][0] = c & 1 ? two.x : one.x; v[x][1] = c & 1 ? two.y : one.y; v[x][2] = c & 1 ? one.x : two.x; v[x][3] = c & 1 ? one.y : two.y;
      } else {
        const uint2 raw = *reinterpret_cast<const uint2*>(src);
        v[x][0] = raw.x; v[x][1] = raw.y;
      }
    }
  }
};

// what a warp makes of its tokens
template <int D, int NT>
struct Running : Results<D, NT> {
  using Results<D, NT>::o;
  using Results<D, NT>::m;
  using Results<D, NT>::l;
  // 16 tokens from `at` on; `least`: tokens that every row sees, `end`: that some row sees
  template <typename R>
  __device__ __forceinline__ void add(Tile<D>& x, const R& rows, int at, int least, int end, int lane) {
    const int g = lane >> 2, c = lane & 3;
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint32_t a[4] = {x.k[0][i].x, x.k[0][i].y, x.k[0][i].z, x.k[0][i].w}, b[4] = {x.k[1][i].x, x.k[1][i].y, x.k[1][i].z, x.k[1][i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a0 = from_e4m3(a[j] & 0xFFFFu), a1 = from_e4m3(b[j] & 0xFFFFu), a2 = from_e4m3(a[j] >> 16), a3 = from_e4m3(b[j] >> 16);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_16816(s[t], a0, a1, a2, a3, rows.q[4 * i + j][t][0], rows.q[4 * i + j][t][1]);
      }
    }
    const float lv = __log2f(x.vs), inv = __fdividef(kSumUnit, x.vs);  // of a power of two: exact
    const bool edge = at + 16 > least;
    bool grows = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {                        // token g + 8 (i / 2), row 2 c + i % 2
        const float v = fmaf(s[t][i], rows.scale[t][i & 1] * x.ks, lv);
        s[t][i] = edge && at + g + 8 * (i >> 1) >= rows.end[t][i & 1] ? kNone : v;
        grows |= s[t][i] > m[t][i & 1] + 15.5f;
      }
    if (__any_sync(htr::kFullWarp, grows)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 2; ++y) this->raise(t, y, fmaxf(s[t][y], s[t][2 + y]));
    }
    uint32_t p[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = exp2_fast(s[t][i] - (m[t][i & 1] == kNone ? 0.f : m[t][i & 1]));
        l[t][i & 1] = fmaf(e[i], inv, l[t][i & 1]);
      }
      p[t][0] = transposed(pack_half(e[0], e[1]));
      p[t][1] = transposed(pack_half(e[2], e[3]));
    }
    if (edge) {                                            // tokens that some row or none sees: a NaN there is not for the others
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = at + 2 * c + (i & 1) + 8 * (i >> 1);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          if (token >= end) x.v[i][j] = 0;                 // behind the request's tokens lies what an earlier one left
          if (token >= least) any |= nan_bytes(x.v[i][j]);
        }
      }
      if (__any_sync(htr::kFullWarp, any != 0)) spread_nan(x, rows, at, least, lane);
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t a0 = __byte_perm(x.v[0][j], x.v[1][j], 0x5140), a1 = __byte_perm(x.v[0][j], x.v[1][j], 0x7362);
      const uint32_t b0 = __byte_perm(x.v[2][j], x.v[3][j], 0x5140), b1 = __byte_perm(x.v[2][j], x.v[3][j], 0x7362);
      const uint32_t f[8] = {from_e4m3(a0 & 0xFFFFu), from_e4m3(a0 >> 16), from_e4m3(b0 & 0xFFFFu), from_e4m3(b0 >> 16),
                             from_e4m3(a1 & 0xFFFFu), from_e4m3(a1 >> 16), from_e4m3(b1 & 0xFFFFu), from_e4m3(b1 >> 16)};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        mma_16816(o[2 * j][t], f[0], f[1], f[2], f[3], p[t][0], p[t][1]);
        mma_16816(o[2 * j + 1][t], f[4], f[5], f[6], f[7], p[t][0], p[t][1]);
      }
    }
  }
  // A NaN among the values of a token that not every row sees would reach them all as 0 * NaN: it is taken out of the fragments and given
  // to the rows that see it.  The values are spread over the lanes by token, the results by row, both by dimension.
  template <typename R>
  __device__ __forceinline__ void spread_nan(Tile<D>& x, const R& rows, int at, int least, int lane) {
    const int c = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = (i & 1) + 8 * (i >> 1);
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint32_t mine = at + 2 * c + place >= least ? nan_bytes(x.v[i][j]) : 0;
        x.v[i][j] &= ~mine;
#pragma unroll
        for (int from = 0; from < 4; ++from) {
          const uint32_t b = __shfl_sync(htr::kFullWarp, mine, (lane & ~3) | from);
          const int token = at + 2 * from + place;
#pragma unroll
          for (int d = 0; d < 4; ++d)                      // dimension 4 j + d of this lane's D / 8: tile 2 j + d / 2, half d % 2
            if (b >> (8 * d) & 1)
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                  if (token < rows.end[t][y]) o[2 * j + (d >> 1)][t][2 * (d & 1) + y] = __int_as_float(0x7FC00000);
        }
      }
    }
  }
};

// what an item costs besides its units (0: 171 us, 2: 133, 3: 128, 4: 128 at the sizes above)
constexpr int kBegin = 3;
using Work = Span<kUnit, kBegin>;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, (kAttBlocks<D, NT>)) paged_attention_kernel(const AttentionArgs a) {
  constexpr int kRows = 8 * NT, kRing = kRingBytes<D>;
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
  // ---- this thread block's run of units
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
    // ---- the tokens of this warp, 16 at a time: kDepth tiles are on their way.  Lane i holds page and scales of tile i of 32, and of the 32 after
    // them, which are fetched in time.
    if (segment) {                                         // the results of the last tile have been read
      __syncthreads();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const int* table = a.tables + r * a.table_stride;
    const int stop = min(u1 * kUnit, end), first_at = u0 * kUnit + warp * 16;
    const int tiles = first_at < stop && ok ? (stop - first_at + kUnit - 1) / kUnit : 0;
    struct Pages {
      int id;
      float ks, vs;
    };
    Pages some, then;
    const auto ids_of = [&](Pages& p, int tile) {          // (of a tile that is none: 0, not used)
      p.id = tile + lane < tiles ? table[(first_at + (tile + lane) * kUnit) >> a.shift] : 0;
    };
    const auto scales_of = [&](Pages& p) {
      const bool real = p.id >= 0 && p.id < a.pages;       // no such page: its tokens are not seen
      bad |= !real;
      const size_t unit = (size_t)(real ? p.id : 0) * a.kv_heads + kvh;
      if (!real) p.id = -1;
      p.ks = a.k_scale[unit];
      p.vs = a.v_scale[unit];
    };
    const auto request = [&](int tile, int id, bool held) {            // by all lanes, of a stage that they have read
      if (lane == 0 && !held) {
        const uint32_t bar = smem_u32(&s_full[warp][put]), to_stage = smem_u32(ring + warp * kRing + put * 32 * D);
        if (id >= 0 && id < a.pages) {
          const size_t base = ((((size_t)id * a.kv_heads + kvh) << a.shift) + ((first_at + tile * kUnit) & ((1 << a.shift) - 1))) * D;
          bar_expect(bar, 32 * D);
          bulk_load(to_stage, a.k_cache + base, 16 * D, bar);
          bulk_load(to_stage + 16 * D, a.v_cache + base, 16 * D, bar);
        } else {
          bar_arrive(bar);
        }
      }
      if (++put == kDepth) put = 0;
      ++ahead;
    };
    ids_of(some, 0);
    for (int i = 0; i < min(kDepth, tiles); ++i)
      request(i, __shfl_sync(htr::kFullWarp, some.id, i), i == 0 && segment == 0 && warp == 0 && a.withhold == (int)blockIdx.x + 1);
    scales_of(some);
    then = some;
    Rows<T, D, NT, 16> q;
    q.load(a, x.start, x.n, x.seen, row0, kvh, lane);
    Running<D, NT> run;
    run.clear();
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      const int j = i & 31;
      if (j == 0 && i) some = then;
      if (j == 0 && i + 32 < tiles) ids_of(then, i + 32);
      if (j == 8 && i + 24 < tiles) scales_of(then);
      ok = __all_sync(htr::kFullWarp, bar_wait(smem_u32(&s_full[warp][get]), phase, &s_fail, kWarpSpinLimit));
      if (!ok) break;
      const int id = __shfl_sync(htr::kFullWarp, some.id, j);
      Tile<D> tile;
      tile.ks = __shfl_sync(htr::kFullWarp, some.ks, j);
      tile.vs = __shfl_sync(htr::kFullWarp, some.vs, j);
      tile.read(ring + warp * kRing + get * 32 * D, lane);
      __syncwarp();
      --ahead;
      if (++get == kDepth) {
        get = 0;
        phase ^= 1;
      }
      if (i + kDepth < tiles) request(i + kDepth, __shfl_sync(htr::kFullWarp, j + kDepth < 32 ? some.id : then.id, (j + kDepth) & 31), false);
      if (id >= 0) run.add(tile, q, first_at + i * kUnit, least, end, lane);
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
  if (__any_sync(htr::kFullWarp, bad) && a.status && lane == 0) atomicOr(a.status, 32);
}

int attention_blocks(int head_dim, int tiles) {            // what the GPU holds at a time
  return current_device_sms() * (head_dim == 128 ? (tiles == 1 ? kAttBlocks<128, 1> : kAttBlocks<128, 2>) : tiles == 1 ? kAttBlocks<64, 1> : kAttBlocks<64, 2>);
}
int attention_tiles(int group, int max_new) { return (long long)group * max_new <= 8 ? 1 : 2; }

template <typename T, int D, int NT>
int attention_run(const AttentionArgs& a, cudaStream_t st) {
  const dim3 grid(attention_blocks(D, NT)), block(kAttThreads);
  constexpr int kBytes = kAttWarps * kRingBytes<D>;
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (!e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(paged_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  if (e) return htr::paged_fail(e);
  const int rc = paged_launch(paged_attention_kernel<T, D, NT>, grid, block, 1, kBytes, st, a);
  return rc != HTR_OK ? rc : paged_launch(paged_attention_join_kernel<T, D, NT, Work>, dim3(grid.x, kJoins<D, NT>), block, 1, 0, st, a);
}

template <typename T>
int attention_of(const AttentionArgs& a, int head_dim, int max_new, cudaStream_t st) {
  if (attention_tiles(a.group, max_new) == 1) return head_dim == 128 ? attention_run<T, 128, 1>(a, st) : attention_run<T, 64, 1>(a, st);
  return head_dim == 128 ? attention_run<T, 128, 2>(a, st) : attention_run<T, 64, 2>(a, st);
}

template <typename T, int D>
int append_run(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  return a.shift <= 6 ? paged_launch(rope_append_kernel<T, D, 64>, grid, dim3(kAppendThreads), 1, 0, st, a)
                      : paged_launch(rope_append_kernel<T, D, 128>, grid, dim3(kAppendThreads), 1, 0, st, a);
}
template <typename T>
int append_of(const AppendArgs& a, int head_dim, dim3 grid, cudaStream_t st) {
  return head_dim == 128 ? append_run<T, 128>(a, grid, st) : append_run<T, 64>(a, grid, st);
}

}  // namespace

namespace htr {

int paged_fail(int cuda_error) {
  t_last_cuda = cuda_error;
  return HTR_ERR_CUDA;
}
int attention_withhold() { return t_withhold; }

}  // namespace htr

extern "C" {

int htr_paged_last_cuda_error(void) { return t_last_cuda; }

void htr_paged_attention_withhold(int block) { t_withhold = block < 0 ? 0 : block + 1; }

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
    if (e) return paged_fail(e);
  }
  const int work = max_tokens > requests ? max_tokens : requests;
  const int blocks = work <= kPlanThreads ? 1 : kPlanMaxCluster;
  return paged_launch(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), blocks, smem, static_cast<cudaStream_t>(stream), a);
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
  const int units = 2 * kv_heads + (q_heads + kQueryHeads - 1) / kQueryHeads;
  int window = 1;                                          // tokens of a thread block: few where there is little to share out
  while (window < page_size && (int64_t)tokens * units > (int64_t)window * htr::current_device_sms() * 8) window *= 2;
  const AppendArgs a = {qkv, row_stride, positions, slots, tokens, cosv, sinv, angle_rows, q_heads, kv_heads, static_cast<uint8_t*>(k_cache),
                        static_cast<uint8_t*>(v_cache), k_scale, v_scale, (int64_t)pages << shift, shift, window, q_out, status};
  const dim3 grid((unsigned)((tokens + window - 1) / window), units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == HTR_DTYPE_BF16 ? append_of<__nv_bfloat16>(a, head_dim, grid, st) : append_of<__half>(a, head_dim, grid, st);
}

size_t htr_paged_attention_workspace_bytes(int tokens, int requests, int q_heads, int kv_heads, int head_dim, int max_new, int table_width, int page_size) {
  if (tokens < 1 || requests < 1 || q_heads < 1 || kv_heads < 1 || max_new < 1 || table_width < 1 || page_shift(page_size) < 0 || (head_dim != 64 && head_dim != 128)) return 0;
  if (attention_tc_serves(tokens, requests, q_heads, q_heads / kv_heads, max_new, (long long)table_width * page_size, head_dim)) return attention_tc_workspace(head_dim);
  const int tiles = attention_tiles(q_heads / kv_heads, max_new);
  const size_t rows = 8 * tiles;
  return attention_blocks(head_dim, tiles) * (2 * rows * (head_dim + 2) * sizeof(float) + sizeof(int4));
}

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
      (int64_t)pages << shift > 0x7FFFFFFF || (int64_t)table_width << shift > 1 << 30)
    return HTR_ERR_TOO_LARGE;
  if (tokens == 0) return HTR_OK;
  if (!q || !starts || !seen || !tables || !k_cache || !v_cache || !k_scale || !v_scale || !out) return HTR_ERR_NULL;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return HTR_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < htr_paged_attention_workspace_bytes(tokens, requests, q_heads, kv_heads, head_dim, max_new, table_width, page_size))
    return HTR_ERR_WORKSPACE;
  if (!aligned16(workspace)) return HTR_ERR_ALIGNMENT;
  const bool tc = attention_tc_serves(tokens, requests, q_heads, q_heads / kv_heads, max_new, (long long)table_width * page_size, head_dim);
  int4* cuts = static_cast<int4*>(workspace);
  const AttentionArgs a = {q, starts, seen, tables, table_stride, table_width, requests, tokens, q_heads, kv_heads, q_heads / kv_heads, max_new,
                           static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale, pages, shift,
                           scale * 1.4426950408889634f, out, status, reinterpret_cast<float*>(cuts + attention_blocks(head_dim, attention_tiles(q_heads / kv_heads, max_new))), cuts, t_withhold};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tc) return attention_tc_run(a, dtype, head_dim, workspace, st);
  return dtype == HTR_DTYPE_BF16 ? attention_of<__nv_bfloat16>(a, head_dim, max_new, st) : attention_of<__half>(a, head_dim, max_new, st);
}

}  // extern "C"
