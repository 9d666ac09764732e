// Attention over the paged 8-bit cache for many rows a request (prompts, shared key/value heads): tcgen05.mma with accumulators in tensor
// memory.
//
// A tile is up to 128 rows: the query heads of one key/value head for as many whole tokens as fit (row = token * group + head).  Per unit of 64
// cached tokens: S = Q K^T (128 x 64), P = 2^(S - m) in fp16, O += P V.  S, P and O are in tensor memory (P over S, two of them in turns), Q, K and V
// in shared memory as core matrices.
//  * Keys are multiplied as they are, e4m3, and go from memory straight to their core matrices; a row of Q is a sum of e4m3 parts of four significant
//    bits each under one power of two (two parts for bf16, three for fp16: exact down to 2^-18 of the row's largest element), which costs what
//    one product of 16-bit operands would, without its conversions.
//  * Values become fp16, exactly, on their way (P would need three e4m3 parts, at four conversions an element), transposed by byte permutes
//    of eight rows in registers: their operand wants eight tokens of a dimension side by side.
// Two roles per thread block, two thread blocks per SM:
//   warps 0-3  a thread per row (its lane of tensor memory): scale, mask, running maximum and sum, exponentials, P.  No shuffles.  S of the next unit
//              is there when one is done.
//   warps 4-7  keys and values of the next unit; the first of them issues the products, Q K^T of the next unit before P V of this one.
// What bounds it: per 128 rows and 64 tokens 512 cycles of tensor pipe, 512 of exponentials (16 a cycle and SM) and about 400 of issue on each
// scheduler, which the two thread blocks overlap.
// The scales of keys and values are powers of two per page: they enter the exponent (S * scale + log2 scale of the values - m) and leave
// the sum; see paged_kernels.cu, whose cut of the work into even runs over the thread blocks, parts and join this kernel shares, with
// runs of units of (request, tile, head), each as many as its last token sees.
#include "paged_common.cuh"

namespace {

using namespace htr;

constexpr int kThreads = 256, kRows = 128, kUnit = 64, kGroups = kUnit / 16, kMaxRequests = 1024, kBlocksPerSm = 2;
constexpr int kTmemColumns = 256;                          // S (P over it) at 0 and 64, O at 128
constexpr unsigned kSpinLimit = 2000000u;                  // polls of a wait before it gives up (about two seconds)

template <typename T, int D>
struct Layout {                                            // bytes of the operands: core matrices of 8 rows x 16 bytes
  // Q as a sum of e4m3 of four significant bits each: two for the 8 bits of bf16, three for the 11 of fp16
  static constexpr int kParts = Half<T>::kBits > 8 ? 3 : 2;
  static constexpr int kGroup = 8 * D;                     // Q, K: between groups of 8 rows; 128 between neighbours in K
  static constexpr int kTokens = 16 * D + 16;              // V: between groups of 8 tokens (16 more: stores of 8 groups meet 8 bank groups)
  static constexpr int kQ = 0, kPart = 16 * kGroup, kK = kQ + kParts * kPart, kKeys = 8 * kGroup, kV = kK + 2 * kKeys,
                       kValues = 8 * kTokens, kBytes = kV + 2 * kValues;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// start, distance of core matrices adjacent in K, distance of groups of 8 rows, in 16 bytes; version 1, no swizzle
__device__ __forceinline__ uint64_t descriptor(uint32_t at, int next_k, int next_rows) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(next_k >> 4) << 16 | (uint64_t)(next_rows >> 4) << 32 | 1ull << 46;
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.b32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
  return done != 0;
}
// bounded: false when the limit ran out or another role has given up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* fail) {
  if (bar_try(bar, parity)) return true;
  for (unsigned i = 0; i < kSpinLimit; ++i) {
    if (bar_try(bar, parity)) return true;
    if ((i & 255) == 255 && *fail) return false;
  }
  *fail = 1;
  return false;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {      // e4m3
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
               "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
               "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 16 or 32 columns of this thread's lane of tensor memory
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at) : "memory");
}
// (what was loaded goes through the wait, so that no use of it is moved before)
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two lanes of float32 arithmetic in one instruction
__device__ __forceinline__ void fma2(float& x, float& y, uint32_t a, uint32_t b, float by, float add) {
  asm("{\n\t.reg .b64 r, s, t;\n\tmov.b64 r, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\tmov.b64 t, {%5, %5};\n\tfma.rn.f32x2 r, r, s, t;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(x), "=f"(y) : "r"(a), "r"(b), "f"(by), "f"(add));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 r, s;\n\tmov.b64 r, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tadd.rn.f32x2 r, r, s;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ uint32_t max_half2(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// a request's tiles, and what one of them sees
struct Request {
  int start, n, seen, per, tiles;                          // per: tokens of a tile
  __device__ __forceinline__ Request(const AttentionArgs& a, int r) {
    start = max(a.starts[r], 0);
    n = max(min(a.starts[r + 1], a.tokens) - start, 0);
    seen = min(max(a.seen[r], 0), a.width << a.shift);
    per = kRows / a.group;
    tiles = (min(n, a.max_new) + per - 1) / per;
  }
  __device__ __forceinline__ int tokens(const AttentionArgs& a, int tile) const { return min(per, min(n, a.max_new) - tile * per); }
  __device__ __forceinline__ int end(const AttentionArgs& a, int tile) const { return max(seen - n + tile * per + tokens(a, tile), 0); }
  __device__ __forceinline__ int units(const AttentionArgs& a, int tile) const { return max((end(a, tile) + kUnit - 1) / kUnit, 1); }
};

struct Shared {
  unsigned long long k_full[2], s_full[2], v_full[2], p_full[2], pv_done[2], q_full, drained;    // of the units in turns
  long long sums[kMaxRequests];                            // units of each request
  long long total, skip;
  int r, tile, head, unit;                                 // where this thread block's run begins
  uint32_t tmem;
  int fail, nan;
  float ks[2][kGroups], lv[2][kGroups], inv[2][kGroups];                     // of the 16-token groups of a unit: scales; log2 and inverse of those of the values
  unsigned real[2];                                        // groups that have a page
};

// the run of a thread block, piece by piece: every role walks it for itself
struct Walk {
  int r, tile, head, u0, u1, units;
  long long left;
  int start, n, seen, per, tiles, row_tokens, least, end;
  __device__ __forceinline__ Walk(const Shared& s, long long count) : r(s.r), tile(s.tile), head(s.head), u0(s.unit), left(count) {}
  __device__ __forceinline__ void look(const AttentionArgs& a) {
    Request x(a, r);
    while (x.tiles == 0) x = Request(a, ++r);              // (there is one: `left` counts its units)
    start = x.start; n = x.n; seen = x.seen; per = x.per; tiles = x.tiles;
    row_tokens = x.tokens(a, tile);
    least = max(seen - n + tile * per + 1, 0);
    end = x.end(a, tile);
    units = x.units(a, tile);
    u1 = (int)min((long long)units, u0 + left);
  }
  __device__ __forceinline__ void next(const AttentionArgs& a) {
    left -= u1 - u0;
    u0 = 0;
    if (++head < a.kv_heads) return;
    head = 0;
    if (++tile < tiles) return;
    tile = 0;
    ++r;
  }
};

template <int D>
constexpr int kPartFloats = kRows * (D + 2);

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) paged_attention_tc_kernel(const AttentionArgs a) {
  using Y = Layout<T, D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Shared s;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* fail = &s.fail;
  // ---- this thread block's run: units of each request by its warps, then the place where the run begins
  for (int r = warp; r < a.requests; r += kThreads / 32) {
    const Request x(a, r);
    long long sum = 0;
    for (int t = lane; t < x.tiles; t += 32) sum += x.units(a, t);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullWarp, sum, o);
    if (lane == 0) s.sums[r] = sum * a.kv_heads;
  }
  if (tid == 0) {
    s.fail = s.nan = 0;
    for (int i = 0; i < 2; ++i) {
      bar_init(smem_u32(&s.k_full[i]), 128);
      bar_init(smem_u32(&s.s_full[i]), 1);
      bar_init(smem_u32(&s.v_full[i]), 128);
      bar_init(smem_u32(&s.p_full[i]), 128);
      bar_init(smem_u32(&s.pv_done[i]), 1);
    }
    bar_init(smem_u32(&s.q_full), 128);
    bar_init(smem_u32(&s.drained), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    a.cuts[blockIdx.x] = {0, 0, 0, 0};
  }
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"((uint32_t)kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  // (tensor memory is ours: a dependent launch that starts early cannot take it from thread blocks of this one)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  long long total = 0, share = 1, from = 0;
  if (warp == 0) {
    for (int r = lane; r < a.requests; r += 32) total += s.sums[r];
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(kFullWarp, total, o);
    share = max((total + gridDim.x - 1) / gridDim.x, 1LL);
    from = blockIdx.x * share;
    if (lane == 0) s.total = total;
    if (from < total) {
      int r = 0;
      long long before = 0;                                // units before the request
      for (int base = 0; base < a.requests; base += 32) {
        const long long mine = base + lane < a.requests ? s.sums[base + lane] : 0;
        long long end = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long x = __shfl_up_sync(kFullWarp, end, o);
          if (lane >= o) end += x;
        }
        const unsigned hit = __ballot_sync(kFullWarp, before + end > from);
        if (hit) {
          r = base + __ffs(hit) - 1;
          before += __shfl_sync(kFullWarp, end - mine, __ffs(hit) - 1);
          break;
        }
        before += __shfl_sync(kFullWarp, end, 31);
      }
      const Request x(a, r);
      for (int base = 0; base < x.tiles; base += 32) {
        const long long mine = base + lane < x.tiles ? (long long)x.units(a, base + lane) * a.kv_heads : 0;
        long long end = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(kFullWarp, end, o);
          if (lane >= o) end += y;
        }
        const unsigned hit = __ballot_sync(kFullWarp, before + end > from);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            const long long rest = from - (before + end - mine);
            const int units = x.units(a, base + lane);
            s.r = r;
            s.tile = base + lane;
            s.head = (int)(rest / units);
            s.unit = (int)(rest % units);
          }
          break;
        }
        before += __shfl_sync(kFullWarp, end, 31);
      }
    }
  }
  __syncthreads();
  total = s.total;
  share = max((total + gridDim.x - 1) / gridDim.x, 1LL);
  from = blockIdx.x * share;
  const long long count = min(share, total - from);
  const uint32_t tmem = s.tmem;
  const uint32_t k_full = smem_u32(s.k_full), s_full = smem_u32(s.s_full), v_full = smem_u32(s.v_full), p_full = smem_u32(s.p_full),
                 pv_done = smem_u32(s.pv_done), q_full = smem_u32(&s.q_full);
  // barrier and phase of unit n of this thread block
  const auto reached = [&](uint32_t bars, uint32_t n) { return bar_wait(bars + 8 * (n & 1), n >> 1 & 1, fail); };
  uint32_t n = 0;                                          // units so far
  if (count > 0 && warp < 4) {
    // ================= softmax: a thread per row
    const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
    const int row = tid;
    bool ok = true;
    const auto follow = [&](float f) {                     // results relative to a new reference
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_load16(lanes + 128 + c, o);
#pragma unroll
        for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
        tmem_store(lanes + 128 + c, o);
      }
      tmem_stored();
    };
    Walk w(s, count);
    for (int segment = 0; w.left > 0 && ok; ++segment, w.next(a)) {
      w.look(a);
      const int i = row / a.group, head = w.head * a.group + row - i * a.group, rows = w.row_tokens * a.group;
      const bool mine = row < rows;
      const size_t place = ((size_t)(w.start + w.tile * w.per + i) * a.q_heads + head) * D;
      const int row_end = mine ? max(w.seen - w.n + w.tile * w.per + i + 1, 0) : 0;
      // queries: e4m3 parts under a power of two per row
      float row_scale;
      {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + place);
        float most = 0.f;
        if (mine)
#pragma unroll 4
          for (int j = 0; j < D / 8; ++j) {
            const uint4 raw = src[j];
            const float2 f[4] = {Half<T>::wide(raw.x), Half<T>::wide(raw.y), Half<T>::wide(raw.z), Half<T>::wide(raw.w)};
#pragma unroll
            for (int x = 0; x < 4; ++x) most = fmaxf(most, fmaxf(fabsf(f[x].x), fabsf(f[x].y)));
          }
        const int e = query_exponent(most) - 7;            // the largest between 2^7 and 2^8
        const float up = most > 3.402823466e38f ? __int_as_float(0x7FC00000) : exp2i(e);       // (an infinite element: all scores are NaN or infinite)
        row_scale = exp2i(-e) * a.scale;
        uint8_t* dst = smem + Y::kQ + (row >> 3) * Y::kGroup + (row & 7) * 16;
#pragma unroll 1
        for (int j = 0; j < D / 16; ++j) {                 // 16 dimensions: 16 bytes of each part
          float f[16];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint4 raw = mine ? src[2 * j + x] : uint4{0, 0, 0, 0};
            const uint32_t w4[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float2 v = Half<T>::wide(w4[y]);
              f[8 * x + 2 * y] = v.x * up;
              f[8 * x + 2 * y + 1] = v.y * up;
            }
          }
#pragma unroll
          for (int part = 0; part < Y::kParts; ++part) {
            uint32_t r[4];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const uint32_t two = to_e4m3(f[2 * x], f[2 * x + 1]);
              const float2 held = Half<__half>::wide(from_e4m3(two));
              f[2 * x] -= held.x;                          // what is left for the next part, exactly
              f[2 * x + 1] -= held.y;
              r[x >> 1] = x & 1 ? r[x >> 1] | two << 16 : two;
            }
            *reinterpret_cast<uint4*>(dst + part * Y::kPart + j * 128) = make_uint4(r[0], r[1], r[2], r[3]);
          }
        }
        fence_async();
        fence_before();
        bar_arrive(q_full);
      }
      float m = kNone, l = 0.f;
      for (int u = w.u0; u < w.u1 && ok; ++u, ++n) {
        ok = __all_sync(kFullWarp, reached(k_full, n) && reached(s_full, n));
        if (!ok) break;
        fence_after();
        const int at = u * kUnit, turn = n & 1;
        const unsigned real = s.real[turn];
        const uint32_t scores = lanes + 64 * turn;
        if (32 * warp < rows) {
          uint32_t raw[2][32];
          tmem_load(scores, raw[0]);
          tmem_load(scores + 32, raw[1]);
          tmem_loaded(raw[0]);
          tmem_loaded(raw[1]);
          float v[kUnit], base = m == kNone ? 0.f : m;
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            const float by = row_scale * s.ks[turn][g], add = s.lv[turn][g] - base;
#pragma unroll
            for (int c = 16 * g; c < 16 * g + 16; c += 2) fma2(v[c], v[c + 1], raw[c >> 5][c & 31], raw[c >> 5][(c & 31) + 1], by, add);
          }
          if (at + kUnit > w.least || real != (1u << kGroups) - 1) {
#pragma unroll
            for (int c = 0; c < kUnit; ++c)
              if (at + c >= row_end || !(real >> (c >> 4) & 1)) v[c] = kNone;
          }
          float sum[kGroups][2];
          uint32_t p[kUnit / 2];
          const auto exponentials = [&] {
#pragma unroll
            for (int c = 0; c < kUnit / 2; ++c) {
              const float x = exp2_fast(v[2 * c]), y = exp2_fast(v[2 * c + 1]);
              if (c & 7) add2(sum[c >> 3][0], sum[c >> 3][1], x, y);
              else sum[c >> 3][0] = x, sum[c >> 3][1] = y;
              p[c] = pack_half(x, y);
            }
          };
          exponentials();
          // whether P stays below 2^14: of its halves, whose overflow is infinite
          uint32_t most[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) most[c] = max_half2(max_half2(p[c], p[c + 8]), max_half2(p[c + 16], p[c + 24]));
#pragma unroll
          for (int c = 4; c; c >>= 1)
#pragma unroll
            for (int x = 0; x < c; ++x) most[x] = max_half2(most[x], most[x + c]);
          const float2 pair = Half<__half>::wide(most[0]);
          const bool grows = m == kNone || fmaxf(pair.x, pair.y) > 16384.f;
          if (__any_sync(kFullWarp, grows)) {              // a new reference, 2^6 above which the largest lies; what there is follows
            float top = kNone;
#pragma unroll
            for (int c = 0; c < kUnit; ++c) top = fmaxf(top, v[c]);
            const bool moves = grows && top > kNone;
            const float now = moves ? base + top - 6.f : m, f = moves && m != kNone ? exp2_fast(m - now) : 1.f, down = moves ? base - now : 0.f;
#pragma unroll
            for (int c = 0; c < kUnit; ++c) v[c] += down;
            m = now;
            l *= f;
            if (u > w.u0) {
              ok = __all_sync(kFullWarp, reached(pv_done, n - 1));   // (S of this unit came before the results of the last one)
              fence_after();
              if (ok) follow(f);
            }
            exponentials();
          }
#pragma unroll
          for (int g = 0; g < kGroups; ++g) l = fmaf(sum[g][0] + sum[g][1], s.inv[turn][g], l);
          __syncwarp();
          tmem_store(scores, reinterpret_cast<const uint32_t (&)[16]>(p[0]));
          tmem_store(scores + 16, reinterpret_cast<const uint32_t (&)[16]>(p[16]));
          tmem_stored();
        }
        fence_before();
        bar_arrive(p_full + 8 * turn);
      }
      if (!ok) break;
      ok = __all_sync(kFullWarp, reached(pv_done, n - 1));
      if (!ok) break;
      fence_after();
      // ---- the tile, or this run's part of it
      const bool whole = w.u0 == 0 && w.u1 == w.units;
      float* part = a.parts + ((size_t)blockIdx.x * 2 + (segment != 0)) * kPartFloats<D>;
      const float by = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;     // a row that sees nothing: zeros
      const bool empty = l == 0.f;
      const bool nan = *(volatile int*)&s.nan != 0;
      if (32 * warp < rows) {
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          __syncwarp();
          tmem_load16(lanes + 128 + c, o);
          if (mine) {
          float f[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) f[x] = empty ? 0.f : __uint_as_float(o[x]) * by;
          if (nan)                                         // values that are NaN were left out of the last units: given to the rows that see them
            for (int token = max(w.least, w.u0 * kUnit); token < min(row_end, w.u1 * kUnit); ++token) {
              const int id = a.tables[w.r * a.table_stride + (token >> a.shift)];
              if (id < 0 || id >= a.pages) continue;
              const uint8_t* v = a.v_cache + ((((size_t)id * a.kv_heads + w.head) << a.shift) + (token & ((1 << a.shift) - 1))) * D + c;
#pragma unroll
              for (int x = 0; x < 16; ++x)
                if ((v[x] & 0x7F) == 0x7F) f[x] = __int_as_float(0x7FC00000);
            }
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + place + c);
#pragma unroll
            for (int x = 0; x < 2; ++x)
              dst[x] = {Half<T>::narrow(f[8 * x], f[8 * x + 1]), Half<T>::narrow(f[8 * x + 2], f[8 * x + 3]),
                        Half<T>::narrow(f[8 * x + 4], f[8 * x + 5]), Half<T>::narrow(f[8 * x + 6], f[8 * x + 7])};
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              *reinterpret_cast<float4*>(part + ((c / 4 + x) * kRows + row) * 4) = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
          }
          }
        }
        if (!whole && mine) {
          part[kRows * D + row] = m;
          part[kRows * D + kRows + row] = l;
        }
      }
      if (!whole && w.u0 == 0 && tid == 0)                 // it begins here and ends elsewhere: request, tile, parts, head and place of the first
        a.cuts[blockIdx.x] = {w.r, w.tile, 1 + (int)((w.units - w.u1 + share - 1) / share), 2 * w.head + (segment != 0)};
      fence_before();                                      // (the next tile's first product into O comes after this thread's next arrival)
    }
  } else if (count > 0 && warp < 8) {
    // ================= cache -> fp16 core matrices
    const int t = tid - 128, cw = warp - 4;
    const int tg = lane & 7, dc = (lane >> 3) + 4 * cw;    // values: group of 8 tokens, piece of D / 16 dimensions
    bool ok = true, bad = false;
    uint32_t vr[8][D / 64];
    Walk w(s, count);
    w.look(a);
    // three units are under way: one that is written, the next, whose rows are being fetched, and the one after it, whose pages are
    Walk f = w;
    int fu = w.u0;                                         // of the pages that are fetched
    struct Pages {
      int k, v, scale, head, at;
      bool all;                                            // every token of the unit lies in a page and before the end
    };
    const auto pages_of = [&](Pages& p) {
      p.at = fu * kUnit;
      p.head = f.head;
      const int* table = a.tables + f.r * a.table_stride;
      const auto page = [&](int token) { return token < f.end ? table[token >> a.shift] : -1; };
      p.k = page(p.at + 16 * cw);
      p.v = page(p.at + 8 * tg);
      p.scale = page(p.at + 16 * (t & (kGroups - 1)));
      p.all = p.at + kUnit <= f.end;
      if (++fu == f.u1) {
        f.next(a);
        if (f.left > 0) {
          f.look(a);
          fu = f.u0;
        }
      }
    };
    const int place_mask = (1 << a.shift) - 1;
    const auto valid = [&](int id) { return id >= 0 && id < a.pages; };
    // (a page that is none is read as the first one and left aside later)
    const auto keys_of = [&](const Pages& p, uint32_t n) { // straight to their core matrices
      const int id = valid(p.k) ? p.k : 0;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int token = p.at + 16 * cw + 8 * b + (lane & 7);
        const uint8_t* src = a.k_cache + ((((size_t)id * a.kv_heads + p.head) << a.shift) + (token & place_mask)) * D + (lane >> 3) * 16;
        const uint32_t dst = smem_u32(smem + Y::kK + (n & 1) * Y::kKeys + (2 * cw + b) * Y::kGroup + (lane & 7) * 16 + (lane >> 3) * 128);
#pragma unroll
        for (int x = 0; x < D / 64; ++x)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + x * 512), "l"(src + 64 * x) : "memory");
      }
    };
    const auto values_of = [&](const Pages& p) {
      const int id = valid(p.v) ? p.v : 0, token = p.at + 8 * tg;
      const uint8_t* src = a.v_cache + ((((size_t)id * a.kv_heads + p.head) << a.shift) + (token & place_mask)) * D + dc * (D / 16);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if constexpr (D == 128) {
          const uint2 raw = *reinterpret_cast<const uint2*>(src + x * D);
          vr[x][0] = raw.x; vr[x][1] = raw.y;
        } else {
          vr[x][0] = *reinterpret_cast<const uint32_t*>(src + x * D);
        }
      }
    };
    float ks = 0.f, vs = 1.f;
    const auto scales_of = [&](const Pages& p) {
      const size_t at = (size_t)(valid(p.scale) ? p.scale : 0) * a.kv_heads + p.head;
      ks = a.k_scale[at];
      vs = a.v_scale[at];
    };
    Pages now, next, later;                                // of the unit that is written, of the next, of the one after it
    pages_of(now);
    keys_of(now, 0);
    values_of(now);
    scales_of(now);
    next = now;
    if (f.left > 0) pages_of(next);
    long long owed = count - 1;                            // units that come after this one
    // the products, issued by the first of these warps
    const uint32_t idesc_s = 1u << 4 | (uint32_t)(kUnit >> 3) << 17 | (128u >> 4) << 24, idesc_o = 1u << 4 | ((uint32_t)D >> 3) << 17 | (128u >> 4) << 24;
    const uint64_t dq = descriptor(smem_u32(smem + Y::kQ), 128, Y::kGroup), dk = descriptor(smem_u32(smem + Y::kK), 128, Y::kGroup),
                   dv = descriptor(smem_u32(smem + Y::kV), Y::kTokens, 128);
    uint32_t fresh = 0, q_phase = 0;                       // fresh: 0 where the unit before is the first of its tile
    const auto scores = [&](uint32_t n, bool first) {
      if (!__all_sync(kFullWarp, reached(k_full, n) && (!first || bar_wait(q_full, q_phase, fail)))) return false;
      fence_after();
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < Y::kParts; ++part)
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            mma_ss(tmem + 64 * (n & 1), dq + part * (Y::kPart >> 4) + 16 * k, dk + (n & 1) * (Y::kKeys >> 4) + 16 * k, idesc_s, (part | k) != 0);
        commit(s_full + 8 * (n & 1));
      }
      __syncwarp();
      if (first) q_phase ^= 1;
      return true;
    };
    const auto results = [&](uint32_t n) {                 // (P of the unit is there)
      if (!__all_sync(kFullWarp, reached(v_full, n))) return false;
      fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kUnit / 16; ++k)
          mma_ts(tmem + 128, tmem + 64 * (n & 1) + 8 * k, dv + (n & 1) * (Y::kValues >> 4) + (uint64_t)(k * (2 * Y::kTokens >> 4)), idesc_o, k != 0 ? 1u : fresh);
        commit(pv_done + 8 * (n & 1));
      }
      __syncwarp();
      return true;
    };
    for (; w.left > 0 && ok;) {
      for (int u = w.u0; u < w.u1 && ok; ++u, ++n) {
        const bool first = u == w.u0;                      // of its tile: its queries come after the results of the last tile
        const int turn = n & 1;
        // ---- keys, which are on their way, and scales
        if (cw == 0) {
          const unsigned mask = __ballot_sync(kFullWarp, t < kGroups && valid(now.scale));
          bad |= now.scale != -1 && !valid(now.scale);     // (-1: behind the last token)
          if (t < kGroups) {
            s.ks[turn][t] = ks;
            s.lv[turn][t] = __log2f(vs);                   // of a power of two: exact
            s.inv[turn][t] = __fdividef(1.f, vs);
          }
          // (a group behind the last token has no page either: the rows' ends mask it)
          if (t == 0) s.real[turn] = mask;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_async();
        bar_arrive(k_full + 8 * turn);
        if (cw == 0 && !first && !(ok = scores(n, false))) break;
        later = next;
        if (f.left > 0) pages_of(later);
        // ---- values, once the results of the unit before the last are done
        if (n >= 2) ok = __all_sync(kFullWarp, reached(pv_done, n - 2));
        if (!ok) break;
        const int vtoken = u * kUnit + 8 * tg;
        if (!now.all || !valid(now.v)) {                   // behind the request's tokens lies what an earlier one left
#pragma unroll
          for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
              if (vtoken + x >= w.end || !valid(now.v)) vr[x][j] = 0;
        }
        if (vtoken + 8 > w.least) {                        // tokens that not all rows see: a NaN there is not for the others
          uint32_t any = 0;
#pragma unroll
          for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const uint32_t b = vtoken + x >= w.least ? nan_bytes(vr[x][j]) : 0;
              vr[x][j] &= ~b;
              any |= b;
            }
          if (any) s.nan = 1;
        }
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {                 // four dimensions of eight tokens
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            lo[x] = __byte_perm(vr[2 * x][j], vr[2 * x + 1][j], 0x5140);
            hi[x] = __byte_perm(vr[2 * x][j], vr[2 * x + 1][j], 0x7362);
          }
          const int d = dc * (D / 16) + 4 * j;
          uint8_t* dst = smem + Y::kV + turn * Y::kValues + tg * Y::kTokens + (d >> 3) * 128 + (d & 7) * 16;
          *reinterpret_cast<uint4*>(dst) = {from_e4m3(lo[0] & 0xFFFFu), from_e4m3(lo[1] & 0xFFFFu), from_e4m3(lo[2] & 0xFFFFu), from_e4m3(lo[3] & 0xFFFFu)};
          *reinterpret_cast<uint4*>(dst + 16) = {from_e4m3(lo[0] >> 16), from_e4m3(lo[1] >> 16), from_e4m3(lo[2] >> 16), from_e4m3(lo[3] >> 16)};
          *reinterpret_cast<uint4*>(dst + 32) = {from_e4m3(hi[0] & 0xFFFFu), from_e4m3(hi[1] & 0xFFFFu), from_e4m3(hi[2] & 0xFFFFu), from_e4m3(hi[3] & 0xFFFFu)};
          *reinterpret_cast<uint4*>(dst + 48) = {from_e4m3(hi[0] >> 16), from_e4m3(hi[1] >> 16), from_e4m3(hi[2] >> 16), from_e4m3(hi[3] >> 16)};
        }
        fence_async();
        bar_arrive(v_full + 8 * turn);
        // ---- the next unit's rows; its keys go where those of the last unit were
        if (owed > 0) {
          values_of(next);
          scales_of(next);
          if (n >= 1) ok = __all_sync(kFullWarp, reached(s_full, n - 1));
          if (!ok) break;
          keys_of(next, n + 1);
        }
        --owed;
        now = next;
        next = later;
        // ---- results of the last unit.  (All of these warps wait for its P: none is then two phases ahead of a thread that still waits for keys.)
        if (n >= 1) {
          ok = __all_sync(kFullWarp, reached(p_full, n - 1));
          if (!ok || (cw == 0 && !(ok = results(n - 1)))) break;
        }
        if (cw == 0 && first && !(ok = scores(n, true))) break;
        fresh = !first;
      }
      if (!ok) break;
      w.next(a);
      if (w.left > 0) w.look(a);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (cw == 0) {
      if (ok) ok = __all_sync(kFullWarp, reached(p_full, n - 1)) && results(n - 1);
      if (!ok) {                                           // products in flight end before the tensor memory goes back
        if (elect_one()) commit(smem_u32(&s.drained));
        __syncwarp();
        for (unsigned i = 0; i < kSpinLimit && !bar_try(smem_u32(&s.drained), 0); ++i) {}
      }
    }
    if (bad && a.status) atomicOr(a.status, 32);
  }
  fence_before();
  __syncthreads();
  if (tid == 0 && s.fail && a.status) atomicOr(a.status, 64);
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemColumns) : "memory");
  }
}

// Joins the parts of the tiles that were cut: a thread block per run of the launch before, a thread per row and four dimensions.
template <typename T, int D>
__global__ void __launch_bounds__(512) paged_attention_tc_join_kernel(const AttentionArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.z == 0) return;
  const Request x(a, cut.x);
  const int kvh = cut.w >> 1, rows = x.tokens(a, cut.y) * a.group;
  const float *head = a.parts + ((size_t)blockIdx.x * 2 + (cut.w & 1)) * kPartFloats<D>, *tail = a.parts + (size_t)blockIdx.x * 2 * kPartFloats<D>;
  for (int z = threadIdx.x; z < kRows * (D / 4); z += 512) {
    const int row = z % kRows, d = z / kRows;
    if (row >= rows) continue;
    float m = head[kRows * D + row], l = head[kRows * D + kRows + row];
    float4 y = *reinterpret_cast<const float4*>(head + (d * kRows + row) * 4);
#pragma unroll 2
    for (int i = 1; i < cut.z; ++i) {
      const float* part = tail + (size_t)i * 2 * kPartFloats<D>;
      const float pm = part[kRows * D + row], pl = part[kRows * D + kRows + row];
      const float4 v = *reinterpret_cast<const float4*>(part + (d * kRows + row) * 4);
      const float now = fmaxf(m, pm), f = now == kNone ? 1.f : exp2_fast(m - now), h = now == kNone ? 1.f : exp2_fast(pm - now);
      m = now;
      l = l * f + pl * h;
      y.x = y.x * f + v.x * h; y.y = y.y * f + v.y * h; y.z = y.z * f + v.z * h; y.w = y.w * f + v.w * h;
    }
    const float by = l == 0.f ? 0.f : 1.f / l;
    const int i = row / a.group;
    T* dst = static_cast<T*>(a.out) + ((size_t)(x.start + cut.y * x.per + i) * a.q_heads + (size_t)kvh * a.group + row - i * a.group) * D + 4 * d;
    *reinterpret_cast<uint2*>(dst) = {Half<T>::narrow(y.x * by, y.y * by), Half<T>::narrow(y.z * by, y.w * by)};
  }
}

int device_sms() {
  static int cache[64] = {0};
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64 && cache[dev]) return cache[dev];
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) return 148;
  if (dev >= 0 && dev < 64) cache[dev] = v;
  return v;
}

template <typename T, int D>
int run(const AttentionArgs& a, cudaStream_t st) {
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (!e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(paged_attention_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (Layout<T, D>::kBytes));
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  if (e) return paged_fail(e);
  const dim3 grid(device_sms() * kBlocksPerSm);
  const int rc = paged_launch(paged_attention_tc_kernel<T, D>, grid, dim3(kThreads), 1, (Layout<T, D>::kBytes), st, a);
  return rc != HTR_OK ? rc : paged_launch(paged_attention_tc_join_kernel<T, D>, grid, dim3(512), 1, 0, st, a);
}

}  // namespace

namespace htr {

// More than 16 rows a tile: the other kernel takes 16 of them per pass over the cache.
bool attention_tc_serves(int requests, int group, int max_new) { return requests <= kMaxRequests && group <= kRows && (long long)group * max_new > 16; }

size_t attention_tc_workspace(int head_dim) {
  return (size_t)device_sms() * kBlocksPerSm * (sizeof(int4) + 2 * sizeof(float) * (head_dim == 128 ? kPartFloats<128> : kPartFloats<64>));
}

int attention_tc_run(const AttentionArgs& args, int dtype, int head_dim, void* workspace, cudaStream_t st) {
  AttentionArgs a = args;
  a.cuts = static_cast<int4*>(workspace);
  a.parts = reinterpret_cast<float*>(a.cuts + device_sms() * kBlocksPerSm);
  if (dtype == HTR_DTYPE_BF16) return head_dim == 128 ? run<__nv_bfloat16, 128>(a, st) : run<__nv_bfloat16, 64>(a, st);
  return head_dim == 128 ? run<__half, 128>(a, st) : run<__half, 64>(a, st);
}

}  // namespace htr
