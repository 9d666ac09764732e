// Attention over the paged cache, in 8 or 4 bits, for many rows a request (prompts, shared key/value heads): tcgen05.mma with accumulators in tensor
// memory.
//
// An item is up to 256 rows, two tiles of 128: the query heads of one key/value head for as many whole tokens as fit (row = token * group +
// head).  Per unit of 64 cached tokens and tile: S = Q K^T (128 x 64), P = 2^(S - m) in fp16, O += P V.  S, P and O are in tensor memory (P over S, two
// of them in turns), Q, K and V in shared memory.  An item of at most 128 rows is a twin: its units go to the two tiles in
// turns, and their results are joined at the end.
//  * Keys are multiplied as they are, e4m3, and go from memory straight to their core matrices; a row of Q is a sum of e4m3 parts of four significant
//    bits each under one power of two, which costs what one product of 16-bit operands would, without its conversions.  Two parts for the 8 bits of
//    bf16, three for the 11 of fp16; e4m3 ends at 2^-9 and the row's largest element lies at 2^7 to 2^8, so elements down to 2^-9 of it (fp16: 2^-6) are
//    exact, and smaller ones are off by up to 2^-17 of the largest (the other kernel holds 28 binades).
//  * Values become fp16, exactly, on their way (P would need three e4m3 parts, at four conversions an element).
//  * All operands lie in the swizzled layouts (rows of 128 bytes; values with the dimensions inside): from core matrices without a swizzle the
//    products were fetched at a quarter of the rate, 288 us for a prompt of 2048 tokens behind 2048.
// Roles of the one thread block of an SM, whose registers are shared out among them (160 for the softmax, 96 for the others):
//   warps 0-7    a thread per row and tile (its lane of tensor memory): scale, mask, running maximum and sum, exponentials, P.  No shuffles.
//   warps 8-11   values of the units, two of them on their way in registers, into a ring of four
//   warps 12-13  keys (copies that pass no register) and scales, into a ring of four
//   warp 14      (of 16) the products: Q K^T up to two units (a twin: four) before the P V that follow
// What bounds it: per 256 rows and 64 tokens 1024 cycles of tensor pipe and as many of exponentials (16 a cycle and SM).  Measured, a prompt's second
// 2048 tokens over 4096 (32 heads of 128 on 8, 103 GFLOP), in a chain of launches: 176 us, 587 TFLOP/s (fp16, with its third part of the queries, 189); a unit
// takes 2650 cycles where no reference moves, of which the exponentials of the two tiles side by side take 1350, tensor memory to registers and back 600, the
// hand-over between roles 500; 12000 to begin and end an item.  References that move cost 6 of the 176: with 2^4 in place of 2^12 below, 170.  (A unit of 128 tokens
// with one hand-over, but the products of a tile in line with its softmax, took 179 where this took 165.)
// Reference of a row's softmax: 2^12 under the largest term when it moves, and it moves when the sum of eight terms leaves the range of fp16 (eight
// that are equal do not): terms down to 2^-26 of the largest keep all bits of fp16 (its step below that is 2^-24, of which P V sees at most a half each).
// The scales of keys and values are powers of two per page: they enter the exponent (S * scale + log2 scale of the values - m) and leave
// the sum; see paged_kernels.cu, whose cut of the work into even runs over the thread blocks, parts and join this kernel shares, with
// runs of units of (request, item, head), each as many as its last token sees.
// Over the cache of 4 bits everything is fp16: a code times its token's scale (2 and 8 significant bits) is, exactly, under a power of two for each 16
// tokens of keys and of values, which takes the place of a page's scale; the warps that feed keys and values widen both on their way.  A row of Q is one part
// of fp16 (28 binades), for the same tensor pipe as bf16's two of e4m3.  A value whose scale is NaN is a zero, and its key NaN, which reaches those that see it.
// Where the scales of 16 keys lie more than 13 binades apart, or those of 16 values more than 4, each of the tokens keeps its own: codes are widened as they are, and the scale
// multiplies the scores or enters the exponent and the sum token by token.  The power of two comes from all 16, and a row need not see all of them: so keys and values are exact
// whatever lies beside them, and what a token's neighbours, seen or not, can do to its probability is to take less than five binades from the bits below.  A unit
// with such tokens takes some two times as long: the prompt above 384 us where every unit has one, 180 where one page in 64 has; and that they are looked for costs it 3 us of 176.
// Seven warps (8-13, 15) feed both, 16 tokens at a time, by code that stands once and is not unrolled: twice and unrolled it drove the softmax out of the instruction cache
// (339 us where this took 208).  The reference lies 2^4 under the largest term when it moves, and then for all rows of the warp whose largest lies higher: terms down to 2^-18 of the
// largest keep all bits, smaller ones are off by up to 2^-29 of it.  Keys whose norms differ by token make references move, a move costs 1900 cycles, and with 2^12 every second unit of the
// prompt above had one: 200 us, with 2^8 183, with 2^4 172 (2^0: 169; none: 146).  P goes to tensor memory before the
// sums are looked at, and once more where a reference moves: 171 (these without scales of tokens, with which it is 176).  Two threads a row (16 softmax warps of 88 registers) took 186, a thread for each kind of product 191.
#pragma once
#include <type_traits>

#include "paged_common.cuh"

namespace {

using namespace htr;

constexpr int kThreads = 512, kTile = 128, kRows = 256, kUnit = 64, kGroups = kUnit / 16, kMaxRequests = 1024;
constexpr int kTmemColumns = 512;                          // of a tile: S (P over it) at 0 and 64, O at 128
template <int kBits>
constexpr float kTopOf = kBits == 4 ? 4.f : 12.f;          // where a row's largest term lies when its reference moves
constexpr int kRing = 4, kScales = 8;                      // units of keys and of values in shared memory; of their scales, read by all rows
constexpr int kKeySpread = 13, kValueSpread = 4;           // binades between the scales of 16 tokens of 4 bits from which on each token keeps its own

template <typename T, int D, int kBits>
struct Layout {                                            // bytes of the operands
  static constexpr bool kFour = kBits == 4;
  // Q as a sum of e4m3 of four significant bits each: two for the 8 bits of bf16, three for the 11 of fp16
  static constexpr int kParts = kFour ? 1 : Half<T>::kBits > 8 ? 3 : 2, kWide = kFour ? 2 : 1;      // kWide: bytes of an element of Q and K
  static constexpr int kQ = 0, kPart = kTile * D * kWide, kQTile = kParts * kPart, kK = kQ + 2 * kQTile, kKeys = kUnit * D * kWide, kV = kK + kRing * kKeys,
                       kValues = kUnit * 2 * D, kBytes = kV + kRing * kValues + 1024;      // (1024: to align the first)
  // 16-byte piece of a row of D bytes, swizzled (128 or 64 bytes)
  static __device__ __forceinline__ int piece(int row, int chunk) { return row * D + ((D == 128 ? chunk ^ (row & 7) : chunk ^ (row >> 1 & 3)) << 4); }
  // 8 dimensions of a row in fp16, in blocks of kRows rows of 64 dimensions: of a token's values, and of its key and of a row of Q where they are fp16
  template <int kRows = kUnit>
  static __device__ __forceinline__ int value(int row, int chunk) { return (chunk >> 3) * (kRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }
};

// start; distances of 128-byte columns (where rows are longer) and of groups of 8 rows, in 16 bytes; version 1; swizzle of 128 bytes (2) or 64 (4)
__device__ __forceinline__ uint64_t descriptor(uint32_t at, int next_column, int next_rows, uint64_t swizzle) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(next_column >> 4) << 16 | (uint64_t)(next_rows >> 4) << 32 | 1ull << 46 | swizzle << 61;
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
__device__ __forceinline__ void mma_ss_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
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

// 32 columns of this thread's lane of tensor memory (stores: 16)
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
  unsigned long long k_full[kRing], k_free[kRing], v_full[kRing], v_free[kRing];      // of the units in turns
  unsigned long long s_full[4], p_full[4], pv_done[4];     // of a tile's units in turns: 2 * tile + turn
  unsigned long long q_full, twin_full, twin_done, drained;
  long long sums[kMaxRequests];                            // units of each request
  long long total;
  int r, tile, head, unit;                                 // where this thread block's run begins
  uint32_t tmem;
  int fail, nan;
  alignas(16) float ks[kScales][kGroups], lv[kScales][kGroups], inv[kScales][kGroups];     // of the 16-token groups of a unit: scales; log2 and inverse of those of the values
  unsigned char real[kScales][kGroups];                    // 1: groups that have a page; 2: whose tokens keep their own scales
  float twin_m[kTile], twin_l[kTile];
  int finished[8];                                         // items of the run that the rows of a warp are through with
};

// the run of a thread block, piece by piece: every role walks it for itself
struct Walk {
  int r, tile, head, u0, u1, units;
  long long left;
  int start, n, seen, per, tiles, rows, least, end;
  bool twin;
  __device__ __forceinline__ Walk(const Shared& s, long long count) : r(s.r), tile(s.tile), head(s.head), u0(s.unit), left(count) {}
  __device__ __forceinline__ void look(const AttentionArgs& a) {
    Request x(a, r);
    while (x.tiles == 0) x = Request(a, ++r);              // (there is one: `left` counts its units)
    start = x.start; n = x.n; seen = x.seen; per = x.per; tiles = x.tiles;
    rows = x.tokens(a, tile) * a.group;
    twin = rows <= kTile;
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
constexpr int kJoins = kRows * (D / 4) / 512;
template <int D>
constexpr int kPartFloats = kRows * (D + 2);

template <typename T, int D, int kBits>
__global__ void __launch_bounds__(kThreads, 1) paged_attention_tc_kernel(const AttentionArgs a) {
  using Y = Layout<T, D, kBits>;
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  uint8_t* smem = raw_smem + (-smem_u32(raw_smem) & 1023);
  __shared__ Shared s;
  // of tokens that keep their own scales, as ks, lv and inv
  constexpr int kOwn = kBits == 4 ? kScales : 1;
  __shared__ __align__(16) float own_ks[kOwn][kUnit], own_lv[kOwn][kUnit], own_inv[kOwn][kUnit];
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
    for (int i = 0; i < kRing; ++i) {
      bar_init(smem_u32(&s.k_full[i]), (kBits == 4 ? 128 : 64) + (i == 0 && a.withhold == (int)blockIdx.x + 1));      // (withheld: one arrival more than come)
      bar_init(smem_u32(&s.k_free[i]), 1);
      bar_init(smem_u32(&s.v_full[i]), 128);
      bar_init(smem_u32(&s.v_free[i]), 1);
    }
    for (int i = 0; i < 4; ++i) {
      bar_init(smem_u32(&s.s_full[i]), 1);
      bar_init(smem_u32(&s.p_full[i]), 128);
      bar_init(smem_u32(&s.pv_done[i]), 1);
    }
    bar_init(smem_u32(&s.q_full), 256);
    bar_init(smem_u32(&s.twin_full), 128);
    bar_init(smem_u32(&s.twin_done), 128);
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
  // unit n of the thread block in a ring of bars, and unit c of a tile in its two
  const auto ring = [&](unsigned long long* bars, uint32_t size, uint32_t n) { return bar_wait(smem_u32(bars + n % size), n / size & 1, fail); };
  const auto turn = [&](unsigned long long* bars, int x, uint32_t c) { return bar_wait(smem_u32(bars + 2 * x + (c & 1)), c >> 1 & 1, fail); };
  // ================= values (warps 8-11) and keys (12-13)
  const auto feed = [&](auto which) {
    constexpr bool keys = decltype(which)::value;
    const int kw = warp - 12, vw = warp - 8;
    const int place_mask = (1 << a.shift) - 1;
    const auto valid = [&](int id) { return id >= 0 && id < a.pages; };
    bool ok = true, bad = false;
    // units one after the other; the pages of the next are fetched while the rows of one are
    struct Unit {
      int id[2], head, at, end, least;
    };
    Walk f(s, count);
    f.look(a);
    int fu = f.u0;
    const auto pages_of = [&](Unit& p) {
      p.at = fu * kUnit;
      p.head = f.head;
      p.end = f.end;
      p.least = f.least;
      const int* table = a.tables + f.r * a.table_stride;
      const int token = p.at + (keys ? 32 * kw : 16 * vw);
      p.id[0] = token < f.end ? table[token >> a.shift] : -1;
      if (keys) p.id[1] = token + 16 < f.end ? table[(token + 16) >> a.shift] : -1;
      if (++fu < f.u1) return;
      f.next(a);
      if (f.left <= 0) return;
      f.look(a);
      fu = f.u0;
    };
    Unit next;
    pages_of(next);
    if constexpr (keys) {
      // ---- straight to their place; a unit is announced when the copies of the two after it are under way
      float ks = 0.f, vs = 1.f;
      bool real = false;
      const auto write_scales = [&](uint32_t n) {          // lane g holds those of group 2 kw + g
        const int slot = n % kScales;
        if (lane < 2) {
          s.ks[slot][2 * kw + lane] = ks;
          s.lv[slot][2 * kw + lane] = __log2f(vs);         // of a power of two: exact
          s.inv[slot][2 * kw + lane] = __fdividef(kSumUnit, vs);
          s.real[slot][2 * kw + lane] = real;
        }
      };
      const auto announce_keys = [&](uint32_t n) {
        fence_async();
        bar_arrive(smem_u32(&s.k_full[n % kRing]));
      };
      uint32_t n = 0;
      for (; n < count && ok; ++n) {
        const Unit now = next;
        if (n + 1 < count) pages_of(next);
        if (n >= kRing) ok = __all_sync(kFullWarp, ring(s.k_free, kRing, n - kRing));
        if (!ok) break;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int id = valid(now.id[b >> 1]) ? now.id[b >> 1] : 0, token = now.at + 32 * kw + 8 * b + (lane & 7);
          const uint8_t* src = a.k_cache + ((((size_t)id * a.kv_heads + now.head) << a.shift) + (token & place_mask)) * D + (lane >> 3) * 16;
          const uint32_t dst = smem_u32(smem + Y::kK + (n % kRing) * Y::kKeys);
#pragma unroll
          for (int y = 0; y < D / 64; ++y)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + Y::piece(32 * kw + 8 * b + (lane & 7), (lane >> 3) + 4 * y)), "l"(src + 64 * y)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (n >= 1) write_scales(n - 1);
        {
          const int id = now.id[lane & 1];
          real = valid(id);
          bad |= id != -1 && !real;                        // (-1: behind the last token)
          const size_t at = (size_t)(real ? id : 0) * a.kv_heads + now.head;
          ks = a.k_scale[at];
          vs = a.v_scale[at];
        }
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        if (n >= 2) announce_keys(n - 2);
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (ok) {
        write_scales(n - 1);
        if (n >= 2) announce_keys(n - 2);
        announce_keys(n - 1);
      }
      if (bad && a.status) atomicOr(a.status, 32);
    } else {
      // ---- through registers, widened: a warp takes 16 tokens, a lane two of them (8 apart), 16 dimensions of each 64
      uint4 v[2][2][D / 64];
      Unit unit[2];
      const auto rows_of = [&](const Unit& p, uint4 (&v)[2][D / 64]) {         // (a page that is none is read as the first one and left aside later)
        const int id = valid(p.id[0]) ? p.id[0] : 0, token = p.at + 16 * vw + (lane & 7);
        const uint8_t* src = a.v_cache + ((((size_t)id * a.kv_heads + p.head) << a.shift) + (token & place_mask)) * D + (lane >> 3) * 16;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int y = 0; y < D / 64; ++y) v[b][y] = *reinterpret_cast<const uint4*>(src + 8 * b * D + 64 * y);
      };
      const auto write = [&](const Unit& p, uint4 (&v)[2][D / 64], uint32_t n) {
        if (p.at + 16 * vw + 16 > p.least || !valid(p.id[0])) {
          uint32_t any = 0;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            // behind the request's tokens lies what an earlier one left; a NaN of a token that not all rows see is not for the others
            const int token = p.at + 16 * vw + 8 * b + (lane & 7);
            const bool gone = token >= p.end || !valid(p.id[0]), some = token >= p.least;
            const auto clean = [&](uint32_t& w) {
              if (gone) w = 0;
              const uint32_t nan = some ? nan_bytes(w) : 0;
              w &= ~nan;
              any |= nan;
            };
#pragma unroll
            for (int y = 0; y < D / 64; ++y) {
              clean(v[b][y].x);
              clean(v[b][y].y);
              clean(v[b][y].z);
              clean(v[b][y].w);
            }
          }
          if (any) s.nan = 1;
        }
        uint8_t* dst = smem + Y::kV + (n % kRing) * Y::kValues;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int y = 0; y < D / 64; ++y) {
            const uint4 w = v[b][y];
            const int token = 16 * vw + 8 * b + (lane & 7), chunk = 2 * ((lane >> 3) + 4 * y);
            *reinterpret_cast<uint4*>(dst + Y::template value<>(token, chunk)) = {from_e4m3(w.x & 0xFFFFu), from_e4m3(w.x >> 16), from_e4m3(w.y & 0xFFFFu), from_e4m3(w.y >> 16)};
            *reinterpret_cast<uint4*>(dst + Y::template value<>(token, chunk + 1)) = {from_e4m3(w.z & 0xFFFFu), from_e4m3(w.z >> 16), from_e4m3(w.w & 0xFFFFu), from_e4m3(w.w >> 16)};
          }
        fence_async();
        bar_arrive(smem_u32(&s.v_full[n % kRing]));
      };
      // the rows of unit n + 1 are fetched before those of unit n are written, the pages of unit n + 2 before that
      unit[0] = next;
      if (count > 1) pages_of(next);
      rows_of(unit[0], v[0]);
      for (uint32_t n = 0; n < count && ok; n += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (n + h >= count || !ok) break;
          if (n + h + 1 < count) {
            unit[h ^ 1] = next;
            rows_of(unit[h ^ 1], v[h ^ 1]);
            if (n + h + 2 < count) pages_of(next);
          }
          if (n + h >= kRing) ok = __all_sync(kFullWarp, ring(s.v_free, kRing, n + h - kRing));
          if (ok) write(unit[h], v[h], n + h);
        }
      }
    }
  };
  // ================= keys and values of 4 bits (warps 8-13 and 15): 16 tokens of either are a piece of work, eight of which make a unit and go round
  const auto feed4 = [&] {
    constexpr int kFeeders = 7, kPer = D == 128 ? 8 : 16, kPasses = 16 / kPer;           // a lane has 32 dimensions of every kPer-th token
    const int me = warp == 15 ? 6 : warp - 8, place_mask = (1 << a.shift) - 1, in_pass = lane % kPer, piece = lane / kPer;
    const auto valid = [&](int id) { return id >= 0 && id < a.pages; };
    const auto held = [&](float s) { return fminf(fmaxf(s, kScaleLeast), kScaleMost); };         // (NaN: kScaleLeast)
    const uint32_t pieces = 8 * (uint32_t)count;
    bool ok = true, bad = false;
    struct Piece {
      int id, head, at, end;                               // at: its first token
    };
    struct Rows {
      uint4 v[kPasses];
      uint16_t ks, vs;                                     // of token lane % 16
    };
    Walk f(s, count);
    f.look(a);
    int fu = f.u0;
    uint32_t fn = 0;                                       // the unit of the thread block that fu is
    const auto page_of = [&](uint32_t n) {                 // pieces come in rising order
      while (fn < n >> 3) {
        ++fn;
        if (++fu < f.u1) continue;
        f.next(a);
        f.look(a);
        fu = f.u0;
      }
      Piece p;
      p.at = fu * kUnit + 16 * (n & 3);
      p.head = f.head;
      p.end = f.end;
      p.id = p.at < f.end ? (a.tables + f.r * a.table_stride)[p.at >> a.shift] : -1;
      return p;
    };
    const auto rows_of = [&](const Piece& p, uint32_t n, Rows& x) {            // (a page that is none is read as the first one and left aside later)
      const size_t row = ((((size_t)(valid(p.id) ? p.id : 0) * a.kv_heads + p.head) << a.shift) + (p.at & place_mask));
      const uint8_t* src = (n & 4 ? a.v_cache : a.k_cache) + row * (D / 2) + in_pass * (D / 2) + 16 * piece;
#pragma unroll
      for (int b = 0; b < kPasses; ++b) x.v[b] = *reinterpret_cast<const uint4*>(src + kPer * b * (D / 2));
      x.ks = reinterpret_cast<const uint16_t*>(a.k_scale)[row + (lane & 15)];
      x.vs = reinterpret_cast<const uint16_t*>(a.v_scale)[row + (lane & 15)];
    };
    // the exponent of the largest scale of the 16; `s`: 0 where there is none
    const auto exponent = [&](float s) {
      const unsigned most = __reduce_max_sync(kFullWarp, __float_as_uint(s));
      return most ? (int)(most >> 23) - 127 : 0;
    };
    const auto write = [&](const Piece& p, uint32_t piece_n, const Rows& x) {
      const uint32_t n = piece_n >> 3;
      const bool values = piece_n & 4, real = valid(p.id), there = real && p.at + (lane & 15) < p.end;
      const int group = piece_n & 3;
      bad |= p.at < p.end && !real;
      const float vs = __uint_as_float((uint32_t)x.vs << 16), ks = __uint_as_float((uint32_t)x.ks << 16);
      const bool nan_v = vs != vs, nan_k = ks != ks;
      const int ev = exponent(there && !nan_v ? held(vs) : 0.f);
      const bool own_v = __any_sync(kFullWarp, there && !nan_v && held(vs) < exp2i(ev - kValueSpread));      // (ev >= -100)
      float by;
      if (values) {
        by = there && !nan_v ? own_v ? 1.f : held(vs) * exp2i(-ev) : 0.f;
        if (n >= kRing) ok = __all_sync(kFullWarp, ring(s.v_free, kRing, n - kRing));
        if (!ok) return;
      } else {
        const int ek = exponent(there && !nan_k ? held(ks) : 0.f);
        const bool own_k = __any_sync(kFullWarp, there && !nan_k && held(ks) < exp2i(ek - kKeySpread));
        by = !there ? 0.f : nan_k || nan_v ? __int_as_float(0x7FC00000) : own_k ? 1.f : held(ks) * exp2i(-ek);
        if (n >= kRing) ok = __all_sync(kFullWarp, ring(s.k_free, kRing, n - kRing));
        if (!ok) return;
        const int slot = n % kScales;
        if (lane == 0) {
          s.ks[slot][group] = exp2i(ek);
          s.lv[slot][group] = (float)ev;
          s.inv[slot][group] = exp2i(-ev) * kSumUnit;
          s.real[slot][group] = real | (own_k || own_v ? 2 : 0);
        }
        if ((own_k || own_v) && lane < 16) {               // (what is not there is masked)
          own_ks[slot][16 * group + lane] = own_k ? held(ks) : exp2i(ek);
          own_lv[slot][16 * group + lane] = own_v ? __log2f(held(vs)) : (float)ev;
          own_inv[slot][16 * group + lane] = own_v ? __fdividef(kSumUnit, held(vs)) : exp2i(-ev) * kSumUnit;
        }
      }
      const uint32_t two = pack_half(by, by);
      uint8_t* dst = smem + (values ? Y::kV + (n % kRing) * Y::kValues : Y::kK + (n % kRing) * Y::kKeys);
#pragma unroll
      for (int b = 0; b < kPasses; ++b) {
        const uint32_t scale = __shfl_sync(kFullWarp, two, kPer * b + in_pass);
        const uint32_t w[4] = {x.v[b].x, x.v[b].y, x.v[b].z, x.v[b].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          uint32_t r[4];
          from_e2m1(w[y], r);
#pragma unroll
          for (int z = 0; z < 4; ++z) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(r[z]) : "r"(scale));
          *reinterpret_cast<uint4*>(dst + Y::template value<>(16 * group + kPer * b + in_pass, 4 * piece + y)) = {r[0], r[1], r[2], r[3]};
        }
      }
      fence_async();
      bar_arrive(smem_u32((values ? s.v_full : s.k_full) + n % kRing));
    };
    // the rows of a warp's next piece are fetched before those of one are written, the page of the piece after it before that.  (Two at a time, without the moves,
    // were code that the softmax had to fetch its own again after: the prompt below took 339 us in place of 208.)
    Piece one, next;
    Rows x;
    uint32_t n = me;
    if (n < pieces) {
      one = page_of(n);
      rows_of(one, n, x);
    }
    if (n + kFeeders < pieces) next = page_of(n + kFeeders);
#pragma unroll 1
    for (; n < pieces && ok; n += kFeeders) {
      const Piece now = one;
      const Rows held_rows = x;
      if (n + kFeeders < pieces) {
        one = next;
        rows_of(one, n + kFeeders, x);
        if (n + 2 * kFeeders < pieces) next = page_of(n + 2 * kFeeders);
      }
      write(now, n, held_rows);
    }
    if (bad && a.status) atomicOr(a.status, 32);
  };
  // registers of the four warpgroups: 2 * 160 + 2 * 96 = 4 * 128, what the launch has
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    if (count > 0) {
    // ================= softmax: a thread per row of tile x
    constexpr float kTop = kTopOf<kBits>;
    const int x = warp >> 2, row = tid & (kTile - 1);
    const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), mine_at = lanes + 256 * x;
    bool ok = true;
    const auto follow = [&](float f) {                     // results relative to a new reference
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_load(mine_at + 128 + c, o);
        tmem_loaded(o);
#pragma unroll
        for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
        tmem_store(mine_at + 128 + c, reinterpret_cast<const uint32_t (&)[16]>(o[0]));
        tmem_store(mine_at + 128 + c + 16, reinterpret_cast<const uint32_t (&)[16]>(o[16]));
      }
      tmem_stored();
    };
    Walk w(s, count);
    uint32_t n = 0, done = 0, twins = 0;                   // units of the thread block, of this tile; twins so far
    int segment = 0;
    for (; w.left > 0 && ok; ++segment, w.next(a)) {
      w.look(a);
      const int place_row = w.twin ? row : x * kTile + row, i = place_row / a.group, head = w.head * a.group + place_row - i * a.group;
      const bool mine = place_row < w.rows, warp_has_rows = (w.twin ? 0 : x * kTile) + 32 * (warp & 3) < w.rows;
      const size_t place = ((size_t)(w.start + w.tile * w.per + i) * a.q_heads + head) * D;
      const int row_end = mine ? max(w.seen - w.n + w.tile * w.per + i + 1, 0) : 0;
      // 16 bytes of a row as it is in memory: of queries before they are taken apart, of results where the queries were, whose products are done
      const auto staged = [&](int row, int chunk) {
        if constexpr (kBits == 4) return smem + Y::kQ + x * Y::kQTile + Y::template value<kTile>(row, chunk);
        else return smem + Y::kQ + x * Y::kQTile + chunk / (D / 16) * Y::kPart + Y::piece(row, chunk % (D / 16));
      };
      // queries: e4m3 parts under a power of two per row (of a twin: both tiles hold them)
      float row_scale;
      {
        // 8 lanes a row, 4 rows at once: whole lines are read; a lane holds dimensions 8 * (lane & 7) to + 7 of each 64
        uint8_t* dst = smem + Y::kQ + x * Y::kQTile;
        const int first = row & ~31;                       // of this warp
        const auto row_of = [&](int t) { return 4 * t + (lane >> 3); };
        const long long at = mine ? (long long)place : -1;
#pragma unroll 4
        for (int t = 0; t < 8; ++t) {                      // all rows on their way, to where the parts will lie
          const long long from = __shfl_sync(kFullWarp, at, row_of(t));
          const T* src = static_cast<const T*>(a.q) + max(from, 0LL) + 8 * (lane & 7);
#pragma unroll
          for (int y = 0; y < D / 64; ++y)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(staged(first + row_of(t), 8 * y + (lane & 7)))), "l"(src + 64 * y),
                         "r"(from >= 0 ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        row_scale = 0.f;
#pragma unroll 2
        for (int t = 0; t < 8; ++t) {
          uint4 raw[D / 64];                               // (read by the lane that fetched it; the parts of a row go where its lanes' pieces were)
#pragma unroll
          for (int y = 0; y < D / 64; ++y) raw[y] = *reinterpret_cast<const uint4*>(staged(first + row_of(t), 8 * y + (lane & 7)));
          __syncwarp();
          float f[D / 64][8], most = 0.f;
#pragma unroll
          for (int y = 0; y < D / 64; ++y) {
            const uint32_t w4[4] = {raw[y].x, raw[y].y, raw[y].z, raw[y].w};
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float2 v = Half<T>::wide(w4[z]);
              f[y][2 * z] = v.x;
              f[y][2 * z + 1] = v.y;
              most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
          }
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(kFullWarp, most, o));
          const int e = query_exponent(most, kBits == 4 ? 14 : 7);     // the largest between 2^7 and 2^8, as fp16 between 2^14 and 2^15
          const float up = most > 3.402823466e38f ? __int_as_float(0x7FC00000) : exp2i(e);     // (an infinite element: all scores are NaN or infinite)
          const int owner = __shfl_sync(kFullWarp, e, (lane & 3) * 8);
          if (lane >> 2 == t) row_scale = exp2i(-owner) * a.scale;
#pragma unroll
          for (int y = 0; y < D / 64; ++y) {
#pragma unroll
            for (int z = 0; z < 8; ++z) f[y][z] *= up;
            if constexpr (kBits == 4) {
              *reinterpret_cast<uint4*>(staged(first + row_of(t), 8 * y + (lane & 7))) = {pack_half(f[y][0], f[y][1]), pack_half(f[y][2], f[y][3]), pack_half(f[y][4], f[y][5]),
                                                                                         pack_half(f[y][6], f[y][7])};
            } else {
#pragma unroll
            for (int part = 0; part < Y::kParts; ++part) {
              uint32_t r[2];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const uint32_t two = to_e4m3(f[y][2 * z], f[y][2 * z + 1]);
                const float2 held = Half<__half>::wide(from_e4m3(two));
                f[y][2 * z] -= held.x;                     // what is left for the next part, exactly
                f[y][2 * z + 1] -= held.y;
                r[z >> 1] = z & 1 ? r[z >> 1] | two << 16 : two;
              }
              *reinterpret_cast<uint2*>(dst + part * Y::kPart + Y::piece(first + row_of(t), 4 * y + ((lane & 7) >> 1)) + 8 * (lane & 1)) = make_uint2(r[0], r[1]);
            }
            }
          }
        }
        fence_async();
        fence_before();
        bar_arrive(smem_u32(&s.q_full));
      }
      float m = kNone, l = 0.f;
      bool results = false;                                // of an earlier unit of this tile
      const uint32_t step = w.twin ? 2 : 1;                // of this tile's units
      n += w.twin ? x : 0;
      int u = w.u0 + (w.twin ? x : 0);
      // a unit with tokens that keep their own scales: as below, in less code and more time
      const auto by_token = [&](uint32_t scores, int slot, unsigned real, int at) {
        uint32_t raw[32];
        float v[32];
        const auto terms = [&](int h, float base) {
          __syncwarp();
          tmem_load(scores + 32 * h, raw);
          tmem_loaded(raw);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int g = 2 * h + (c >> 4), t = 32 * h + c;
            const bool own = real >> (8 * g) & 2;
            const float ks = own ? own_ks[slot][t] : s.ks[slot][g], lv = own ? own_lv[slot][t] : s.lv[slot][g];
            v[c] = at + t >= row_end || !(real >> (8 * g) & 1) ? kNone : fmaf(__uint_as_float(raw[c]), row_scale * ks, lv - base);
          }
        };
        float top = kNone;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          terms(h, 0.f);
#pragma unroll
          for (int c = 0; c < 32; ++c) top = fmaxf(top, v[c]);
        }
        const bool moves = m == kNone ? top > kNone : top - m > kTop;
        if (__any_sync(kFullWarp, moves)) {
          const float now = moves ? top - kTop : m, f = moves && m != kNone ? exp2_fast(m - now) : 1.f;
          m = now;
          l *= f;
          if (results) {
            ok = __all_sync(kFullWarp, turn(s.pv_done, x, done - 1));
            fence_after();
            if (ok) follow(f);
          }
        }
        const float base = m == kNone ? 0.f : m;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {                      // P goes over scores that have been read: 16 columns of the first 32 each time
          terms(h, base);
          uint32_t p[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const int g = 2 * h + (c >> 4), t = 32 * h + c;
            const bool own = real >> (8 * g) & 2;
            const float y = exp2_fast(v[c]), z = exp2_fast(v[c + 1]);
            l = fmaf(y, own ? own_inv[slot][t] : s.inv[slot][g], fmaf(z, own ? own_inv[slot][t + 1] : s.inv[slot][g], l));
            p[c >> 1] = pack_half(y, z);
          }
          __syncwarp();
          tmem_store(scores + 16 * h, p);
          tmem_stored();
        }
      };
      for (; u < w.u1 && ok; u += step, n += step) {
        // (the scales were there before the keys, the keys before the scores)
        ok = __all_sync(kFullWarp, turn(s.s_full, x, done));
        if (!ok) break;
        fence_after();
        const int at = u * kUnit, slot = n % kScales;
        const uint32_t scores = mine_at + 64 * (done & 1);
        if (warp_has_rows) {
          do {
          uint32_t raw[2][32];
          tmem_load(scores, raw[0]);
          tmem_load(scores + 32, raw[1]);
          const float4 ks = *reinterpret_cast<const float4*>(s.ks[slot]), lv = *reinterpret_cast<const float4*>(s.lv[slot]),
                       inv = *reinterpret_cast<const float4*>(s.inv[slot]);
          const unsigned real = *reinterpret_cast<const unsigned*>(s.real[slot]);
          const float base = m == kNone ? 0.f : m;
          const float by[kGroups] = {row_scale * ks.x, row_scale * ks.y, row_scale * ks.z, row_scale * ks.w};
          const float add[kGroups] = {lv.x - base, lv.y - base, lv.z - base, lv.w - base};
          tmem_loaded(raw[0]);
          tmem_loaded(raw[1]);
          float v[kUnit];
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int c = 16 * g; c < 16 * g + 16; c += 2) fma2(v[c], v[c + 1], raw[c >> 5][c & 31], raw[c >> 5][(c & 31) + 1], by[g], add[g]);
          if (at + kUnit > w.least || real != 0x01010101u) {
            if (kBits == 4 && (real & 0x02020202u)) {      // (asked here, where most units do not come by: before the terms a prompt took 178 us where it takes 176)
              by_token(scores, slot, real, at);
              break;
            }
#pragma unroll
            for (int c = 0; c < kUnit; ++c)
              if (at + c >= row_end || !(real >> (8 * (c >> 4)) & 1)) v[c] = kNone;
          }
          float sum[kGroups][2];
          uint32_t p[kUnit / 2];
          const auto exponentials = [&] {
#pragma unroll
            for (int c = 0; c < kUnit / 2; ++c) {
              const float y = exp2_fast(v[2 * c]), z = exp2_fast(v[2 * c + 1]);
              if (c & 7) add2(sum[c >> 3][0], sum[c >> 3][1], y, z);
              else sum[c >> 3][0] = y, sum[c >> 3][1] = z;
              p[c] = pack_half(y, z);
            }
          };
          const auto store = [&] {
            tmem_store(scores, reinterpret_cast<const uint32_t (&)[16]>(p[0]));
            tmem_store(scores + 16, reinterpret_cast<const uint32_t (&)[16]>(p[16]));
          };
          exponentials();
          if (kBits == 4) {                                // (on its way while it is looked at)
            __syncwarp();
            store();
          }
          // a sum within the range of fp16: so is each of its terms
          const float most = fmaxf(fmaxf(fmaxf(sum[0][0], sum[0][1]), fmaxf(sum[1][0], sum[1][1])), fmaxf(fmaxf(sum[2][0], sum[2][1]), fmaxf(sum[3][0], sum[3][1])));
          const bool grows = m == kNone || most > 60000.f;
          if (__any_sync(kFullWarp, grows)) {              // a new reference, 2^12 above which the largest lies; what there is follows
            float top = kNone;
#pragma unroll
            for (int c = 0; c < kUnit; ++c) top = fmaxf(top, v[c]);
            const bool moves = (grows || (kBits == 4 && top > kTop)) && top > kNone;
            const float now = moves ? base + top - kTop : m, f = moves && m != kNone ? exp2_fast(m - now) : 1.f, down = moves ? base - now : 0.f;
#pragma unroll
            for (int c = 0; c < kUnit; ++c) v[c] += down;
            m = now;
            l *= f;
            if (kBits == 4) exponentials();                // (the last unit's products are under way meanwhile)
            if (results) {
              ok = __all_sync(kFullWarp, turn(s.pv_done, x, done - 1));        // (S of this unit came before the results of the last one)
              fence_after();
              if (ok) follow(f);
            }
            if (kBits == 8) exponentials();
            if (kBits == 4) {
              tmem_stored();
              store();
            }
          }
          l = fmaf(sum[0][0] + sum[0][1], inv.x, fmaf(sum[1][0] + sum[1][1], inv.y, fmaf(sum[2][0] + sum[2][1], inv.z, fmaf(sum[3][0] + sum[3][1], inv.w, l))));
          if (kBits == 8) {
            __syncwarp();
            store();
          }
          tmem_stored();
          } while (false);
        }
        fence_before();
        bar_arrive(smem_u32(&s.p_full[2 * x + (done & 1)]));
        results = true;
        ++done;
      }
      n += w.u1 - u;                                       // (a twin's tiles end one apart)
      if (!ok) break;
      if (results) ok = __all_sync(kFullWarp, turn(s.pv_done, x, done - 1));
      if (!ok) break;
      fence_after();
      // ---- a twin's results are joined by the threads of the first tile, which can read both
      float here = 1.f, there = 0.f;                       // factors of this tile's results and of the other's
      bool other = false;
      if (w.twin) {
        if (x == 1) {
          s.twin_m[row] = m;
          s.twin_l[row] = l;
          fence_before();
          bar_arrive(smem_u32(&s.twin_full));
          ok = __all_sync(kFullWarp, bar_wait(smem_u32(&s.twin_done), twins & 1, fail));
          ++twins;
          fence_after();
          continue;
        }
        ok = __all_sync(kFullWarp, bar_wait(smem_u32(&s.twin_full), twins & 1, fail));
        ++twins;
        if (!ok) break;
        fence_after();
        const float tm = s.twin_m[row], tl = s.twin_l[row], now = fmaxf(m, tm);
        other = w.u1 - w.u0 > 1;
        if (now != kNone) {
          here = exp2_fast(m - now);
          there = exp2_fast(tm - now);
        }
        l = l * here + tl * there;
        m = now;
      }
      // ---- the item, or this run's part of it
      const bool whole = w.u0 == 0 && w.u1 == w.units;
      float* part = a.parts + ((size_t)blockIdx.x * 2 + (segment != 0)) * kPartFloats<D>;
      const bool empty = l == 0.f;                         // a row that sees nothing: zeros
      const float by = whole && !empty ? kSumUnit / l : 1.f;
      const bool nan = *(volatile int*)&s.nan != 0;
      if (warp_has_rows) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          __syncwarp();
          tmem_load(mine_at + 128 + c, o);
          tmem_loaded(o);
          float f[32];
#pragma unroll
          for (int y = 0; y < 32; ++y) f[y] = empty ? 0.f : __uint_as_float(o[y]) * here * by;
          if (other) {
            __syncwarp();
            tmem_load(mine_at + 256 + 128 + c, o);
            tmem_loaded(o);
#pragma unroll
            for (int y = 0; y < 32; ++y) f[y] = empty ? 0.f : fmaf(__uint_as_float(o[y]) * there, by, f[y]);
          }
          if (mine) {
            if (kBits == 8 && nan)                         // values that are NaN were left out of the last units: given to the rows that see them
              for (int token = max(w.least, w.u0 * kUnit); token < min(row_end, w.u1 * kUnit); ++token) {
                const int id = a.tables[w.r * a.table_stride + (token >> a.shift)];
                if (id < 0 || id >= a.pages) continue;
                const uint8_t* v = a.v_cache + ((((size_t)id * a.kv_heads + w.head) << a.shift) + (token & ((1 << a.shift) - 1))) * D + c;
#pragma unroll
                for (int y = 0; y < 32; ++y)
                  if ((v[y] & 0x7F) == 0x7F) f[y] = __int_as_float(0x7FC00000);
              }
            if (whole) {
#pragma unroll
              for (int y = 0; y < 4; ++y)
                *reinterpret_cast<uint4*>(staged(row, c / 8 + y)) = {Half<T>::narrow(f[8 * y], f[8 * y + 1]), Half<T>::narrow(f[8 * y + 2], f[8 * y + 3]),
                                                                     Half<T>::narrow(f[8 * y + 4], f[8 * y + 5]), Half<T>::narrow(f[8 * y + 6], f[8 * y + 7])};
            } else {
#pragma unroll
              for (int y = 0; y < 8; ++y)
                *reinterpret_cast<float4*>(part + ((c / 4 + y) * kRows + place_row) * 4) = make_float4(f[4 * y], f[4 * y + 1], f[4 * y + 2], f[4 * y + 3]);
            }
          }
        }
        if (whole) {                                       // whole lines are written: D / 8 lanes a row
          __syncwarp();
          const long long at = mine ? (long long)place : -1;
#pragma unroll 4
          for (int t = 0; t < D / 8; ++t) {
            const int from = t * (256 / D) + lane / (D / 8), chunk = lane % (D / 8);
            const long long to = __shfl_sync(kFullWarp, at, from);
            const uint4 v = *reinterpret_cast<const uint4*>(staged((row & ~31) + from, chunk));
            if (to >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to + 8 * chunk) = v;
          }
        }
        if (!whole && mine) {
          part[kRows * D + place_row] = m;
          part[kRows * D + kRows + place_row] = l;
        }
      }
      __syncwarp();
      fence_before();
      if (w.twin) bar_arrive(smem_u32(&s.twin_done));
      if (!whole && w.u0 == 0 && tid == 0)                 // it begins here and ends elsewhere: request, item, parts, head and place of the first
        a.cuts[blockIdx.x] = {w.r, w.tile, 1 + (int)((w.units - w.u1 + share - 1) / share), 2 * w.head + (segment != 0)};
    }
    if (lane == 0) s.finished[warp] = segment;
    }
  } else if (kBits == 8 && warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (count > 0) feed(std::false_type{});
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if constexpr (kBits == 4) {
      if (count > 0 && warp != 14) feed4();
    } else {
      if (count > 0 && warp < 14) feed(std::true_type{});
    }
    if (count > 0 && warp == 14) {
    // ================= products: one thread, and as few instructions between two of them as can be (24 a unit, 50 to 60 cycles each to issue)
    if (elect_one()) {
      const uint32_t idesc_s = 1u << 4 | (uint32_t)(kUnit >> 3) << 17 | (128u >> 4) << 24,
                     idesc_o = 1u << 4 | 1u << 16 | ((uint32_t)D >> 3) << 17 | (128u >> 4) << 24;      // (1 << 16: values with the dimensions inside)
      constexpr uint64_t kSwizzle = kBits == 4 || D == 128 ? 2 : 4;
      constexpr int kNextRows = kBits == 4 ? 1024 : 8 * D;
      const uint64_t dq = descriptor(smem_u32(smem + Y::kQ), 16, kNextRows, kSwizzle), dk = descriptor(smem_u32(smem + Y::kK), 16, kNextRows, kSwizzle),
                     dv = descriptor(smem_u32(smem + Y::kV), kUnit * 128, 1024, 2);
      const uint32_t k_full = smem_u32(s.k_full), k_free = smem_u32(s.k_free), v_full = smem_u32(s.v_full), v_free = smem_u32(s.v_free),
                     s_full = smem_u32(s.s_full), p_full = smem_u32(s.p_full), pv_done = smem_u32(s.pv_done), q_full = smem_u32(&s.q_full);
      bool ok = true;
      uint32_t items = 0, qn = 0, pn = 0;                  // items, units of the thread block whose scores and whose results have been issued
      uint32_t qc[2] = {0, 0}, pc[2] = {0, 0};             // the same of the tiles
      const auto scores_of = [&](auto tile) {
        constexpr int x = decltype(tile)::value;
        // over the P of two units before: products of another kind are not kept in order by themselves
        if (qc[x] >= 2 && !bar_wait(pv_done + 16 * x + 8 * (qc[x] & 1), (qc[x] - 2) >> 1 & 1, fail)) return false;
        fence_after();
        const uint64_t k = dk + (qn % kRing) * (Y::kKeys >> 4);
        const uint32_t to = tmem + 256 * x + 64 * (qc[x] & 1);
        if constexpr (kBits == 4) {
#pragma unroll
          for (int y = 0; y < D / 16; ++y)
            mma_ss_f16(to, dq + (x * Y::kQTile + (y >> 2) * (kTile * 128) >> 4) + 2 * (y & 3), k + ((y >> 2) * (kUnit * 128) >> 4) + 2 * (y & 3), idesc_s, y != 0);
        } else
#pragma unroll
        for (int part = 0; part < Y::kParts; ++part)
#pragma unroll
          for (int y = 0; y < D / 32; ++y)
            mma_ss(to, dq + (x * Y::kQTile + part * Y::kPart >> 4) + 2 * y, k + 2 * y, idesc_s, (part | y) != 0);
        commit(s_full + 16 * x + 8 * (qc[x] & 1));
        ++qc[x];
        return true;
      };
      const auto results_of = [&](auto tile, uint32_t fresh) {
        constexpr int x = decltype(tile)::value;
        if (!bar_wait(p_full + 16 * x + 8 * (pc[x] & 1), pc[x] >> 1 & 1, fail)) return false;
        fence_after();
        const uint64_t v = dv + (pn % kRing) * (Y::kValues >> 4);
        const uint32_t from = tmem + 256 * x + 64 * (pc[x] & 1);
#pragma unroll
        for (int y = 0; y < kUnit / 16; ++y) mma_ts(tmem + 256 * x + 128, from + 8 * y, v + y * (2048 >> 4), idesc_o, y != 0 ? 1u : fresh);
        commit(pv_done + 16 * x + 8 * (pc[x] & 1));
        ++pc[x];
        return true;
      };
      Walk w(s, count);
      for (; w.left > 0 && ok; w.next(a)) {
        w.look(a);
        ok = bar_wait(q_full, items++ & 1, fail);
        const int units = w.u1 - w.u0, ahead = w.twin ? 4 : 2;
        // scores of unit i of the item come `ahead` places before the results of the unit that is that far behind
        for (int i = 1 - ahead; i < units && ok; ++i) {
          const int j = i + ahead - 1;
          if (j < units) {
            if (!(ok = bar_wait(k_full + 8 * (qn % kRing), qn / kRing & 1, fail))) break;
            fence_after();
            if (!w.twin || !(j & 1)) ok = scores_of(std::integral_constant<int, 0>{});
            if (ok && (!w.twin || (j & 1))) ok = scores_of(std::integral_constant<int, 1>{});
            if (!ok) break;
            commit(k_free + 8 * (qn % kRing));
            ++qn;
          }
          if (i < 0) continue;
          if (!(ok = bar_wait(v_full + 8 * (pn % kRing), pn / kRing & 1, fail))) break;
          const uint32_t fresh = i >= (w.twin ? 2 : 1);    // 0: the tile's first unit of this item
          if (!w.twin || !(i & 1)) ok = results_of(std::integral_constant<int, 0>{}, fresh);
          if (ok && (!w.twin || (i & 1))) ok = results_of(std::integral_constant<int, 1>{}, fresh);
          commit(v_free + 8 * (pn % kRing));
          ++pn;
        }
      }
      // products in flight end before the tensor memory goes back
      commit(smem_u32(&s.drained));
      for (unsigned i = 0; i < kSpinLimit && !bar_try(smem_u32(&s.drained), 0); ++i) {}
    }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (s.fail && warp < 8) {                                // a wait ran out: rows that are not finished become NaN (of parts: by way of the sum)
    // (the run once more, after all else: inside the loop over its items this costs the softmax registers, 197 us in place of 176 at the sizes above)
    const int x = warp >> 2, row = tid & (kTile - 1);
    const long long all = *(volatile long long*)&s.total, share = max((all + gridDim.x - 1) / gridDim.x, 1LL);
    Walk w(s, min(share, all - blockIdx.x * share));
    for (int segment = 0; w.left > 0; ++segment, w.next(a)) {
      w.look(a);
      if (segment < s.finished[warp]) continue;
      const int place_row = w.twin ? row : x * kTile + row;
      const bool whole = w.u0 == 0 && w.u1 == w.units;
      if (!(w.twin && x) && place_row < w.rows) {
        if (whole) {
          const int i = place_row / a.group, head = w.head * a.group + place_row - i * a.group;
          T* dst = static_cast<T*>(a.out) + ((size_t)(w.start + w.tile * w.per + i) * a.q_heads + head) * D;
          for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(dst + c) = {0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu};
        } else {
          float* part = a.parts + ((size_t)blockIdx.x * 2 + (segment != 0)) * kPartFloats<D>;
          part[kRows * D + place_row] = 0.f;
          part[kRows * D + kRows + place_row] = __int_as_float(0x7FC00000);
        }
      }
      if (!whole && w.u0 == 0 && tid == 0)
        a.cuts[blockIdx.x] = {w.r, w.tile, 1 + (int)((w.units - w.u1 + share - 1) / share), 2 * w.head + (segment != 0)};
    }
    if (tid == 0 && a.status) atomicOr(a.status, 64);
  }
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemColumns) : "memory");
  }
}

// Joins the parts of the tiles that were cut: kJoins thread blocks per run of the launch before, a thread per row and four dimensions (a prompt's items have
// two parts as a rule: batches of eight cost it 3 us, and of four 1).
template <typename T, int D>
__global__ void __launch_bounds__(512) paged_attention_tc_join_kernel(const AttentionArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.z == 0) return;
  const Request x(a, cut.x);
  const int kvh = cut.w >> 1, rows = x.tokens(a, cut.y) * a.group;
  const float *head = a.parts + ((size_t)blockIdx.x * 2 + (cut.w & 1)) * kPartFloats<D>, *tail = a.parts + (size_t)blockIdx.x * 2 * kPartFloats<D>;
  for (int z = blockIdx.y * 512 + threadIdx.x; z < kRows * (D / 4); z += kJoins<D> * 512) {
    const int row = z % kRows, d = z / kRows;
    if (row >= rows) continue;
    float m = head[kRows * D + row], l = head[kRows * D + kRows + row];
    float4 y = *reinterpret_cast<const float4*>(head + (d * kRows + row) * 4);
    const auto part = [&](int i) { return tail + (size_t)i * 2 * kPartFloats<D>; };
    join_parts<4>(cut.z, m, l, y, [&](int i) { return part(i) + kRows * D + row; }, [&](int i) { return part(i) + kRows * D + kRows + row; },
               [&](int i) { return reinterpret_cast<const float4*>(part(i) + (d * kRows + row) * 4); });
    const float by = l == 0.f ? 0.f : kSumUnit / l;
    const int i = row / a.group;
    T* dst = static_cast<T*>(a.out) + ((size_t)(x.start + cut.y * x.per + i) * a.q_heads + (size_t)kvh * a.group + row - i * a.group) * D + 4 * d;
    *reinterpret_cast<uint2*>(dst) = {Half<T>::narrow(y.x * by, y.y * by), Half<T>::narrow(y.z * by, y.w * by)};
  }
}

template <typename T, int D, int kBits>
int run(const AttentionArgs& a, cudaStream_t st) {
  constexpr int kBytes = Layout<T, D, kBits>::kBytes;
  static bool allowed[64] = {false};                       // shared memory beyond 48 KB: opted in once per device
  int dev = 0, e = (int)cudaGetDevice(&dev);
  if (!e && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = (int)cudaFuncSetAttribute(paged_attention_tc_kernel<T, D, kBits>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (!e && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  if (e) return paged_fail(e);
  const dim3 grid(current_device_sms());
  const int rc = paged_launch(paged_attention_tc_kernel<T, D, kBits>, grid, dim3(kThreads), 1, kBytes, st, a);
  return rc != HTR_OK ? rc : paged_launch(paged_attention_tc_join_kernel<T, D>, dim3(grid.x, kJoins<D>), dim3(512), 1, 0, st, a);
}

template <int kBits>
int run_of(const AttentionArgs& args, int dtype, int head_dim, void* workspace, cudaStream_t st) {
  AttentionArgs a = args;
  a.cuts = static_cast<int4*>(workspace);
  a.parts = reinterpret_cast<float*>(a.cuts + current_device_sms());
  if (dtype == HTR_DTYPE_BF16) return head_dim == 128 ? run<__nv_bfloat16, 128, kBits>(a, st) : run<__nv_bfloat16, 64, kBits>(a, st);
  return head_dim == 128 ? run<__half, 128, kBits>(a, st) : run<__half, 64, kBits>(a, st);
}

}  // namespace
