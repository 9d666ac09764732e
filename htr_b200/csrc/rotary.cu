// Cosines and sines of the positions of a rotary embedding, for contexts where a float32 angle has no bits left behind the point.
#include <cmath>

#include "paged_common.cuh"

namespace {

using namespace htr;

constexpr int kMostPairs = 128, kThreads = 256, kFirsts = 16;

struct AnglesArgs {
  double half_turns[kMostPairs];                           // of each pair, per position
  long long first;
  int rows, pairs;
  float magnitude;
  float *cosv, *sinv;
};

// Cosine and sine of position * frequency.  The product and what is left of it after whole turns are taken in 64 bits; the sine and cosine of that by sincospif of
// the float32 nearest to it, and what this leaves over to first order: sin(x + e) = sin x + e cos x.
__device__ __forceinline__ float2 turned(double position, double half_turns) {
  const double t = position * half_turns, r = t - 2.0 * rint(0.5 * t);             // half turns, -1 to 1
  const float x = (float)r, e = (float)(r - (double)x) * 3.14159265f;
  float s, c;
  sincospif(x, &s, &c);
  return make_float2(fmaf(-s, e, c), fmaf(c, e, s));
}

template <int V>
__device__ __forceinline__ void put(const AnglesArgs& a, size_t at, const float2 (&z)[V]) {
  if constexpr (V == 4) {
    *reinterpret_cast<float4*>(a.cosv + at) = make_float4(z[0].x, z[1].x, z[2].x, z[3].x);
    *reinterpret_cast<float4*>(a.sinv + at) = make_float4(z[0].y, z[1].y, z[2].y, z[3].y);
  } else {
    a.cosv[at] = z[0].x;
    a.sinv[at] = z[0].y;
  }
}

// Few rows: a thread has V neighbouring pairs of one position.  Bound by latency.
template <int V>
__global__ void __launch_bounds__(kThreads) rope_angles_kernel(const __grid_constant__ AnglesArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ double s_freq[kMostPairs];                    // (lanes that index the arguments each for itself read them one after the other)
  if (threadIdx.x < a.pairs) s_freq[threadIdx.x] = a.half_turns[threadIdx.x];
  __syncthreads();
  const int groups = a.pairs / V;
  const long long n = (long long)blockIdx.x * kThreads + threadIdx.x, row = n / groups;
  const int group = (int)(n - row * groups);
  if (row >= a.rows) return;
  float2 z[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    z[v] = turned((double)(a.first + row), s_freq[group * V + v]);
    z[v].x *= a.magnitude;
    z[v].y *= a.magnitude;
  }
  put<V>(a, (size_t)row * a.pairs + group * V, z);
}

// Many rows: 2 * deep of them are a strip (deep: rows that the threads of a block hold at a time).  A thread keeps the angles of its two places in a strip, times
// magnitude, in registers; those of the strips' first rows are laid out in shared memory, kFirsts at a time; and the others are products of the two, float32 of
// numbers each off by a step or so.  What is left is bound by the bytes written: evaluating every angle took 36 us for 262144 rows of 64 pairs (134 MB), this 22.
template <int V>
__global__ void __launch_bounds__(kThreads) rope_angles_rows_kernel(const __grid_constant__ AnglesArgs a) {
  __shared__ double s_freq[kMostPairs];                    // (lanes that index the arguments each for itself read them one after the other)
  __shared__ __align__(16) float first_c[kFirsts * kMostPairs], first_s[kFirsts * kMostPairs];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int groups = a.pairs / V, deep = kThreads / groups, tid = threadIdx.x, group = tid % groups, y = tid / groups;
  if (tid < a.pairs) s_freq[tid] = a.half_turns[tid];
  __syncthreads();
  const bool works = y < deep;
  float2 w[2][V];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      w[h][v] = turned((double)(y + h * deep), s_freq[group * V + v]);
      w[h][v].x *= a.magnitude;
      w[h][v].y *= a.magnitude;
    }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long step = (long long)gridDim.x * 2 * deep;
  for (long long row0 = (long long)blockIdx.x * 2 * deep; row0 < a.rows; row0 += kFirsts * step) {
    const int count = (int)min((long long)kFirsts, (a.rows - row0 + step - 1) / step);
    __syncthreads();                                       // the last ones have been read
    if (works)
      for (int i = y; i < count; i += deep)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 z = turned((double)(a.first + row0) + (double)(i * step), s_freq[group * V + v]);
          first_c[i * a.pairs + group * V + v] = z.x;
          first_s[i * a.pairs + group * V + v] = z.y;
        }
    __syncthreads();
    if (!works) continue;
    size_t at = (size_t)(row0 + y) * a.pairs + group * V;
    for (int k = 0; k < count; ++k, at += (size_t)step * a.pairs) {
      float zc[V], zs[V];
      if constexpr (V == 4) {
        const float4 c = *reinterpret_cast<const float4*>(first_c + k * a.pairs + group * V), s = *reinterpret_cast<const float4*>(first_s + k * a.pairs + group * V);
        zc[0] = c.x; zc[1] = c.y; zc[2] = c.z; zc[3] = c.w;
        zs[0] = s.x; zs[1] = s.y; zs[2] = s.z; zs[3] = s.w;
      } else {
        zc[0] = first_c[k * a.pairs + group];
        zs[0] = first_s[k * a.pairs + group];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row0 + k * step + y + h * deep >= a.rows) continue;
        float2 r[V];
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = make_float2(fmaf(zc[v], w[h][v].x, -zs[v] * w[h][v].y), fmaf(zc[v], w[h][v].y, zs[v] * w[h][v].x));
        put<V>(a, at + (size_t)h * deep * a.pairs, r);
      }
    }
  }
}

template <int V>
int run(const AnglesArgs& a, cudaStream_t st) {
  const long long groups = a.pairs / V;
  if (a.rows < 64 * current_device_sms()) return paged_launch(rope_angles_kernel<V>, dim3((unsigned)((a.rows * groups + kThreads - 1) / kThreads)), dim3(kThreads), 1, 0, st, a);
  const long long strip = 2 * (kThreads / groups), strips = (a.rows + strip - 1) / strip, most = 6LL * current_device_sms();
  return paged_launch(rope_angles_rows_kernel<V>, dim3((unsigned)(strips < most ? strips : most)), dim3(kThreads), 1, 0, st, a);
}

}  // namespace

extern "C" int htr_rope_angles(int64_t first, int rows, int dim, double theta, double factor, double original, double low, double high, float magnitude,
                               float* cosv, float* sinv, htr_stream_t stream) {
  if (rows < 0 || first < 0 || dim < 2 || dim % 2 || !(theta > 0) || !(factor > 0) || !(original >= 0) || !(low < high) || !std::isfinite(theta) ||
      !std::isfinite(factor) || !std::isfinite(original) || !std::isfinite(low) || !std::isfinite(high))
    return HTR_ERR_BAD_SHAPE;
  if (dim > 2 * kMostPairs || first > 0x7FFFFFFF || first + rows > 0x7FFFFFFF) return HTR_ERR_TOO_LARGE;
  if (rows == 0) return HTR_OK;
  if (!cosv || !sinv) return HTR_ERR_NULL;
  constexpr double kPi = 3.14159265358979323846;
  AnglesArgs a;
  a.first = first;
  a.rows = rows;
  a.pairs = dim / 2;
  a.magnitude = magnitude;
  a.cosv = cosv;
  a.sinv = sinv;
  for (int i = 0; i < a.pairs; ++i) {
    const double f = std::pow(theta, -2.0 * i / dim);      // radians
    // share of the frequency that stays: none below `low` turns within `original` positions, all from `high` on
    double keep = 0;
    if (original > 0) keep = std::fmin(std::fmax((original * f / (2 * kPi) - low) / (high - low), 0.0), 1.0);
    a.half_turns[i] = f / kPi * (keep + (1 - keep) / factor);
  }
  const bool four = a.pairs % 4 == 0 && ((reinterpret_cast<uintptr_t>(cosv) | reinterpret_cast<uintptr_t>(sinv)) & 15u) == 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return four ? run<4>(a, st) : run<1>(a, st);
}
