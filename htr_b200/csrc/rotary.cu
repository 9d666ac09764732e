// Cosines and sines of the positions of a rotary embedding, for contexts where a float32 angle has no bits left behind the point.
#include <cmath>

#include "paged_common.cuh"

namespace {

using namespace htr;

constexpr int kMostPairs = 128, kThreads = 256, kRows = 8;

struct AnglesArgs {
  double half_turns[kMostPairs];                           // of each pair, per position
  long long first;
  int rows, pairs;
  float magnitude;
  float *cosv, *sinv;
};

// What bounds it: the bytes written, as long as 64-bit arithmetic stays short.  The product position * frequency and what is left of it after whole turns are
// taken in 64 bits; its sine and cosine by sincospif of the float32 nearest to that, and what this leaves over to first order: sin(x + e) = sin x + e cos x.
// A thread has V neighbouring pairs, whose frequencies stay in registers, and kRows positions.
template <int V>
__global__ void __launch_bounds__(kThreads) rope_angles_kernel(const __grid_constant__ AnglesArgs a) {
  __shared__ double s_freq[kMostPairs];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int groups = a.pairs / V, deep = kThreads / groups, tid = threadIdx.x;
  if (tid < a.pairs) s_freq[tid] = a.half_turns[tid];
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int group = tid % groups, y = tid / groups;
  if (y >= deep) return;
  double f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = s_freq[group * V + v];
  for (int i = 0; i < kRows; ++i) {
    const long long row = ((long long)blockIdx.x * kRows + i) * deep + y;
    if (row >= a.rows) break;
    const double p = (double)(a.first + row);
    float c[V], s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const double t = p * f[v], r = t - 2.0 * rint(0.5 * t);          // half turns, -1 to 1
      const float x = (float)r, e = (float)(r - (double)x) * 3.14159265f;
      float sx, cx;
      sincospif(x, &sx, &cx);
      c[v] = fmaf(-sx, e, cx) * a.magnitude;
      s[v] = fmaf(cx, e, sx) * a.magnitude;
    }
    const size_t at = (size_t)row * a.pairs + group * V;
    if constexpr (V == 4) {
      *reinterpret_cast<float4*>(a.cosv + at) = make_float4(c[0], c[1], c[2], c[3]);
      *reinterpret_cast<float4*>(a.sinv + at) = make_float4(s[0], s[1], s[2], s[3]);
    } else {
      a.cosv[at] = c[0];
      a.sinv[at] = s[0];
    }
  }
}

}  // namespace

extern "C" int htr_rope_angles(int64_t first, int rows, int dim, double theta, double factor, double original, double low, double high, float magnitude,
                               float* cosv, float* sinv, htr_stream_t stream) {
  if (rows < 0 || first < 0 || dim < 2 || dim % 2 || !(theta > 0) || !(factor > 0) || !(original >= 0) || !(low < high) || !std::isfinite(theta) ||
      !std::isfinite(factor) || !std::isfinite(original) || !std::isfinite(low) || !std::isfinite(high))
    return HTR_ERR_BAD_SHAPE;
  if (dim > 2 * kMostPairs || first + rows > 0x7FFFFFFF || first > 0x7FFFFFFF) return HTR_ERR_TOO_LARGE;
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
  const int deep = kThreads / (a.pairs / (four ? 4 : 1));
  const dim3 grid((unsigned)((rows + (long long)deep * kRows - 1) / ((long long)deep * kRows)));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return four ? paged_launch(rope_angles_kernel<4>, grid, dim3(kThreads), 1, 0, st, a) : paged_launch(rope_angles_kernel<1>, grid, dim3(kThreads), 1, 0, st, a);
}
