// Rotary positions from a prepared table of frequencies: part of a head or all of it, both pairings, any scaling of the frequencies.
//
//   angle = position * f_j     x_a' = (x_a cos - x_b sin) * magnitude     x_b' = (x_b cos + x_a sin) * magnitude
//
// for the pairs (a, b) = (j, R/2 + j) or (2j, 2j + 1) of the first R values of a head; the others are copied.
//
// Bound by HBM once a launch is large: a value is read and written once, 8 bytes; 4096 positions of 72 heads of 128 (302 MB) take 53.7 us =
// 5630 GB/s (a copy: 6555), a decode step of 32 positions is a launch, 3.5 us. What stands in the way of that is the angle of far
// positions, which f32 does not hold: position * f_j is taken in f64, in half turns (the table holds f_j / pi), reduced there
// to [-1, 1] by whole turns, and only the rest goes through the f32 sine and cosine, its own rounding added back to first order. That
// is six f64 instructions per angle where a sine and cosine in f64 are some hundred. A thread keeps four neighbouring pairs and
// their angles and walks the heads of one position, so that an angle serves every head a thread has; loads are 16 bytes, those of
// four heads at a time.
#include <algorithm>
#include <type_traits>

#include "chain.cuh"
#include "kernels.h"

namespace etc {

namespace {

constexpr int kThreads = 256;
constexpr int kHeadsAhead = 4;  // heads whose loads are in flight together

// Heads are cut into units of 2 VEC values in two pieces, each on a boundary of its size: VEC pairs that are rotated, or values behind them
// that are copied. VEC is 4 where a head's parts and the addresses allow, else 2, else 1 (the last unit may then be a single value).
template <int VEC, bool HALVES>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a) {
  using Piece = std::conditional_t<VEC == 4, float4, std::conditional_t<VEC == 2, float2, float>>;
  chain_release();
  chain_wait();
  const int64_t row = blockIdx.x;
  const int64_t b = row / a.steps, step = row - b * a.steps;
  const int rotated = a.rotary_half / VEC, units = rotated + (a.head_dim - 2 * a.rotary_half + 2 * VEC - 1) / (2 * VEC);
  const int width = min(units, kThreads), at_once = kThreads / width;  // units side by side, heads side by side
  const int u0 = threadIdx.x % width, h0 = blockIdx.y * at_once + threadIdx.x / width, h_step = gridDim.y * at_once;
  if (threadIdx.x >= width * at_once) return;
  const double position = (double)(a.offsets[a.n_offsets == 1 ? 0 : b] + step);
  const float* x = a.x + b * a.x_stride[0] + step * a.x_stride[2];
  float* out = a.out + b * a.out_stride[0] + step * a.out_stride[2];
  for (int u = u0; u < units; u += width) {
    const bool turns = u < rotated;
    if (!turns && a.in_place) continue;
    // where the two pieces start: the first and the second values of the pairs, or one behind the other
    const int first = turns ? (HALVES ? u * VEC : 2 * u * VEC) : 2 * (a.rotary_half + (u - rotated) * VEC);
    const int second = turns && HALVES ? a.rotary_half + u * VEC : first + VEC;
    const bool both = VEC > 1 || second < a.head_dim;
    float cosine[VEC], sine[VEC];
    if (turns) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        double turn = position * a.half_turns[u * VEC + i];
        turn -= 2.0 * rint(0.5 * turn);
        const float near = (float)turn, rest = (float)(turn - (double)near) * 3.14159265f;
        float s, c;
        sincospif(near, &s, &c);
        cosine[i] = fmaf(-s, rest, c) * a.magnitude;
        sine[i] = fmaf(c, rest, s) * a.magnitude;
      }
    }
    for (int hb = h0; hb < a.heads; hb += kHeadsAhead * h_step) {
      float p[kHeadsAhead][2 * VEC];
#pragma unroll
      for (int k = 0; k < kHeadsAhead; ++k) {
        const int h = hb + k * h_step;
        if (h >= a.heads) break;
        const float* src = x + h * a.x_stride[1];
        *reinterpret_cast<Piece*>(p[k]) = *reinterpret_cast<const Piece*>(src + first);
        if (both) *reinterpret_cast<Piece*>(p[k] + VEC) = *reinterpret_cast<const Piece*>(src + second);
      }
#pragma unroll
      for (int k = 0; k < kHeadsAhead; ++k) {
        const int h = hb + k * h_step;
        if (h >= a.heads) break;
        if (turns) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float &va = p[k][HALVES ? i : 2 * i], &vb = p[k][HALVES ? VEC + i : 2 * i + 1];
            const float ra = va * cosine[i] - vb * sine[i], rb = vb * cosine[i] + va * sine[i];
            va = ra;
            vb = rb;
          }
        }
        float* dst = out + h * a.out_stride[1];
        *reinterpret_cast<Piece*>(dst + first) = *reinterpret_cast<const Piece*>(p[k]);
        if (both) *reinterpret_cast<Piece*>(dst + second) = *reinterpret_cast<const Piece*>(p[k] + VEC);
      }
    }
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& args, int64_t batch, int sm_count, cudaStream_t stream) {
  RotaryArgs a = args;
  const int64_t rows = batch * a.steps;
  if (rows == 0 || a.heads == 0) return cudaSuccess;
  auto allows = [&](int vec) {
    bool ok = a.rotary_half % vec == 0 && (vec == 1 || a.head_dim % (2 * vec) == 0) && ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & (4 * vec - 1)) == 0;
    for (int i = 0; i < 3; ++i) ok = ok && a.x_stride[i] % vec == 0 && a.out_stride[i] % vec == 0;
    return ok;
  };
  const int vec = allows(4) ? 4 : allows(2) ? 2 : 1, units = a.rotary_half / vec + (a.head_dim - 2 * a.rotary_half + 2 * vec - 1) / (2 * vec);
  const int at_once = kThreads / std::min(units, kThreads);
  // few positions: their heads go to several CTAs, until there are four for every SM
  const int64_t most = (a.heads + at_once - 1) / at_once, wanted = (4 * sm_count + rows - 1) / rows;
  const dim3 grid((unsigned)rows, (unsigned)std::min<int64_t>(std::min(most, wanted), 65535));
  auto launch = [&](auto kernel) { return launch_chained(kernel, grid, dim3(kThreads), 0, stream, a); };
  if (a.layout == 0) return vec == 4 ? launch(rotary_kernel<4, true>) : vec == 2 ? launch(rotary_kernel<2, true>) : launch(rotary_kernel<1, true>);
  return vec == 4 ? launch(rotary_kernel<4, false>) : vec == 2 ? launch(rotary_kernel<2, false>) : launch(rotary_kernel<1, false>);
}

}  // namespace etc
