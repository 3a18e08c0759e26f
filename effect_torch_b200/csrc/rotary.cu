// Rotary positions from a prepared table of frequencies: part of a head or all of it, both pairings, any scaling of the frequencies.
//
//   angle = position * f_j     x_a' = (x_a cos - x_b sin) * magnitude     x_b' = (x_b cos + x_a sin) * magnitude
//
// for the pairs (a, b) = (j, R/2 + j) or (2j, 2j + 1) of the first R values of a head; the others are copied.
//
// Bound by HBM once a launch is large: a value is read and written once, 8 bytes; 4096 positions of 72 heads of 128 (302 MB) take 52.4 us =
// 5760 GB/s (a copy: 6555), a decode step of 32 positions is a launch, 3.5 us. What stands in the way of that is the angle of far
// positions, which f32 does not hold: position * f_j is taken in f64, in half turns (the table holds f_j / pi), reduced there
// to [-1, 1] by whole turns, and only the rest goes through the f32 sine and cosine, its own rounding added back to first order. That
// is six f64 instructions per angle where a sine and cosine in f64 are some hundred. A CTA works its angles out once, in shared memory,
// while its first loads are on their way, and its threads then walk the heads by 16-byte pieces, five rows' loads at a time. With
// few heads it takes several positions, so that there is an angle for every thread and five rows of them: 8192 positions of 20 heads
// of 64 take 16.5 us against 39 with each thread working out its own, 4096 of 8 heads of 128 9.5 against 20.
#include <algorithm>
#include <type_traits>

#include "chain.cuh"
#include "kernels.h"

namespace etc {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 5;          // rows whose loads are in flight together (four: 55.9 us for 4096 positions of 72 heads)
constexpr int kMostPositions = 16; // of a CTA
constexpr int kFewHeads = 4096;    // with fewer a CTA may take several positions: row / heads by f32 is exact

// A row is one position's values of one head, cut into units of 2 VEC values in two pieces, each on a boundary of its size: VEC pairs that are
// rotated, or values behind them that are copied. VEC is 4 where a head's parts and the addresses allow, else 2, else 1 (the last unit may
// then be a single value). Grid: (groups of `positions` positions, shares of their rows, groups of kThreads units).
template <int VEC, bool HALVES>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, int rows, int positions) {
  using Piece = std::conditional_t<VEC == 4, float4, std::conditional_t<VEC == 2, float2, float>>;
  __shared__ __align__(16) float2 turns_of[kThreads * VEC];  // [position][pair of these units]: cosine and sine
  chain_release();
  chain_wait();
  const int rotated = a.rotary_half / VEC, units = rotated + (a.head_dim - 2 * a.rotary_half + 2 * VEC - 1) / (2 * VEC);
  const int width = min(units, kThreads), at_once = kThreads / width;  // units side by side, rows side by side
  const int unit0 = blockIdx.z * kThreads, u = unit0 + threadIdx.x % width, pairs = max(min(rotated - unit0, width), 0) * VEC;
  const int row0 = blockIdx.x * positions, here = min(positions, rows - row0), b0 = row0 / a.steps, step0 = row0 - b0 * a.steps;
  const bool turns = u < rotated, idle = threadIdx.x >= width * at_once || u >= units || (!turns && a.in_place);
  // where the two pieces start: the first and the second values of the pairs, or one behind the other
  const int first = turns ? (HALVES ? u * VEC : 2 * u * VEC) : 2 * (a.rotary_half + (u - rotated) * VEC);
  const int second = turns && HALVES ? a.rotary_half + u * VEC : first + VEC;
  const bool both = VEC > 1 || second < a.head_dim;
  const float per_steps = 1.0f / (float)a.steps, per_heads = 1.0f / (float)a.heads;
  // batch entry and step of the CTA's position p
  auto entry_of = [&](int p, int& b, int& step) {
    b = b0;
    step = step0 + p;
    if (step >= a.steps) {
      const int over = a.steps >= kMostPositions ? 1 : (int)(((float)step + 0.5f) * per_steps);
      b += over;
      step -= over * a.steps;
    }
  };
  const int count = idle ? 0 : here * a.heads, stride = gridDim.y * at_once;
  auto place = [&](int r, int& p, int& h, int& b, int& step) {
    p = positions == 1 ? 0 : (int)(((float)r + 0.5f) * per_heads);
    h = r - p * a.heads;
    entry_of(p, b, step);
  };
  float x[kAhead][2 * VEC];
  auto load = [&](int from) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = from + k * stride;
      if (r >= count) break;
      int p, h, b, step;
      place(r, p, h, b, step);
      const float* src = a.x + b * a.x_stride[0] + h * a.x_stride[1] + step * a.x_stride[2];
      *reinterpret_cast<Piece*>(x[k]) = *reinterpret_cast<const Piece*>(src + first);
      if (both) *reinterpret_cast<Piece*>(x[k] + VEC) = *reinterpret_cast<const Piece*>(src + second);
    }
  };
  int from = blockIdx.y * at_once + threadIdx.x / width;
  load(from);
  for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
    const int p = i / pairs;
    int b, step;
    entry_of(p, b, step);
    double turn = (double)(a.offsets[a.n_offsets == 1 ? 0 : b] + step) * a.half_turns[unit0 * VEC + i - p * pairs];
    turn -= 2.0 * rint(0.5 * turn);
    const float near = (float)turn, rest = (float)(turn - (double)near) * 3.14159265f;
    float s, c;
    sincospif(near, &s, &c);
    turns_of[i] = make_float2(fmaf(-s, rest, c) * a.magnitude, fmaf(c, rest, s) * a.magnitude);
  }
  __syncthreads();
  while (from < count) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = from + k * stride;
      if (r >= count) break;
      int p, h, b, step;
      place(r, p, h, b, step);
      if (turns) {
        __align__(16) float2 turn[VEC];
        const float2* kept = turns_of + p * pairs + (u - unit0) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          if constexpr (VEC > 1) *reinterpret_cast<float4*>(turn + i) = *reinterpret_cast<const float4*>(kept + i);
          else turn[i] = kept[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float &va = x[k][HALVES ? i : 2 * i], &vb = x[k][HALVES ? VEC + i : 2 * i + 1];
          const float ra = va * turn[i].x - vb * turn[i].y, rb = vb * turn[i].x + va * turn[i].y;
          va = ra;
          vb = rb;
        }
      }
      float* dst = a.out + b * a.out_stride[0] + h * a.out_stride[1] + step * a.out_stride[2];
      *reinterpret_cast<Piece*>(dst + first) = *reinterpret_cast<const Piece*>(x[k]);
      if (both) *reinterpret_cast<Piece*>(dst + second) = *reinterpret_cast<const Piece*>(x[k] + VEC);
    }
    from += kAhead * stride;
    load(from);
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
  const int width = std::min(units, kThreads), at_once = kThreads / width, pairs = std::max(std::min(a.rotary_half / vec, kThreads) * vec, 1);
  // as many positions as give every thread an angle, but no more rows than are loaded at once, as long as there are four CTAs for every SM
  int64_t positions = a.heads < kFewHeads ? std::min<int64_t>(std::min({std::max(kThreads / pairs, 1), kMostPositions, (kAhead * at_once + a.heads - 1) / a.heads}), std::max<int64_t>(rows / (4 * sm_count), 1)) : 1;
  // few positions: their heads go to several CTAs, until there are four for every SM
  const int64_t groups = (rows + positions - 1) / positions, most = (a.heads + at_once - 1) / at_once, wanted = (4 * sm_count + groups - 1) / groups;
  const dim3 grid((unsigned)groups, (unsigned)std::min<int64_t>(std::min(most, wanted), 65535), (unsigned)((units + kThreads - 1) / kThreads));
  auto launch = [&](auto kernel) { return launch_chained(kernel, grid, dim3(kThreads), 0, stream, a, (int)rows, (int)positions); };
  if (a.layout == 0) return vec == 4 ? launch(rotary_kernel<4, true>) : vec == 2 ? launch(rotary_kernel<2, true>) : launch(rotary_kernel<1, true>);
  return vec == 4 ? launch(rotary_kernel<4, false>) : vec == 2 ? launch(rotary_kernel<2, false>) : launch(rotary_kernel<1, false>);
}

}  // namespace etc
