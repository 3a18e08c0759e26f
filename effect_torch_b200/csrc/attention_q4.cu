// Decode attention over pages held in 4 bits (kv_q4.cuh): one query token per lane, 16-token pages, head dim 64 or 128, and results as
// close to the stored values as f32 arithmetic comes.
//
// Mathematics. With codes c (whole numbers -8 .. 7) and a scale per row and block of 32 columns,
//   s[tok] = scale * sum_b dk[tok][b] * (sum_{d in b} q[d] ck[tok][d])      o[d] = sum_tok p[tok] dv[tok][b(d)] cv[tok][d] / sum_tok p[tok]
// so codes go through mma.sync.m16n8k16 as exact f16 numbers, a block of columns at a time, and scales are applied in f32: to the
// sums of a block (K), to the weights ahead of the product (V). What f16 would round, q and p * dv, is split in two f16 numbers, value and rest
// (22 bits together), after scaling by powers of two that keep the rest out of the subnormals; the products of both are added in f32.
// Nothing else is below f32.
//
// Layout. Tokens are the rows of the first product and the columns of the second: S^T = K Q^T and O^T = V^T P^T. A group of four query
// heads fills the eight columns of a tile with (value, rest) pairs, so the split costs no instructions of the tensor pipe as long as
// four heads or fewer would leave columns empty anyway, and a thread's accumulators hold both parts of one head's scores, which it adds. A code
// page is read from shared memory as it was stored: 16 bytes of a K row per thread are its operands of all eight steps, 8
// bytes of a V row its operands of all eight tiles; two codes are widened by one mask and one f16 operation.
//
// Work. The pages of all (lane, KV head) units in a row are cut into as many equal runs as there are CTAs, whatever the lengths of the
// lanes: no CTA waits for the longest. Warps take a run's pages in turn through a ring of cp.async copies that runs on across the
// units. A unit within one run is finished there; the parts of one that is cut go to scratch (two per CTA at most) and a second kernel
// adds them up. Short tables (kDirectPages) take one CTA per unit and no second kernel.
//
// Scores are compared with a reference that is raised, with everything accumulated, only when one exceeds it by 2^kSlack: a few times per
// run instead of once per page.
#include <cuda_fp16.h>

#include <algorithm>

#include "activation.cuh"
#include "chain.cuh"
#include "kernels.h"
#include "kv_q4.cuh"

namespace etc {

namespace {

constexpr int kPage = 16;
constexpr int kStages = 3;
constexpr int kDirectPages = 16;
constexpr float kSlack = 6.0f;
constexpr int kWeightBits = 8;  // weights p * dv / reference are scaled by 2^8: at most 2^14 with the slack
constexpr float kSmallestScale = 5.9604645e-8f;  // 2^-24, the smallest f16

struct Q4Args {
  const uint8_t* k;
  const uint8_t* v;
  const float* q;  // [B, Hq, D]
  const LaneInfo* lanes;
  const int* tables;
  float* out;      // [B, Hq, D]
  __half* out_xh;  // optional: in the hand-off layout
  int out_xh_nv;
  float* partial;  // [CTAs][2][heads of a unit][D + 2]: O, then reference and sum of the weights
  int batch, q_heads, kv_heads;
  int groups, heads;  // query-head groups per KV head, heads of a group (the last may have fewer)
  int direct;
  float scale_log2;
  long long op_window;
};

// What a lane attends over: positions [begin, end) in pages [first, first + pages).
struct Span {
  int begin, end, first, pages;
};
__device__ __forceinline__ Span span_of(const LaneInfo& info, long long op_window) {
  Span s;
  s.end = info.cursor + info.advance;
  s.begin = info.start;
  if (op_window >= 0) s.begin = max((int)max((long long)s.end - op_window, 0ll), info.start);
  s.first = s.begin / kPage;
  s.pages = info.advance == 0 || s.end <= s.begin ? 0 : (s.end - 1) / kPage + 1 - s.first;
  return s;
}

// Pages of all lanes, by every warp for itself.
__device__ __forceinline__ long long all_pages(const Q4Args& a) {
  long long sum = 0;
  for (int i = threadIdx.x & 31; i < a.batch; i += 32) sum += span_of(a.lanes[i], a.op_window).pages;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  return sum;
}
// The lane that holds the page `at` (of all lanes' pages times `units`), and how many pages times units come before it.
__device__ __forceinline__ void lane_at(const Q4Args& a, long long at, int units, int* found, long long* before) {
  long long base = 0;
  for (int i0 = 0; i0 < a.batch; i0 += 32) {
    const int i = i0 + (threadIdx.x & 31);
    const long long mine = i < a.batch ? (long long)span_of(a.lanes[i], a.op_window).pages * units : 0;
    long long upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, upto, off);
      if ((threadIdx.x & 31) >= off) upto += o;
    }
    const unsigned holds = __ballot_sync(0xffffffffu, base + upto > at);
    if (holds) {
      const int l = __ffs(holds) - 1;
      *found = i0 + l;
      *before = base + __shfl_sync(0xffffffffu, upto - mine, l);
      return;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  *found = a.batch;
  *before = base;
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {  // of an 8 x 8 tile of f16 pairs
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_flushed(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 halves(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// Codes in bits 0-3 (LOW) or 4-7 of both halves of w -> two f16 numbers code - 8, exact: 1024 + code less 1032, or 1024 + 16 code over 16.
template <bool LOW>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  if (LOW) return bits(__hsub2(halves((w & 0x000F000Fu) | 0x64006400u), __floats2half2_rn(1032.0f, 1032.0f)));
  return bits(__hfma2(halves((w & 0x00F000F0u) | 0x64006400u), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f)));
}
// 2^k with |x| 2^k in [2^13, 2^14), for a finite x that is not 0; 1 otherwise.
__device__ __forceinline__ float to_f16_range(float x) {
  const int e = (int)((__float_as_uint(x) >> 23) & 255u);
  if (e == 255 || x == 0.0f) return 1.0f;
  return __uint_as_float((unsigned)min(max(127 + 13 - (e - 127), 1), 254) << 23);
}

template <int D, int NT, int WARPS>
struct Q4Cfg {
  static constexpr int kBlocks = D / 32;
  static constexpr int kCodes = kPage * D / 2;                  // code bytes of a record
  static constexpr int kRecord = kCodes + kPage * kBlocks * 2;
  static constexpr int kStage = 2 * kRecord;                    // K, then V
  static constexpr int kHeads = 4 * NT;
  static constexpr int kPitch = D + 8;                          // of a head's partial sums: no bank conflicts
  static constexpr int kRing = WARPS * kStages * kStage;
  static constexpr size_t kSmem = kRing + (size_t)WARPS * kHeads * (kPitch + 2) * sizeof(float);
};

// A run of work, page by page for one warp: the unit it is in and its next page there.
struct Cursor {
  long long at, stop;  // position of the current unit's first page of this run in the row of all pages, and the run's end
  int lane, unit;      // unit: KV head * groups + group
  Span span;
  int table;
  int page0, page1;    // this run's pages of the unit (block-table indexes)
};

template <int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 16 / WARPS : 12 / WARPS) attention_q4_kernel(Q4Args a) {
  using Cfg = Q4Cfg<D, NT, WARPS>;
  constexpr int NB = Cfg::kBlocks;
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int units = a.kv_heads * a.groups, G = a.q_heads / a.kv_heads;
  chain_release();
  chain_wait();

  Cursor run;
  auto enter = [&](Cursor& c) {  // c.lane, c.unit and c.at are set; page0 relative to the unit's first page
    const LaneInfo info = a.lanes[c.lane];
    c.span = span_of(info, a.op_window);
    c.table = info.table_offset;
  };
  auto clip = [&](Cursor& c, int skipped) {
    c.page0 = c.span.first + skipped;
    c.page1 = c.span.first + (int)min((long long)c.span.pages, skipped + (c.stop - c.at));
  };
  // the next unit of the run; false when it is done
  auto advance = [&](Cursor& c) {
    c.at += c.page1 - c.page0;
    if (c.at >= c.stop) return false;
    if (++c.unit == units) {
      c.unit = 0;
      do ++c.lane; while (c.lane < a.batch && span_of(a.lanes[c.lane], a.op_window).pages == 0);
      if (c.lane >= a.batch) return false;
      enter(c);
    }
    clip(c, 0);
    return true;
  };
  if (a.direct) {
    run.lane = blockIdx.x / units;
    run.unit = blockIdx.x - run.lane * units;
    run.at = 0;
    enter(run);
    run.stop = run.span.pages;
    if (run.stop == 0) {
      run.page0 = run.page1 = 0;
    } else {
      clip(run, 0);
    }
  } else {
    const long long total = all_pages(a) * units;
    const long long begin = total * blockIdx.x / gridDim.x;
    run.stop = total * (blockIdx.x + 1) / gridDim.x;
    if (begin >= run.stop) return;
    long long before;
    lane_at(a, begin, units, &run.lane, &before);
    enter(run);
    run.at = begin;
    const long long inside = begin - before;
    run.unit = (int)(inside / run.span.pages);
    clip(run, (int)(inside - (long long)run.unit * run.span.pages));
  }
  const bool idle = run.page0 == run.page1;  // direct: a lane with nothing to attend over

  // the ring: this warp's pages, from `ahead`, the cursor that copies are issued from
  unsigned char* ring = smem + warp * (kStages * Cfg::kStage);
  Cursor ahead = run;
  int ahead_page = idle ? 0 : run.page0 + warp;
  bool more = !idle;
  const size_t page_stride = (size_t)a.kv_heads * Cfg::kRecord;
  auto issue = [&](int stage) {
    while (more && ahead_page >= ahead.page1) {
      more = advance(ahead);
      ahead_page = ahead.page0 + warp;
    }
    if (more) {
      const size_t off = (size_t)a.tables[ahead.table + ahead_page] * page_stride + (size_t)(ahead.unit / a.groups) * Cfg::kRecord;
      unsigned char* dst = ring + stage * Cfg::kStage;
#pragma unroll
      for (int c = lane; c < Cfg::kRecord / 16; c += 32) {
        copy16(dst + c * 16, a.k + off + c * 16);
        copy16(dst + Cfg::kRecord + c * 16, a.v + off + c * 16);
      }
      ahead_page += WARPS;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);

  float* sums = reinterpret_cast<float*>(smem + Cfg::kRing);  // [warp][head][pitch], then references and weights [warp][head]
  float* refs = sums + WARPS * Cfg::kHeads * Cfg::kPitch;
  float* weights = refs + WARPS * Cfg::kHeads;
  const int row_lo = (g >> 1) + 4 * (g & 1), row_hi = row_lo + 8;  // tokens of this thread's scores: row r of a tile is token r/2 + 4 (r%2)
  const bool wide_q = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
  int stage = 0;
  bool first_unit = true;
  while (true) {
    const int kv_head = run.unit / a.groups, head0 = kv_head * G + (run.unit - kv_head * a.groups) * a.heads;
    const int live_heads = min(a.heads, (kv_head + 1) * G - head0);
    // queries: column g of tile n is the value (g even) or the rest (g odd) of head 4 n + g / 2
    uint32_t qf[NT][NB][2][2];
    float unscale[NT];  // of the scores of head 4 n + t
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = 4 * n + (g >> 1);
      const bool live = h < live_heads;
      const float* q = a.q + ((size_t)run.lane * a.q_heads + head0 + (live ? h : 0)) * D + 8 * t;
      float4 x[NB][2];
      float most = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float* src = q + 32 * b + 4 * s;
          x[b][s] = wide_q ? *reinterpret_cast<const float4*>(src) : make_float4(src[0], src[1], src[2], src[3]);
          if (!live) x[b][s] = make_float4(0.f, 0.f, 0.f, 0.f);
          most = fmaxf(fmaxf(most, fmaxf(fabsf(x[b][s].x), fabsf(x[b][s].y))), fmaxf(fabsf(x[b][s].z), fabsf(x[b][s].w)));
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const float f = to_f16_range(most);
      unscale[n] = __shfl_sync(0xffffffffu, a.scale_log2 / f, 8 * t);
      auto split = [&](float u, float v) {
        u *= f;
        v *= f;
        const __half2 value = __floats2half2_rn(u, v);
        if ((g & 1) == 0) return bits(value);
        return bits(__floats2half2_rn(u - __low2float(value), v - __high2float(value)));
      };
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          qf[n][b][s][0] = split(x[b][s].x, x[b][s].y);
          qf[n][b][s][1] = split(x[b][s].z, x[b][s].w);
        }
    }
    float o[NT][2 * NB][4];
    float ref[NT], weight[NT];  // of head 4 n + t; the sum of weights is this thread's share
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      ref[n] = -INFINITY;
      weight[n] = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    }
    float top_scale = kSmallestScale;  // power of two that no |dv| so far exceeds

    for (int page = run.page0 + warp; page < run.page1; page += WARPS) {
      issue((stage + kStages - 1) % kStages);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const unsigned char* ks = ring + stage * Cfg::kStage;
      const unsigned char* vs = ks + Cfg::kRecord;
      const bool live_lo = page * kPage + row_lo >= run.span.begin && page * kPage + row_lo < run.span.end;
      const bool live_hi = page * kPage + row_hi >= run.span.begin && page * kPage + row_hi < run.span.end;

      // scores of tokens row_lo and row_hi
      float s_lo[NT], s_hi[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) s_lo[n] = s_hi[n] = 0.0f;
      {
        __align__(16) uint32_t w_lo[NB], w_hi[NB];
        __align__(8) uint32_t d_lo[NB / 2], d_hi[NB / 2];
        const unsigned char *lo = ks + row_lo * (D / 2) + t * (4 * NB), *hi = ks + row_hi * (D / 2) + t * (4 * NB);
        const unsigned char *scale_lo = ks + Cfg::kCodes + row_lo * (2 * NB), *scale_hi = ks + Cfg::kCodes + row_hi * (2 * NB);
        if constexpr (NB == 4) {
          *reinterpret_cast<uint4*>(w_lo) = *reinterpret_cast<const uint4*>(lo);
          *reinterpret_cast<uint4*>(w_hi) = *reinterpret_cast<const uint4*>(hi);
          *reinterpret_cast<uint2*>(d_lo) = *reinterpret_cast<const uint2*>(scale_lo);
          *reinterpret_cast<uint2*>(d_hi) = *reinterpret_cast<const uint2*>(scale_hi);
        } else {
          *reinterpret_cast<uint2*>(w_lo) = *reinterpret_cast<const uint2*>(lo);
          *reinterpret_cast<uint2*>(w_hi) = *reinterpret_cast<const uint2*>(hi);
          d_lo[0] = *reinterpret_cast<const uint32_t*>(scale_lo);
          d_hi[0] = *reinterpret_cast<const uint32_t*>(scale_hi);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t x = w_lo[b], y = w_hi[b], x8 = x >> 8, y8 = y >> 8;
          const uint32_t a00 = widen<true>(x), a01 = widen<true>(y), a02 = widen<false>(x), a03 = widen<false>(y);
          const uint32_t a10 = widen<true>(x8), a11 = widen<true>(y8), a12 = widen<false>(x8), a13 = widen<false>(y8);
          const float2 dl = __half22float2(halves(d_lo[b / 2])), dh = __half22float2(halves(d_hi[b / 2]));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma(c, a00, a01, a02, a03, qf[n][b][0][0], qf[n][b][0][1]);
            mma(c, a10, a11, a12, a13, qf[n][b][1][0], qf[n][b][1][1]);
            s_lo[n] = fmaf(b & 1 ? dl.y : dl.x, c[0] + c[1], s_lo[n]);
            s_hi[n] = fmaf(b & 1 ? dh.y : dh.x, c[2] + c[3], s_hi[n]);
          }
        }
      }
      __align__(8) uint32_t dv_lo[NB / 2], dv_hi[NB / 2];
      {
        const unsigned char *scale_lo = vs + Cfg::kCodes + row_lo * (2 * NB), *scale_hi = vs + Cfg::kCodes + row_hi * (2 * NB);
        if constexpr (NB == 4) {
          *reinterpret_cast<uint2*>(dv_lo) = *reinterpret_cast<const uint2*>(scale_lo);
          *reinterpret_cast<uint2*>(dv_hi) = *reinterpret_cast<const uint2*>(scale_hi);
        } else {
          dv_lo[0] = *reinterpret_cast<const uint32_t*>(scale_lo);
          dv_hi[0] = *reinterpret_cast<const uint32_t*>(scale_hi);
        }
      }
      // a masked token's rows may hold anything: neither its score nor its scale is looked at
      bool rises = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s_lo[n] = live_lo ? s_lo[n] * unscale[n] : -INFINITY;
        s_hi[n] = live_hi ? s_hi[n] * unscale[n] : -INFINITY;
        rises = rises || !(s_lo[n] <= ref[n] + kSlack) || !(s_hi[n] <= ref[n] + kSlack);
      }
      __half2 largest = __float2half2_rn(0.0f);
#pragma unroll
      for (int i = 0; i < NB / 2; ++i) {
        if (!live_lo) dv_lo[i] = 0u;
        if (!live_hi) dv_hi[i] = 0u;
        largest = __hmax2(largest, __hmax2(__habs2(halves(dv_lo[i])), __habs2(halves(dv_hi[i]))));
      }
      // an infinite scale spoils its own columns only: the reference stays finite
      const float largest_scale = fminf(fmaxf(__low2float(largest), __high2float(largest)), 65504.0f);
      rises = rises || largest_scale > top_scale;
      if (__any_sync(0xffffffffu, rises)) {
        float scale = largest_scale;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) scale = fmaxf(scale, __shfl_xor_sync(0xffffffffu, scale, off));
        float shrink = 1.0f;
        if (scale > top_scale) {
          const float raised = __uint_as_float((__float_as_uint(scale) + 0x7fffffu) & 0x7f800000u);  // the power of two at or above it
          shrink = top_scale / raised;
          top_scale = raised;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float most = fmaxf(s_lo[n], s_hi[n]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
          float f = 1.0f;
          if (most > ref[n] + kSlack) {  // each head for itself: its result does not depend on the others
            f = exp2_flushed(ref[n] - most);
            ref[n] = most;
          }
          weight[n] *= f;
          f *= shrink;
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) {
            o[n][i][0] *= f; o[n][i][1] *= f; o[n][i][2] *= f; o[n][i][3] *= f;
          }
        }
      }
      // weights, and their products with the V scales as (value, rest) pairs, transposed into operand order
      uint32_t pf[NT][NB][2];
      const float to_range = (float)(1 << kWeightBits) / top_scale;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float sub = ref[n] == -INFINITY ? 0.0f : ref[n];
        float p_lo = exp2_flushed(s_lo[n] - sub), p_hi = exp2_flushed(s_hi[n] - sub);
        weight[n] += p_lo + p_hi;
        p_lo *= to_range;
        p_hi *= to_range;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float2 dl = __half22float2(halves(dv_lo[b / 2])), dh = __half22float2(halves(dv_hi[b / 2]));
          const float w_lo = p_lo * (b & 1 ? dl.y : dl.x), w_hi = p_hi * (b & 1 ? dh.y : dh.x);
          const __half2 value = __floats2half2_rn(w_lo, w_hi);
          const __half2 rest = __floats2half2_rn(w_lo - __low2float(value), w_hi - __high2float(value));
          pf[n][b][0] = transpose8(bits(__lows2half2(value, rest)));
          pf[n][b][1] = transpose8(bits(__highs2half2(value, rest)));
        }
      }
      {
        __align__(8) uint32_t w[4][NB / 2];  // of tokens t, t + 4, t + 8, t + 12: columns 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned char* src = vs + (4 * i + t) * (D / 2) + g * (2 * NB);
          if constexpr (NB == 4) *reinterpret_cast<uint2*>(w[i]) = *reinterpret_cast<const uint2*>(src);
          else w[i][0] = *reinterpret_cast<const uint32_t*>(src);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const unsigned pick = b & 1 ? 0x7632u : 0x5410u;
          const uint32_t x = __byte_perm(w[0][b / 2], w[1][b / 2], pick), y = __byte_perm(w[2][b / 2], w[3][b / 2], pick), x8 = x >> 8, y8 = y >> 8;
          const uint32_t a00 = widen<true>(x), a01 = widen<false>(x), a02 = widen<true>(y), a03 = widen<false>(y);
          const uint32_t a10 = widen<true>(x8), a11 = widen<false>(x8), a12 = widen<true>(y8), a13 = widen<false>(y8);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma(o[n][2 * b], a00, a01, a02, a03, pf[n][b][0], pf[n][b][1]);
            mma(o[n][2 * b + 1], a10, a11, a12, a13, pf[n][b][0], pf[n][b][1]);
          }
        }
      }
      __syncwarp();
      stage = (stage + 1) % kStages;
    }

    // the unit's sums over the warps
    const float back = top_scale / (float)(1 << kWeightBits);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) weight[n] += __shfl_xor_sync(0xffffffffu, weight[n], off);
      float* dst = sums + (warp * Cfg::kHeads + 4 * n + t) * Cfg::kPitch + g;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        dst[16 * i] = (o[n][i][0] + o[n][i][1]) * back;
        dst[16 * i + 8] = (o[n][i][2] + o[n][i][3]) * back;
      }
      if (g == 0) {
        refs[warp * Cfg::kHeads + 4 * n + t] = ref[n];
        weights[warp * Cfg::kHeads + 4 * n + t] = weight[n];
      }
    }
    __syncthreads();
    const bool whole = run.page0 == run.span.first && run.page1 == run.span.first + run.span.pages;
    for (int i = threadIdx.x; i < live_heads * D; i += WARPS * 32) {
      const int h = i / D, d = i - h * D;
      float m = -INFINITY, acc = 0.0f, l = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) m = fmaxf(m, refs[w * Cfg::kHeads + h]);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float r = refs[w * Cfg::kHeads + h], f = r == -INFINITY ? 0.0f : exp2_flushed(r - m);
        acc += f * sums[(w * Cfg::kHeads + h) * Cfg::kPitch + d];
        l += f * weights[w * Cfg::kHeads + h];
      }
      if (whole || idle) {
        const float val = l == 0.0f ? 0.0f : acc / l;
        const int k = (head0 + h) * D + d;
        if (a.out) a.out[(size_t)run.lane * a.q_heads * D + k] = val;
        if (a.out_xh) a.out_xh[hand_off_cell(k >> 3, run.lane, a.out_xh_nv, a.q_heads * (D / 8)) + (k & 7)] = half_sat(val);
      } else {
        float* dst = a.partial + ((size_t)(2 * blockIdx.x + (first_unit ? 0 : 1)) * a.heads + h) * (D + 2);
        dst[d] = acc;
        if (d == 0) { dst[D] = m; dst[D + 1] = l; }
      }
    }
    first_unit = false;
    if (idle || !advance(run)) break;
    __syncthreads();  // the sums have been read
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Adds up the parts of units that were cut, and clears the rows of lanes with nothing to attend over. Grid (units of a lane, lanes).
__global__ void attention_q4_merge_kernel(Q4Args a, int D, int ctas) {
  chain_release();
  chain_wait();
  const int units = a.kv_heads * a.groups, unit = blockIdx.x, lane_id = blockIdx.y, G = a.q_heads / a.kv_heads;
  const long long total = all_pages(a) * units;
  const int pages = span_of(a.lanes[lane_id], a.op_window).pages;
  const int kv_head = unit / a.groups, head0 = kv_head * G + (unit - kv_head * a.groups) * a.heads;
  const int live_heads = min(a.heads, (kv_head + 1) * G - head0);
  auto store = [&](int h, int d, float val) {
    const int k = (head0 + h) * D + d;
    if (a.out) a.out[(size_t)lane_id * a.q_heads * D + k] = val;
    if (a.out_xh) a.out_xh[hand_off_cell(k >> 3, lane_id, a.out_xh_nv, a.q_heads * (D / 8)) + (k & 7)] = half_sat(val);
  };
  if (pages == 0) {
    for (int i = threadIdx.x; i < live_heads * D; i += blockDim.x) store(i / D, i % D, 0.0f);
    return;
  }
  long long before = 0;
  for (int i = threadIdx.x & 31; i < lane_id; i += 32) before += span_of(a.lanes[i], a.op_window).pages;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) before += __shfl_xor_sync(0xffffffffu, before, off);
  const long long s = before * units + (long long)unit * pages, e = s + pages;
  // the CTA that holds page x is the last whose run starts at or before it: total * c / ctas <= x
  const int c0 = (int)(((s + 1) * ctas - 1) / total), c1 = (int)((e * ctas - 1) / total);
  if (c0 == c1) return;
  // a run is empty where there are more CTAs than pages
  auto empty = [&](int c) { return total * c / ctas == total * (c + 1) / ctas; };
  auto part = [&](int c, int h) {
    const int slot = total * c / ctas >= s ? 0 : 1;  // the run's first unit or its last
    return a.partial + ((size_t)(2 * c + slot) * a.heads + h) * (D + 2);
  };
  for (int i = threadIdx.x; i < live_heads * D; i += blockDim.x) {
    const int h = i / D, d = i - h * D;
    float m = -INFINITY, acc = 0.0f, l = 0.0f;
    for (int c = c0; c <= c1; ++c)
      if (!empty(c)) m = fmaxf(m, part(c, h)[D]);
    for (int c = c0; c <= c1; ++c) {
      if (empty(c)) continue;
      const float* p = part(c, h);
      const float f = p[D] == -INFINITY ? 0.0f : exp2_flushed(p[D] - m);
      acc += f * p[d];
      l += f * p[D + 1];
    }
    store(h, d, l == 0.0f ? 0.0f : acc / l);
  }
}

// Query heads of a KV head in groups of at most eight: with more the accumulators of a warp do not fit its registers.
int head_groups(int q_heads, int kv_heads) { return (q_heads / kv_heads + 7) / 8; }

template <int D, int NT, int WARPS>
cudaError_t launch_t(const Q4Args& a, unsigned ctas, cudaStream_t stream) {
  auto kernel = attention_q4_kernel<D, NT, WARPS>;
  constexpr size_t smem = Q4Cfg<D, NT, WARPS>::kSmem;
  const cudaError_t e = opt_in_shared_memory(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, dim3(ctas), dim3(WARPS * 32), smem, stream, a);
}

}  // namespace

bool attention_q4_supported(const PoolView& pool, int q_heads) {
  return pool.dtype == kKvQ4 && pool.block_size == kPage && (pool.head_dim == 64 || pool.head_dim == 128) && pool.kv_heads > 0 && q_heads % pool.kv_heads == 0 &&
         q_heads / pool.kv_heads >= 1 && q_heads / pool.kv_heads <= 16;
}

Q4Plan plan_attention_q4(int batch, int q_heads, int kv_heads, int head_dim, int max_pages, int sm_count) {
  Q4Plan p;
  const int groups = head_groups(q_heads, kv_heads), heads = (q_heads / kv_heads + groups - 1) / groups;
  const int64_t units = (int64_t)batch * kv_heads * groups;
  const bool narrow = heads <= 4;
  const int warps = narrow ? 8 : 4, resident = narrow ? 2 : 3;
  p.direct = max_pages <= kDirectPages;
  // as many CTAs as are resident at once, but two pages for every warp where the tables are short
  p.ctas = p.direct ? units : std::min<int64_t>((int64_t)resident * sm_count, (units * max_pages + 2 * warps - 1) / (2 * warps));
  p.scratch_bytes = p.direct ? 0 : (size_t)p.ctas * 2 * heads * (head_dim + 2) * sizeof(float);
  return p;
}

cudaError_t launch_attention_q4(const PoolView& pool, const float* q, const LaneInfo* lanes, const int* tables, int batch, int q_heads, double scale,
                                long long op_window, float* out, const Q4Plan& plan, float* scratch, cudaStream_t stream, int* launches, __half* out_xh,
                                int xh_nv) {
  if (batch == 0) return cudaSuccess;
  Q4Args a;
  a.k = (const uint8_t*)pool.k;
  a.v = (const uint8_t*)pool.v;
  a.q = q;
  a.lanes = lanes;
  a.tables = tables;
  a.out = out;
  a.out_xh = out_xh;
  a.out_xh_nv = xh_nv;
  a.partial = scratch;
  a.batch = batch;
  a.q_heads = q_heads;
  a.kv_heads = pool.kv_heads;
  a.groups = head_groups(q_heads, pool.kv_heads);
  a.heads = (q_heads / pool.kv_heads + a.groups - 1) / a.groups;
  a.direct = plan.direct;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.op_window = op_window;
  const unsigned ctas = (unsigned)plan.ctas;
  cudaError_t e;
  if (a.heads <= 4) e = pool.head_dim == 128 ? launch_t<128, 1, 8>(a, ctas, stream) : launch_t<64, 1, 8>(a, ctas, stream);
  else e = pool.head_dim == 128 ? launch_t<128, 2, 4>(a, ctas, stream) : launch_t<64, 2, 4>(a, ctas, stream);
  if (e != cudaSuccess) return e;
  if (launches) ++*launches;
  if (plan.direct) return cudaSuccess;
  e = launch_chained(attention_q4_merge_kernel, dim3((unsigned)(a.kv_heads * a.groups), (unsigned)batch), dim3(128), 0, stream, a, pool.head_dim, (int)plan.ctas);
  if (e == cudaSuccess && launches) ++*launches;
  return e;
}

}  // namespace etc
