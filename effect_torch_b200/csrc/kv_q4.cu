// Rows into and out of pages held in 4 bits (kv_q4.cuh). Four neighbouring threads to a block of 32 values, eight each: loads and stores
// of values are 32 bytes per thread and whole lines per warp, codes are put in their places by shuffles among the four. Bound by
// HBM on the f32 side (4 bytes a value against 0.56).
#include <algorithm>

#include "chain.cuh"
#include "kernels.h"
#include "kv_q4.cuh"

namespace etc {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void load8(const float* src, bool wide, float (&v)[8]) {
  if (wide) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *(reinterpret_cast<const float4*>(src) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = src[i];
  }
}

// Division by a number that is mostly a power of two.
struct Divisor {
  int value, shift;  // shift < 0: not one
  __host__ static Divisor of(int v) {
    Divisor d = {v, -1};
    for (int s = 0; s < 31; ++s)
      if (v == 1 << s) d.shift = s;
    return d;
  }
  __device__ __forceinline__ int divide(int x) const { return shift >= 0 ? x >> shift : x / value; }
};

// Grid (parts of the new rows of a lane's head, heads, lanes): a part is eight values, parts of a row next to each other.
__global__ void __launch_bounds__(kThreads) q4_append_kernel(PoolView pool, const float* k, const float* v, const LaneInfo* lanes, const int* tables, int tokens,
                                                             int64_t lane_stride, int64_t head_stride, int64_t token_stride, int wide, Divisor parts, Divisor page_rows) {
  chain_release();
  chain_wait();
  const int head = blockIdx.y;
  const LaneInfo info = lanes[blockIdx.z];
  const int nb = pool.head_dim / 32;
  const int index = blockIdx.x * blockDim.x + threadIdx.x, token = parts.divide(index), part = index - token * parts.value;
  const bool live = token < min(info.advance, tokens);  // the same for the four threads of a block
  float x[8] = {}, y[8] = {};
  Q4Row k_row = {}, v_row = {};
  if (live) {
    const int64_t src = (int64_t)blockIdx.z * lane_stride + head * head_stride + token * token_stride + part * 8;
    load8(k + src, wide, x);
    load8(v + src, wide, y);
    const int pos = info.cursor + token, block = page_rows.divide(pos), page = tables[info.table_offset + block], slot = pos - block * page_rows.value;
    k_row = q4_row(pool, pool.k, page, head, slot);
    v_row = q4_row(pool, pool.v, page, head, slot);
  }
  q4_store_block(x, false, k_row, part / 4, nb, live);
  q4_store_block(y, true, v_row, part / 4, nb, live);
}

// Rows are counted from the CTA's first, so that one division of 64 bits per CTA is enough.
constexpr int kPasses = 4;
__global__ void __launch_bounds__(kThreads) q4_rows_kernel(PoolView pool, const uint32_t* rows, int64_t n, float* out, int which, int64_t pool_rows, int wide,
                                                           DeviceStatus* status, Divisor parts, Divisor row_parts, Divisor page_rows) {
  chain_release();
  chain_wait();
  const int nb = pool.head_dim / 32;
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kPasses), row0 = first / row_parts.value, total = n * row_parts.value;
  const int skew = (int)(first - row0 * row_parts.value);
  // row numbers and codes of all passes are requested before the first is unpacked
  uint32_t number[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int at = skew + p * kThreads + (int)threadIdx.x;
    number[p] = first + p * kThreads + threadIdx.x < total ? rows[row0 + row_parts.divide(at)] : 0u;
  }
  Q4Part fetched[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int at = skew + p * kThreads + (int)threadIdx.x, in_row = at - row_parts.divide(at) * row_parts.value, head = parts.divide(in_row), part = in_row - head * parts.value;
    const bool inside = first + p * kThreads + threadIdx.x < total, live = inside && number[p] < pool_rows;
    if (inside && !live && atomicCAS(&status->code, kStatusNone, kStatusRowOutOfRange) == kStatusNone) {
      status->value = number[p];
      status->bound = pool_rows;
    }
    fetched[p] = {0x88888888u, 0.0f};
    if (live) {
      const int page = page_rows.divide((int)number[p]);
      fetched[p] = q4_fetch(q4_row(pool, which == 0 ? pool.k : pool.v, page, head, (int)number[p] - page * page_rows.value), which != 0, part / 4, nb);
    }
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t index = first + p * kThreads + threadIdx.x;
    const bool inside = index < total;
    float v[8];
    q4_unpack(fetched[p], which != 0, v);
    if (!inside) continue;
    float* dst = out + index * 8;
    if (wide) {
      __stcs(reinterpret_cast<float4*>(dst), make_float4(v[0], v[1], v[2], v[3]));
      __stcs(reinterpret_cast<float4*>(dst) + 1, make_float4(v[4], v[5], v[6], v[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) dst[j] = v[j];
    }
  }
}

}  // namespace

cudaError_t launch_q4_append(const PoolView& pool, const float* k, const float* v, const LaneInfo* lanes, const int* tables, int batch, int tokens,
                             int64_t lane_stride, int64_t head_stride, int64_t token_stride, cudaStream_t stream) {
  const int parts = pool.head_dim / 8;
  const bool wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 && lane_stride % 4 == 0 && head_stride % 4 == 0 && token_stride % 4 == 0;
  const int64_t count = (int64_t)tokens * parts;
  if (count > INT32_MAX - kThreads) return cudaErrorInvalidValue;
  const unsigned threads = (unsigned)std::min<int64_t>(kThreads, (count + 31) / 32 * 32);
  const dim3 grid((unsigned)((count + threads - 1) / threads), (unsigned)pool.kv_heads, (unsigned)batch);
  return launch_chained(q4_append_kernel, grid, dim3(threads), 0, stream, pool, k, v, lanes, tables, tokens, lane_stride, head_stride, token_stride, (int)wide,
                        Divisor::of(parts), Divisor::of(pool.block_size));
}

cudaError_t launch_q4_rows(const PoolView& pool, const uint32_t* rows, int64_t n, float* out, int which, int64_t pool_rows, DeviceStatus* status,
                           cudaStream_t stream) {
  const int parts = pool.head_dim / 8, row_parts = pool.kv_heads * parts;
  const int64_t total = n * row_parts;
  if (total == 0) return cudaSuccess;
  const int64_t grid = (total + kThreads * kPasses - 1) / (kThreads * kPasses);
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  return launch_chained(q4_rows_kernel, dim3((unsigned)grid), dim3(kThreads), 0, stream, pool, rows, n, out, which, pool_rows, (int)((reinterpret_cast<uintptr_t>(out) & 15) == 0),
                        status, Divisor::of(parts), Divisor::of(row_parts), Divisor::of(pool.block_size));
}

}  // namespace etc
