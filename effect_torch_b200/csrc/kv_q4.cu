// Rows into and out of pages held in 4 bits (kv_q4.cuh). Four neighbouring threads to a block of 32 values, eight each: loads and stores
// of values are 32 bytes per thread and whole lines per warp, codes are put in their places by shuffles among the four. Bound by
// HBM on the f32 side (4 bytes a value against 0.56).
#include <algorithm>

#include "kernels.h"
#include "kv_q4.cuh"

namespace etc {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void load8(const float* src, bool wide, float (&v)[8]) {
  if (wide) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __ldg(src + i);
  }
}

// Grid (parts of a lane's new rows, lanes): a part is eight values of a row of one head, parts of a row next to each other.
__global__ void __launch_bounds__(kThreads) q4_append_kernel(PoolView pool, const float* __restrict__ k, const float* __restrict__ v,
                                                             const LaneInfo* __restrict__ lanes, const int* __restrict__ tables, int tokens,
                                                             int64_t lane_stride, int64_t head_stride, int64_t token_stride, int wide) {
  const LaneInfo info = lanes[blockIdx.y];
  const int parts = pool.head_dim / 8, nb = pool.head_dim / 32;
  const int live_tokens = min(info.advance, tokens);
  const int64_t index = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  const int64_t row = index / parts;
  const int part = (int)(index - row * parts), token = (int)(row % tokens), head = (int)(row / tokens);
  const bool live = head < pool.kv_heads && token < live_tokens;  // the same for the four threads of a block
  float x[8] = {}, y[8] = {};
  Q4Row k_row = {}, v_row = {};
  if (live) {
    const int64_t src = (int64_t)blockIdx.y * lane_stride + head * head_stride + token * token_stride + part * 8;
    load8(k + src, wide, x);
    load8(v + src, wide, y);
    const int pos = info.cursor + token, page = tables[info.table_offset + pos / pool.block_size], slot = pos % pool.block_size;
    k_row = q4_row(pool, pool.k, page, head, slot);
    v_row = q4_row(pool, pool.v, page, head, slot);
  }
  q4_store_block(x, false, k_row, part / 4, nb, live);
  q4_store_block(y, true, v_row, part / 4, nb, live);
}

__global__ void __launch_bounds__(kThreads) q4_rows_kernel(PoolView pool, const uint32_t* __restrict__ rows, int64_t n, float* __restrict__ out, int which,
                                                           int64_t pool_rows, int wide, DeviceStatus* status) {
  const int parts = pool.head_dim / 8, nb = pool.head_dim / 32;
  const int64_t total = n * pool.kv_heads * parts;
  // whole warps go round: the threads of a block exchange codes
  for (int64_t base = (blockIdx.x * (int64_t)kThreads + threadIdx.x) & ~31ll; base < total; base += (int64_t)gridDim.x * kThreads) {
    const int64_t index = base + (threadIdx.x & 31);
    const bool inside = index < total;
    const int64_t slice = inside ? index / parts : 0, i = slice / pool.kv_heads;
    const int part = (int)(index - slice * parts), head = (int)(slice - i * pool.kv_heads);
    const uint32_t row = inside ? rows[i] : 0u;
    const bool live = inside && row < pool_rows;
    if (inside && !live && atomicCAS(&status->code, kStatusNone, kStatusRowOutOfRange) == kStatusNone) {
      status->value = row;
      status->bound = pool_rows;
    }
    float v[8];
    const Q4Row src = live ? q4_row(pool, which == 0 ? pool.k : pool.v, (int)(row / pool.block_size), head, (int)(row % pool.block_size)) : Q4Row();
    q4_load_block(src, which != 0, part / 4, nb, live, v);
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
  const int64_t parts = (int64_t)pool.kv_heads * tokens * (pool.head_dim / 8);
  const bool wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 && lane_stride % 4 == 0 && head_stride % 4 == 0 && token_stride % 4 == 0;
  const dim3 grid((unsigned)((parts + kThreads - 1) / kThreads), (unsigned)batch);
  q4_append_kernel<<<grid, kThreads, 0, stream>>>(pool, k, v, lanes, tables, tokens, lane_stride, head_stride, token_stride, wide);
  return cudaGetLastError();
}

cudaError_t launch_q4_rows(const PoolView& pool, const uint32_t* rows, int64_t n, float* out, int which, int64_t pool_rows, DeviceStatus* status,
                           cudaStream_t stream) {
  const int64_t total = n * pool.kv_heads * (pool.head_dim / 8);
  if (total == 0) return cudaSuccess;
  const unsigned grid = (unsigned)std::min<int64_t>((total + kThreads - 1) / kThreads, 148 * 64);
  q4_rows_kernel<<<grid, kThreads, 0, stream>>>(pool, rows, n, out, which, pool_rows, (reinterpret_cast<uintptr_t>(out) & 15) == 0, status);
  return cudaGetLastError();
}

}  // namespace etc
