// Rows into and out of pages held in 4 bits (kv_q4.cuh). Four neighbouring threads to a block of 32 values, eight each: loads and stores
// of values are 32 bytes per thread and whole lines per warp, codes are put in their places by shuffles among the four. The bytes
// are f32 ones (4 a value against 0.56), but large appends are bound by instructions, some 24 per value (extreme of the block, code,
// packing): 8 lanes of 509 tokens, 8 heads of 128, in and out in 21.6 us (76 MB, 3530 GB/s); calls of one token by their launches.
#include <algorithm>
#include <initializer_list>

#include "chain.cuh"
#include "kernels.h"
#include "kv_q4.cuh"

namespace etc {

namespace {

constexpr int kThreads = 256;

// Eight consecutive values; `width` is the boundary in bytes that they start on (32, 16 or 4).
__device__ __forceinline__ void load8(const float* src, int width, float (&v)[8]) {
  if (width == 32) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(src)
                 : "memory");
  } else if (width == 16) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *(reinterpret_cast<const float4*>(src) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = src[i];
  }
}
__device__ __forceinline__ void store8(float* dst, int width, const float (&v)[8]) {
  if (width == 32) {
    asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                 "f"(v[6]), "f"(v[7])
                 : "memory");
  } else if (width == 16) {
    __stcs(reinterpret_cast<float4*>(dst), make_float4(v[0], v[1], v[2], v[3]));
    __stcs(reinterpret_cast<float4*>(dst) + 1, make_float4(v[4], v[5], v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = v[i];
  }
}
// The widest boundary that these addresses and offsets share.
int boundary(std::initializer_list<const void*> addresses, std::initializer_list<int64_t> strides) {
  uint64_t bits = 0;
  for (const void* p : addresses) bits |= reinterpret_cast<uintptr_t>(p);
  for (int64_t s : strides) bits |= (uint64_t)s * sizeof(float);
  return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 4;
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
                                                             int64_t lane_stride, int64_t head_stride, int64_t token_stride, int width, Divisor parts, Divisor page_rows) {
  chain_release();
  chain_wait();
  const int head = blockIdx.y;
  const LaneInfo info = lanes[blockIdx.z];
  const int nb = pool.head_dim / 32;
  const int index = blockIdx.x * blockDim.x + threadIdx.x, token = parts.divide(index), part = index - token * parts.value;
  const bool live = token < min(info.advance, tokens);  // the same for the four threads of a block
  float x[8] = {}, y[8] = {};
  Q4Row k_row = {}, v_row = {};
  if (token < tokens) {  // whether it is live or not, so that it does not wait for the lane
    const int64_t src = (int64_t)blockIdx.z * lane_stride + head * head_stride + token * token_stride + part * 8;
    load8(k + src, width, x);
    load8(v + src, width, y);
  }
  if (live) {
    const int pos = info.cursor + token, block = page_rows.divide(pos), page = tables[info.table_offset + block], slot = pos - block * page_rows.value;
    k_row = q4_row(pool, false, page, head, slot);
    v_row = q4_row(pool, true, page, head, slot);
  }
  q4_store_block(x, false, k_row, part / 4, nb, live);
  q4_store_block(y, true, v_row, part / 4, nb, live);
}

// One part per thread: with two or four, their codes requested ahead, fewer warps hide the latency of two dependent loads (24.6 us for a
// chunk's append and read-back against 26.2 and 30). Rows are counted from the CTA's first, so that divisions stay in 32 bits.
__global__ void __launch_bounds__(kThreads) q4_rows_kernel(PoolView pool, const uint32_t* rows, int64_t n, float* out, int which, int64_t pool_rows, int width,
                                                           DeviceStatus* status, Divisor parts, Divisor row_parts, Divisor page_rows) {
  chain_release();
  chain_wait();
  const int nb = pool.head_dim / 32;
  const int64_t first = (int64_t)blockIdx.x * kThreads, row0 = row_parts.shift >= 0 ? first >> row_parts.shift : first / row_parts.value;
  const int at = (int)(first - row0 * row_parts.value) + (int)threadIdx.x, row = row_parts.divide(at);
  const int in_row = at - row * row_parts.value, head = parts.divide(in_row), part = in_row - head * parts.value;
  const bool inside = row0 + row < n;
  const uint32_t number = inside ? rows[row0 + row] : 0u;
  const bool live = inside && number < pool_rows;
  if (inside && !live && atomicCAS(&status->code, kStatusNone, kStatusRowOutOfRange) == kStatusNone) {
    status->value = number;
    status->bound = pool_rows;
  }
  Q4Part fetched = {0u, 0.0f};
  if (live) {
    const int page = page_rows.divide((int)number);
    fetched = q4_fetch(q4_row(pool, which != 0, page, head, (int)number - page * page_rows.value), which != 0, part / 4, nb);
  }
  float v[8];
  q4_unpack(fetched, which != 0, v);
  if (inside) {
    if (!live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;  // not the -0 of a scale of zero
    }
    store8(out + (first + threadIdx.x) * 8, width, v);
  }
}

}  // namespace

cudaError_t launch_q4_append(const PoolView& pool, const float* k, const float* v, const LaneInfo* lanes, const int* tables, int batch, int tokens,
                             int64_t lane_stride, int64_t head_stride, int64_t token_stride, cudaStream_t stream) {
  const int parts = pool.head_dim / 8;
  const int64_t count = (int64_t)tokens * parts;
  if (count > INT32_MAX - kThreads) return cudaErrorInvalidValue;
  const unsigned threads = (unsigned)std::min<int64_t>(kThreads, (count + 31) / 32 * 32);
  const dim3 grid((unsigned)((count + threads - 1) / threads), (unsigned)pool.kv_heads, (unsigned)batch);
  return launch_chained(q4_append_kernel, grid, dim3(threads), 0, stream, pool, k, v, lanes, tables, tokens, lane_stride, head_stride, token_stride,
                        boundary({k, v}, {lane_stride, head_stride, token_stride}),
                        Divisor::of(parts), Divisor::of(pool.block_size));
}

cudaError_t launch_q4_rows(const PoolView& pool, const uint32_t* rows, int64_t n, float* out, int which, int64_t pool_rows, DeviceStatus* status,
                           cudaStream_t stream) {
  const int parts = pool.head_dim / 8, row_parts = pool.kv_heads * parts;
  const int64_t total = n * row_parts;
  if (total == 0) return cudaSuccess;
  const int64_t grid = (total + kThreads - 1) / kThreads;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  return launch_chained(q4_rows_kernel, dim3((unsigned)grid), dim3(kThreads), 0, stream, pool, rows, n, out, which, pool_rows, boundary({out}, {}), status, Divisor::of(parts), Divisor::of(row_parts), Divisor::of(pool.block_size));
}

}  // namespace etc
