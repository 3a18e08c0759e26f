// Log probabilities of given tokens, the entropy of each distribution and its most likely alternatives, from logits rows.
//
// With m the largest logit of a row, s = sum exp(x - m) and t = sum (x - m) exp(x - m):
//   log p(i) = x_i - m - ln s          entropy = ln s - t / s
// and the alternatives are the first n tokens by (value descending, token ascending).
//
// A row is read once. Every thread carries (m, s, t) of its values, rescaled when its maximum rises, and the triples are merged by
// shuffles, through shared memory and, where several CTAs share a row, through the cluster's. The alternatives need no second
// pass either: the n-th largest of the maxima of 32 groups of threads (a 64-bit key of value and inverted token, so that no two are
// equal) is a lower bound of the n-th largest key. Only threads whose own maximum reaches it can hold an alternative; a warp
// looks at each such thread's values again (some hundred; from L2 where few rows are in flight, else from HBM), lists those that reach the bound, and the list is ranked by
// counting. Should the list overflow (an order of logits made for it), the alternatives are found one after the other instead.
//
// Bound by HBM where rows are many, 2048 of 128256 (1.05 GB) 160 to 171 us (boxes differ) = 6.15 to 6.55 TB/s of a copy's 6.55; by latency where
// they are few, one with 20 alternatives 10.8 us, 32 with 5 alternatives 11.5. Many rows with alternatives read part of the row twice: 2048 with 20 take
// 288 us, with 32 428.
//
// Sums are f32 within a batch of loads (24 values), over a thread's batches (up to 171 of the largest vocabulary) and within a warp, f64 from
// the warps on: no more than 200 additions in a row. (All values of a thread in one row, 4096 of the largest vocabulary: ln s off by 6e-5.)
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "chain.cuh"
#include "kernels.h"

namespace etc {

namespace {

namespace cg = cooperative_groups;

constexpr int kGroups = 32;               // groups of neighbouring threads: as many as alternatives can be asked for
constexpr int kBatch = 6;                 // 16-byte loads in flight per thread
constexpr int kListed = 2048;             // fewer groups than alternatives hold at most 31 * 16 * 4 values between them, of 512 threads
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNothing = -200.0f;       // exp2(kNothing * log2 e) is 0 in f32
static_assert(kMaxAlternatives <= kGroups, "a bound needs a group per alternative");
static_assert((kMaxAlternatives - 1) * 16 * 4 <= kListed, "the list holds what short rows have");

struct LogprobArgs {
  const float* logits;
  int64_t vocab, row_stride;
  const uint32_t* targets;
  float* logprobs;
  float* entropy;
  int top;
  uint32_t* top_tokens;
  float* top_logprobs;
  DeviceStatus* status;
  int chunks;  // 16-byte pieces of a row per CTA
  int64_t first_row;
};

// Larger value -> larger key; of equal values (0 and -0 are equal) the lower token has the larger key. 0 is below every key.
__device__ __forceinline__ uint64_t order_key(float v, uint32_t token) {
  const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));
  const uint32_t ordered = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)ordered << 32) | (uint64_t)(0xFFFFFFFFu - token);
}
__device__ __forceinline__ uint32_t key_token(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t ordered = (uint32_t)(key >> 32);
  return __uint_as_float((ordered & 0x80000000u) ? (ordered ^ 0x80000000u) : ~ordered);
}
// The maximum, NaN if any is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float exp2_flushed(float v) {  // results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// m, s and t of a set of values; s = t = 0 for none.
struct Moments {
  float m = -INFINITY, s = 0.0f, t = 0.0f;
  // onto the sums of a batch, which are added to s and t when it is through
  __device__ __forceinline__ void add(float x, float& batch_s, float& batch_t) const {
    const float d = fmaxf(x - m, kNothing), e = exp2_flushed(d * kLog2e);
    batch_s += e;
    batch_t = fmaf(d, e, batch_t);
  }
  __device__ __forceinline__ void raise(float to) {  // to >= m
    const float d = fmaxf(m - to, kNothing), f = exp2_flushed(d * kLog2e);
    t = fmaf(d, s, t) * f;
    s *= f;
    m = to;
  }
};

constexpr long long kNone = 0x7fffffffffffffffll;

template <int THREADS>
struct Shared {
  float warp_max[THREADS / 32];
  double warp_s[THREADS / 32], warp_t[THREADS / 32];
  float row_max;  // the first CTA: of the row
  double log_s;
  // of the CTA, read by the first of the row's cluster
  float m;
  double s, t;
  long long bad;
  uint64_t group_best[kGroups];
  uint64_t bound;
  uint64_t best[kMaxAlternatives];  // the CTA's alternatives, largest first; 0 where there are none left
  int listed, threads_listed;
  uint64_t round_best[THREADS / 32];
};
template <int THREADS>
struct SharedTop : Shared<THREADS> {
  uint64_t list[kListed];
  short thread_list[THREADS];
  uint64_t merged[kMaxCluster * kMaxAlternatives];  // the first CTA: everybody's
};

template <bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_kernel(LogprobArgs a) {
  constexpr int kThreads = THREADS, kWarps = THREADS / 32, kWidth = THREADS / kGroups;
  using Sh = std::conditional_t<TOP, SharedTop<THREADS>, Shared<THREADS>>;
  __shared__ Sh sh;
  chain_release();  // the next kernel may be scheduled; it waits for this one before touching memory
  chain_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned rank = cluster.block_rank();
  const int64_t row = blockIdx.x / cluster.num_blocks();
  const float* x = a.logits + row * a.row_stride;
  // The row in 16-byte pieces from the boundary at or before it; the first and the last may lie partly outside.
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  const int64_t pieces = (a.vocab + skew + 3) >> 2;
  const int64_t piece0 = min(pieces, (int64_t)rank * a.chunks), piece1 = min(pieces, piece0 + a.chunks);
  auto whole = [&](int64_t p) { return 4 * p >= skew && 4 * p + 4 - skew <= a.vocab; };
  auto load = [&](int64_t p) {  // values outside the row are -inf
    const int64_t i = 4 * p - skew;
    if (whole(p)) return *reinterpret_cast<const float4*>(x + i);
    auto at = [&](int64_t j) { return j >= 0 && j < a.vocab ? x[j] : -INFINITY; };
    return make_float4(at(i), at(i + 1), at(i + 2), at(i + 3));
  };
  if (threadIdx.x == 0) {
    sh.bad = kNone;
    sh.listed = sh.threads_listed = 0;
  }
  if (TOP) {
    for (int i = threadIdx.x; i < kMaxAlternatives; i += kThreads) sh.best[i] = 0;
  }
  __syncthreads();

  Moments mine;
  uint32_t at_best = 0;  // token of mine.m
  bool any = false;
  auto take = [&](const float4 (&v)[kBatch], int64_t p, int n) {
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (u < n) most = max_nan(max_nan(most, max_nan(v[u].x, v[u].y)), max_nan(v[u].z, v[u].w));
    if (!(most < INFINITY)) {  // a NaN or +inf: reported, the row's results mean nothing
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (u < n && !(w[j] < INFINITY)) atomicMin(&sh.bad, (long long)(4 * (p + (int64_t)u * kThreads) - skew + j));
      }
    }
    if (most > mine.m || (TOP && !any)) {
      if (TOP) {  // the first value that is the largest; what lies outside the row is none
        any = true;
        bool found = false;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const float w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int64_t i = 4 * (p + (int64_t)u * kThreads) - skew + j;
            if (u < n && !found && w[j] == most && i >= 0 && i < a.vocab) {
              found = true;
              at_best = (uint32_t)i;
            }
          }
        }
        any = found;
      }
      if (most > mine.m) mine.raise(most);
    }
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (u < n) {
        mine.add(v[u].x, s, t);
        mine.add(v[u].y, s, t);
        mine.add(v[u].z, s, t);
        mine.add(v[u].w, s, t);
      }
    mine.s += s;
    mine.t += t;
  };
  {
    // a thread's pieces are kThreads apart; all but the row's first and last are whole
    int64_t p = piece0 + threadIdx.x;
    float4 v[kBatch];
    for (; p + (int64_t)(kBatch - 1) * kThreads < piece1; p += (int64_t)kBatch * kThreads) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) v[u] = load(p + (int64_t)u * kThreads);
      take(v, p, kBatch);
    }
    if constexpr (TOP) {
      for (; p < piece1; p += kThreads) {
        v[0] = load(p);
        take(v, p, 1);
      }
    } else if (p < piece1) {  // at once, too (with alternatives that needs more than it saves: 344 us against 232 for 2048 rows of 128256 and five of them)
      const int n = (int)((piece1 - p + kThreads - 1) / kThreads);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (u < n) v[u] = load(p + (int64_t)u * kThreads);
      take(v, p, n);
    }
  }

  // (m, s, t) of the CTA
  float m = mine.m;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) sh.warp_max[warp] = m;
  __syncthreads();
  m = sh.warp_max[lane % kWarps];
#pragma unroll
  for (int off = kWarps / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float own_best = mine.m;
  if (m > -INFINITY) mine.raise(m);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    mine.s += __shfl_xor_sync(0xffffffffu, mine.s, off);
    mine.t += __shfl_xor_sync(0xffffffffu, mine.t, off);
  }
  if (lane == 0) { sh.warp_s[warp] = mine.s; sh.warp_t[warp] = mine.t; }

  uint64_t own_key = 0;
  if constexpr (TOP) {
    own_key = any ? order_key(own_best, at_best) : 0;
    uint64_t group_key = own_key;
#pragma unroll
    for (int off = kWidth / 2; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, group_key, off);
      group_key = o > group_key ? o : group_key;
    }
    if (threadIdx.x % kWidth == 0) sh.group_best[threadIdx.x / kWidth] = group_key;
  }
  __syncthreads();
  if (warp == 0) {
    double s = lane < kWarps ? sh.warp_s[lane] : 0.0, t = lane < kWarps ? sh.warp_t[lane] : 0.0;
#pragma unroll
    for (int off = kWarps / 2; off > 0; off >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, off);
      t += __shfl_xor_sync(0xffffffffu, t, off);
    }
    if (lane == 0) { sh.m = m; sh.s = s; sh.t = t; }
    if constexpr (TOP) {
      const uint64_t key = sh.group_best[lane];
      int before = 0;
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const uint64_t o = sh.group_best[j];
        before += o > key || (o == key && j < lane);  // groups without values are equal
      }
      if (before == a.top - 1) sh.bound = key;
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    const uint64_t bound = sh.bound;
    if (own_key > 0 && own_key >= bound) sh.thread_list[atomicAdd(&sh.threads_listed, 1)] = (short)threadIdx.x;
    __syncthreads();
    const int threads_listed = sh.threads_listed;
    // f(key) for the values of the listed threads, a warp for each
    auto each = [&](auto&& f) {
      for (int k = warp; k < threads_listed; k += kWarps)
        for (int64_t p = piece0 + sh.thread_list[k] + (int64_t)lane * kThreads; p < piece1; p += 32ll * kThreads) {
          const float4 v = load(p);
          const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int64_t i = 4 * p - skew + j;
            if (i >= 0 && i < a.vocab) f(order_key(w[j], (uint32_t)i));
          }
        }
    };
    each([&](uint64_t key) {
      if (key < bound) return;
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kListed) sh.list[at] = key;
    });
    __syncthreads();
    const int listed = sh.listed;
    if (listed <= kListed) {
      for (int k = threadIdx.x; k < listed; k += kThreads) {
        const uint64_t key = sh.list[k];
        int before = 0;
#pragma unroll 8
        for (int j = 0; j < listed; ++j) before += sh.list[j] > key;
        if (before < a.top) sh.best[before] = key;
      }
    } else {
      uint64_t below = ~0ull;
      for (int r = 0; r < a.top; ++r) {
        uint64_t most = 0;
        each([&](uint64_t key) {
          if (key < below && key > most) most = key;
        });
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
          const uint64_t o = __shfl_xor_sync(0xffffffffu, most, off);
          most = o > most ? o : most;
        }
        if (lane == 0) sh.round_best[warp] = most;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) most = sh.round_best[w] > most ? sh.round_best[w] : most;
        if (threadIdx.x == 0) sh.best[r] = most;
        below = most;
        __syncthreads();
      }
    }
  }
  if (cluster.num_blocks() > 1) cluster.sync();
  else __syncthreads();
  if (rank == 0) {
    const int peers = (int)cluster.num_blocks();
    if constexpr (TOP) {  // everybody's alternatives are on their way while the sums are put together
      for (int i = threadIdx.x; i < peers * a.top; i += kThreads) sh.merged[i] = cluster.map_shared_rank(&sh, i / a.top)->best[i % a.top];
    }
    if (warp == 0) {  // a lane per CTA of the row
      const bool there = lane < peers;
      const Sh* peer = cluster.map_shared_rank(&sh, there ? lane : 0);
      const float peer_m = there ? peer->m : -INFINITY;
      long long bad = there ? peer->bad : kNone;
      float row_max = peer_m;
#pragma unroll
      for (int off = kMaxCluster / 2; off > 0; off >>= 1) row_max = fmaxf(row_max, __shfl_xor_sync(0xffffffffu, row_max, off));
      double s = 0.0, t = 0.0;
      if (peer_m > -INFINITY) {
        const double d = (double)peer_m - (double)row_max, f = peers > 1 ? exp(d) : 1.0;
        s = peer->s * f;
        t = (peer->t + d * peer->s) * f;
      }
#pragma unroll
      for (int off = kMaxCluster / 2; off > 0; off >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, off);
        t += __shfl_xor_sync(0xffffffffu, t, off);
        bad = min(bad, __shfl_xor_sync(0xffffffffu, bad, off));
      }
      if (lane == 0) {
        const double log_s = log(s);
        sh.row_max = row_max;
        sh.log_s = log_s;
        if (a.entropy) a.entropy[row] = (float)(log_s - t / s);
        if (a.logprobs) {
          const uint32_t target = a.targets[row];
          const bool inside = target < a.vocab;
          a.logprobs[row] = inside ? (float)(((double)x[target] - (double)row_max) - log_s) : NAN;
          if (!inside && atomicCAS(&a.status->code, kStatusNone, kStatusTargetOutOfRange) == kStatusNone) {
            a.status->value = target;
            a.status->bound = a.vocab;
          }
        }
        if (bad != kNone && atomicCAS(&a.status->code, kStatusNone, kStatusBadLogprobLogit) == kStatusNone) {
          a.status->value = bad;
          a.status->bound = a.first_row + row;
        }
      }
    }
    if constexpr (TOP) {
      __syncthreads();
      const int n = peers * a.top;
      if (threadIdx.x < n) {
        const uint64_t key = sh.merged[threadIdx.x];
        int before = 0;
        if (peers == 1) {
          before = threadIdx.x;  // in order as they are
        } else {
#pragma unroll 8
          for (int j = 0; j < n; ++j) before += sh.merged[j] > key;
        }
        if (key > 0 && before < a.top) {
          const size_t o = (size_t)row * a.top + before;
          a.top_tokens[o] = key_token(key);
          a.top_logprobs[o] = (float)(((double)key_value(key) - (double)sh.row_max) - sh.log_s);
        }
      }
    }
  }
  if (cluster.num_blocks() > 1) cluster.sync();  // the other CTAs' shared memory lives until it has been read
}

}  // namespace

cudaError_t launch_logprobs(const float* logits, int64_t rows, int64_t vocab, int64_t row_stride, const uint32_t* targets, float* logprobs,
                            float* entropy, int top, uint32_t* top_tokens, float* top_logprobs, DeviceStatus* status, int sm_count,
                            cudaStream_t stream, int64_t first_row) {
  if (rows == 0) return cudaSuccess;
  LogprobArgs a = {logits, vocab, row_stride, targets, logprobs, entropy, top, top_tokens, top_logprobs, status, 0, first_row};
  // CTAs per row: as many as fill the SMs, two on each, as long as there is a piece for every thread. More rows take one, four of which an SM
  // holds (400 rows of 128256: 41.1 us against 44.5 by two; 1024: 84.3 against 102.5), but up to two for every SM, which would leave it
  // half empty, two where rows are long (256 rows of 128256: 30.3 us by two, 38.5 by one, 36.9 by four; of 32000 12.3 and 11.8).
  const int64_t pieces = (vocab + 3 + 3) / 4;
  unsigned ranks = 1;
  while (ranks < (unsigned)kMaxCluster && rows * ranks <= sm_count && pieces >= 2 * ranks * 512) ranks *= 2;
  if (rows > sm_count && rows <= 2 * sm_count && pieces >= 16384) ranks = 2;
  a.chunks = (int)((pieces + ranks - 1) / ranks);
  const dim3 grid((unsigned)(rows * ranks));
  auto launch = [&](auto kernel, int threads) { return launch_chained_cluster(kernel, grid, dim3((unsigned)threads), 0, stream, ranks, a); };
  // a row of its own: four small CTAs per SM hide one another's starts and ends; a part of a row: the shorter, the sooner
  if (ranks == 1) return top > 0 ? launch(logprobs_kernel<true, 256>, 256) : launch(logprobs_kernel<false, 256>, 256);
  return top > 0 ? launch(logprobs_kernel<true, 512>, 512) : launch(logprobs_kernel<false, 512>, 512);
}

}  // namespace etc
