// Decode attention over pages held in 4 bits (kv_q4.cuh): one query token per lane, 16-token pages, head dim 64 or 128.
//
// Mathematics. With codes c (whole numbers -8 .. 7) and a scale per row and block of 32 columns,
//   s[tok] = scale * sum_b dk[tok][b] * (sum_{d in b} q[d] ck[tok][d])      o[d] = sum_tok p[tok] dv[tok][b(d)] cv[tok][d] / sum_tok p[tok]
// so codes go through mma.sync.m16n8k16 as exact f16 numbers, a block of columns at a time, and scales are applied in f32: to the
// sums of a block (K), to the weights ahead of the product (V). What f16 would round, q and p * dv, is split in two f16 numbers, value and
// rest, 22 bits together, and the products of both are added in f32. Scores, weights, their sum and p * dv are f32.
//
// What the split costs. A query is scaled by a power of two, its largest value to 2^13 .. 2^14, and its values are held to 2^-22 of themselves or
// 2^-38 of the largest. For p * dv the power of two is that of the softmax: a head's reference is the largest (score + log2 of the token's
// largest |dv|), not the largest score, so that the largest product is 2^11 or more whatever the scales are. Products are held to 2^-22 of themselves, or to
// half of the smallest f16 number, 2^-36 of the largest one: a token whose weight is next to nothing adds that error once. With up to four heads
// (below) rests have columns and sums of their own and are held times 2^11, which makes it 2^-47. Scales below 2^-14 count as 2^-14 in this. (A reference of scores alone and one power of
// two for all dv of a run were 2.3 us faster over 64 lanes, and off by 3 % in a block whose scales are 1e6 below another's, and by
// 3e-6 to 5e-5 where one token draws most of the weight of 131072.) What remains is the tensor core's own sums, 16 products onto one f32.
//
// Layout. Tokens are the rows of the first product and the columns of the second: S^T = K Q^T and O^T = V^T P^T. A code page is read from
// shared memory as it was stored: 16 bytes of a K row per thread are its operands of all eight steps, 16 bytes of a pair of V rows its
// operands of all eight tiles; two codes are widened by one mask and one f16 operation. The eight columns of a tile are the heads of a KV head: up to
// four (PAIRS) as (value, rest) pairs, so that the split costs no tensor instruction where columns would stay empty, and a thread
// adds the two sums of its head; five to eight as they are, with a second product for the rests onto the same sums.
//
// What bounds it is instructions and their latency, not HBM: some 390 per page and warp, 152 of them widening codes, at 2.4 per cycle of an
// SM with 12 warps. 64 lanes of 128 to 4096 tokens (32 query heads, 8 KV heads of 128; 158 MB) 47.9 us = 3300 GB/s, one of 131072
// 45.2 us = 3340, 16 lanes of 1024 to 16384 with 64 heads 62.0 us = 2600 (the copy bandwidth is 6555).
//
// Work. The pages of all (lane, KV head) units in a row are cut into as many equal runs as there are warps, whatever the lengths of the
// lanes: nobody waits for the longest. A warp takes its run by pages, or pairs of them, through a ring of cp.async copies that runs on
// across units, and writes the units that lie inside it. What neighbouring warps of a CTA have of one unit is added up in shared memory at the end;
// the parts of a unit that several CTAs share go to scratch (two per CTA at most) and a second kernel adds them up. Short tables
// (kDirectPages) take one CTA per unit and no second kernel. (Runs of whole CTAs, whose warps took pages in turn and met after each
// unit: 67 us against 51 for 64 lanes of 128 to 4096 tokens.) With PAIRS a warp has the registers to take two pages at once, whose scores,
// reference and weights do not wait for each other: 45.8 us against 49.2 by single pages; a ring of two such steps does as well as longer ones.
//
// Scores, each with the size of its token's scales, are compared with a reference that is raised, with everything accumulated, only when one
// exceeds it by 2^kSlack: a few times per run instead of once per page.
#include <cuda_fp16.h>

#include <algorithm>

#include "activation.cuh"
#include "chain.cuh"
#include "kernels.h"
#include "kv_q4.cuh"

namespace etc {

namespace {

constexpr int kPage = 16;
constexpr int kStages = 2;
constexpr int kWarps = 4, kResident = 3;  // of a CTA; CTAs of an SM: 168 registers for a thread
// Tables of up to 32 pages take a CTA per unit. Both ways (directly / by runs, us) for sequences of half to all of 512, 768 and 1024 tokens, 32 heads over 8 of 128: one
// sequence 8.5 / 9.7, 9.9 / 9.9, 11.3 / 11.3; eight 10.4 / 11.3, 12.9 / 11.2, 15.4 / 11.7; 32 sequences 12.4 / 17.8, 15.4 / 20.0, 18.4 / 20.5. 64
// heads: one 11.6 / 11.3, 13.9 / 11.8; eight 14.1 / 13.3, 17.4 / 14.5; 32 16.2 / 19.8, 20.7 / 22.2, 24.8 / 24.2. 4 heads over 1 of 64: 6.1 / 7.8, 7.0 /
// 8.2, 7.9 / 8.2. The pages alone do not decide it: many sequences and small models are up to a quarter slower from 33 to 64 pages than a CTA
// per unit would be, eight sequences of 64 heads 6 % at 32 pages than runs would.
constexpr int kDirectPages = 32;
constexpr int kUnitPages = 6;  // what a unit costs beyond its pages, in pages
constexpr int kPartPad = 4;  // of a head's part: reference, sum of weights, two unused
// The product of weight and largest |dv| of the token that set a head's reference is 2^11, of any other token at most 2^(11 + 3.75 + 0.09)
// (0.09 by size_of), below what f16 holds.
constexpr float kSlack = 3.75f;
constexpr float kProductBits = 11.0f;
constexpr float kRest = 2048.0f;  // PAIRS: rests are held times 2^11
constexpr float kSizeZero = 15.0f;  // size_of(1)
constexpr float kNoReference = -1e38f;  // any finite score raises it, and weights under it are 0

// What a CTA has of units that other CTAs have parts of: the end of one that began before it (part 0), the beginning of one that goes on
// behind it (part 1).
struct Ends {
  int open;             // there is a part 0
  int tail;             // there is a part 1, of:
  int row, head0, heads;
  int last;             // the CTA in which that unit ends
  int unused[2];
};

struct Q4Args {
  const uint8_t* k;
  const uint8_t* v;
  const float* q;  // [B, Hq, D]
  const LaneInfo* lanes;
  const int* tables;
  float* out;      // [B, Hq, D]
  __half* out_xh;  // optional: in the hand-off layout
  int out_xh_nv;
  float* partial;  // [CTAs][2][heads of a unit][D + kPartPad]: O, then reference and sum of the weights
  struct Ends* ends;  // [CTAs]
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

// The work of all units lies in a row, lane by lane: a unit is kUnitPages places that stand for its start and end, then its pages.
__device__ __forceinline__ int places_of(int pages) { return pages > 0 ? pages + kUnitPages : 0; }

// Places of one unit of every lane, by every warp for itself.
__device__ __forceinline__ long long all_places(const Q4Args& a) {
  long long sum = 0;
  for (int i = threadIdx.x & 31; i < a.batch; i += 32) sum += places_of(span_of(a.lanes[i], a.op_window).pages);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  return sum;
}
// The lane that holds the place `at`, and how many places come before it.
__device__ __forceinline__ void lane_at(const Q4Args& a, long long at, int units, int* found, long long* before) {
  long long base = 0;
  for (int i0 = 0; i0 < a.batch; i0 += 32) {
    const int i = i0 + (threadIdx.x & 31);
    const long long mine = i < a.batch ? (long long)places_of(span_of(a.lanes[i], a.op_window).pages) * units : 0;
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

// A record of K and one of V by a warp, 16 bytes per lane and instruction; `rest`: this lane has some of what is left over 512s.
template <int RECORD>
__device__ __forceinline__ void copy_records(unsigned dst, const uint8_t* k, const uint8_t* v, int rest) {
  static_assert(RECORD == 1152 || RECORD == 576, "16 rows of 128 or 64 values");
  if constexpr (RECORD == 1152) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "cp.async.cg.shared.global [%0], [%1], 16;\n\t"
        "cp.async.cg.shared.global [%0+512], [%1+512], 16;\n\t"
        "@p cp.async.cg.shared.global [%0+1024], [%1+1024], 16;\n\t"
        "cp.async.cg.shared.global [%0+1152], [%2], 16;\n\t"
        "cp.async.cg.shared.global [%0+1664], [%2+512], 16;\n\t"
        "@p cp.async.cg.shared.global [%0+2176], [%2+1024], 16;\n\t}" ::"r"(dst), "l"(k), "l"(v), "r"(rest)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "cp.async.cg.shared.global [%0], [%1], 16;\n\t"
        "@p cp.async.cg.shared.global [%0+512], [%1+512], 16;\n\t"
        "cp.async.cg.shared.global [%0+576], [%2], 16;\n\t"
        "@p cp.async.cg.shared.global [%0+1088], [%2+512], 16;\n\t}" ::"r"(dst), "l"(k), "l"(v), "r"(rest)
        : "memory");
  }
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {  // onto zeros
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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
// A value that all lanes have, as one that the compiler knows them to have.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 halves(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// Constants of the widening, each in a register of its own: as immediates they would cost an instruction more per use.
struct Widen {
  uint32_t exponent, bias, sixteenth, shift;
  __device__ __forceinline__ Widen() {
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(exponent));   // 1024 in both halves
    asm volatile("mov.b32 %0, 0xE408E408;" : "=r"(bias));       // -1032
    asm volatile("mov.b32 %0, 0x2C002C00;" : "=r"(sixteenth));  // 1 / 16
    asm volatile("mov.b32 %0, 0xD480D480;" : "=r"(shift));      // -72
  }
  // Codes in bits 0-3 (LOW) or 4-7 of both halves of w -> two f16 numbers code - 8, exact: 1024 + code less 1032, or 1024 + 16 code over 16.
  template <bool LOW>
  __device__ __forceinline__ uint32_t get(uint32_t w) const {
    uint32_t r;
    if (LOW) {
      asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(exponent));
      return bits(__hadd2(halves(r), halves(bias)));
    }
    asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(exponent));
    return bits(__hfma2(halves(r), halves(sixteenth), halves(shift)));
  }
};
// 2^k with |x| 2^k in [2^13, 2^14), for a finite x that is not 0; 1 otherwise.
__device__ __forceinline__ float to_f16_range(float x) {
  const int e = (int)((__float_as_uint(x) >> 23) & 255u);
  if (e == 255 || x == 0.0f) return 1.0f;
  return __uint_as_float((unsigned)min(max(127 + 13 - (e - 127), 1), 254) << 23);
}

// Column k of a lane's output row.
__device__ __forceinline__ void store_out(const Q4Args& a, int D, int row, int k, float val) {
  if (a.out) a.out[(size_t)row * a.q_heads * D + k] = val;
  if (a.out_xh) a.out_xh[hand_off_cell(k >> 3, row, a.out_xh_nv, a.q_heads * (D / 8)) + (k & 7)] = half_sat(val);
}

// log2 of an f16 number that is not negative, plus 15: its bits as a number, over 1024. Exact at powers of two, up to 0.09 too large
// between them and, below 2^-14, by what keeps it from falling under 0.
__device__ __forceinline__ float size_of(uint32_t bits, unsigned place) {  // place: 0x7410 for the low half of `bits`, 0x7432 for the high one
  return fmaf(__uint_as_float(__byte_perm(bits, 0x4B000000u, place)), 1.0f / 1024.0f, -8192.0f);  // 2^23 + bits
}

template <int D, bool PAIRS>
struct Q4Cfg {
  static constexpr int kBlocks = D / 32;
  static constexpr int kCodes = kPage * D / 2;                  // code bytes of a record
  static constexpr int kRecord = kCodes + kPage * kBlocks * 2;
  static constexpr int kTogether = PAIRS ? 2 : 1;               // pages that a warp takes at once
  static constexpr int kBoth = 2 * kRecord;                     // K, then V
  static constexpr int kStage = kTogether * kBoth;
  static constexpr int kHeads = PAIRS ? 4 : 8;
  static constexpr int kPitch = D + 8;                          // of a head's partial sums: no bank conflicts
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr size_t kSmem = kRing + (size_t)2 * kWarps * kHeads * (kPitch + 2) * sizeof(float);
};

// N words (1, 2 or 4) from shared memory, aligned to their size.
template <int N>
__device__ __forceinline__ void load_words(uint32_t* dst, const unsigned char* src) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
  else dst[0] = *reinterpret_cast<const uint32_t*>(src);
}

// What a warp has of a unit that lies not wholly in its run.
struct Record {
  int valid, ends;     // ends: the unit's last page is in it
  int row, head0, heads;
  long long end;       // the place where the unit ends
};

// A warp's run of work: the unit it is in and its pages there.
struct Cursor {
  long long at, stop;  // the places where the unit, or the run, ends
  int lane, unit;      // unit: KV head * groups + group
  Span span;
  int table;
  int page0, page1;    // this run's pages of the unit (block-table indexes)
};

template <int D, bool PAIRS>
__global__ void __launch_bounds__(kWarps * 32, kResident) attention_q4_kernel(Q4Args a) {
  using Cfg = Q4Cfg<D, PAIRS>;
  constexpr int NB = Cfg::kBlocks, PAGES = Cfg::kTogether, MINE = PAIRS ? 1 : 2;  // MINE: heads whose scores a thread holds: t, or 2 t and 2 t + 1
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = uniform(threadIdx.x >> 5), g = lane >> 2, t = lane & 3;
  const int units = a.kv_heads * a.groups, G = a.q_heads / a.kv_heads;
  chain_release();
  chain_wait();

  Cursor run;
  auto enter = [&](Cursor& c) {  // c.lane, c.unit and c.at are set; page0 relative to the unit's first page
    const LaneInfo info = a.lanes[c.lane];
    const Span span = span_of(info, a.op_window);
    c.span = {uniform(span.begin), uniform(span.end), uniform(span.first), uniform(span.pages)};
    c.table = uniform(info.table_offset);
  };
  // the part of the unit from its place `skipped` on; it may hold no page
  auto clip = [&](Cursor& c, int skipped) {
    const int places = c.span.pages + kUnitPages, upto = (int)min((long long)places, skipped + (c.stop - c.at));
    c.page0 = uniform(c.span.first + max(skipped - kUnitPages, 0));
    c.page1 = uniform(c.span.first + max(upto - kUnitPages, 0));
    c.at += upto - skipped;  // where the next unit begins
  };
  // the next unit of the run of which it has pages; false when there is none
  auto advance = [&](Cursor& c) {
    while (c.at < c.stop) {
      if (++c.unit == units) {
        c.unit = 0;
        do ++c.lane; while (c.lane < a.batch && span_of(a.lanes[c.lane], a.op_window).pages == 0);
        if (c.lane >= a.batch) return false;
        enter(c);
      }
      clip(c, 0);
      if (c.page0 < c.page1) return true;
    }
    return false;
  };
  if (!a.direct) {  // lanes with nothing to attend over
    for (int l = blockIdx.x; l < a.batch; l += gridDim.x)
      if (span_of(a.lanes[l], a.op_window).pages == 0)
        for (int i = threadIdx.x; i < a.q_heads * D; i += kWarps * 32) store_out(a, D, l, i, 0.0f);
  }
  __shared__ long long total_places;
  __shared__ Record records[2 * kWarps];  // of each warp the unit that began before its run, the unit that goes on behind it
  if (lane < 2) records[2 * warp + lane].valid = 0;
  bool works = true;
  if (a.direct) {
    run.lane = blockIdx.x / units;
    run.unit = blockIdx.x - run.lane * units;
    enter(run);
    if (run.span.pages == 0) {  // nothing to attend over
      const int kv_head = run.unit / a.groups, head0 = kv_head * G + (run.unit - kv_head * a.groups) * a.heads;
      for (int i = threadIdx.x; i < min(a.heads, (kv_head + 1) * G - head0) * D; i += kWarps * 32) store_out(a, D, run.lane, head0 * D + i, 0.0f);
      return;
    }
    const int from = run.span.pages * warp / kWarps;
    run.at = kUnitPages + from;
    run.stop = kUnitPages + run.span.pages * (warp + 1) / kWarps;
    works = run.at < run.stop;
    clip(run, kUnitPages + from);
  } else {
    const long long total = all_places(a) * units;
    if (threadIdx.x == 0) total_places = total;
    const int runs = (int)gridDim.x * kWarps, mine = (int)blockIdx.x * kWarps + warp;
    const long long begin = total * mine / runs;
    run.stop = total * (mine + 1) / runs;
    works = begin < run.stop;
    if (works) {
      long long before;
      lane_at(a, begin, units, &run.lane, &before);
      enter(run);
      run.at = begin;
      const long long inside = begin - before;
      const int places = places_of(run.span.pages);
      run.unit = (int)(inside / places);
      clip(run, (int)(inside - (long long)run.unit * places));
      works = run.page0 < run.page1 || advance(run);
    }
  }

  // the ring: this warp's pages, from `ahead`, the cursor that copies are issued from; the number of the page that comes next is
  // looked up one copy ahead
  unsigned char* ring = smem + warp * (kStages * Cfg::kStage);
  const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring) + lane * 16;
  Cursor ahead = run;
  int ahead_page = run.page0;
  unsigned ahead_number[PAGES] = {};
  const uint8_t *ahead_k, *ahead_v;  // page 0 of the unit's KV head, this lane's 16 bytes
  bool more = works;
  const unsigned page_stride = (unsigned)(a.kv_heads * Cfg::kRecord);
  auto aim = [&] {
    const size_t from = (size_t)(ahead.unit / a.groups) * Cfg::kRecord + lane * 16;
    ahead_k = a.k + from;
    ahead_v = a.v + from;
  };
  auto look_up = [&] {
    while (more && ahead_page >= ahead.page1) {
      more = advance(ahead);
      ahead_page = ahead.page0;
      aim();
    }
    if (!more) return;
#pragma unroll
    for (int u = 0; u < PAGES; ++u)  // what lies behind the last page is that page again, and masked
      ahead_number[u] = (unsigned)a.tables[ahead.table + min(ahead_page + u, ahead.page1 - 1)];
  };
  if (works) {
    aim();
    look_up();
  }
  const int rest = lane * 16 < Cfg::kRecord % 512;
  auto copy = [&](unsigned offset) {
#pragma unroll
    for (int u = 0; u < PAGES; ++u) {
      const unsigned long long from = (unsigned long long)ahead_number[u] * page_stride;
      copy_records<Cfg::kRecord>(ring_at + offset + u * Cfg::kBoth, ahead_k + from, ahead_v + from, rest);
    }
    ahead_page += PAGES;
  };
  auto issue = [&](unsigned offset) {
    if (more) {
      copy(offset);
      look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  unsigned fill = 0, at = 0;  // ring offsets of the next copy and of the page at hand
  auto step = [](unsigned& offset) { offset = offset == (kStages - 1) * Cfg::kStage ? 0 : offset + Cfg::kStage; };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    issue(fill);
    step(fill);
  }

  float* sums = reinterpret_cast<float*>(smem + Cfg::kRing);  // [record][head][pitch], then references and weights [record][head]
  float* refs = sums + 2 * kWarps * Cfg::kHeads * Cfg::kPitch;
  float* weights = refs + 2 * kWarps * Cfg::kHeads;
  const Widen widen;
  const bool wide_q = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
  while (works) {
    const int kv_head = run.unit / a.groups, head0 = kv_head * G + (run.unit - kv_head * a.groups) * a.heads;
    const int live_heads = min(a.heads, (kv_head + 1) * G - head0);
    // queries: column g is the value (g even) or the rest (g odd) of head g / 2, or value and rest, one after the other, of head g
    uint32_t qf[PAIRS ? 1 : 2][NB][2][2];
    float unscale[MINE];
    {
      const int h = PAIRS ? g >> 1 : g;
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
#pragma unroll
      for (int m = 0; m < MINE; ++m) unscale[m] = __shfl_sync(0xffffffffu, a.scale_log2 / f, PAIRS ? 8 * t : 4 * (2 * t + m));
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float u = f * (p ? x[b][s].z : x[b][s].x), v = f * (p ? x[b][s].w : x[b][s].y);
            const __half2 value = __floats2half2_rn(u, v), rest = __floats2half2_rn(u - __low2float(value), v - __high2float(value));
            if constexpr (PAIRS) {
              qf[0][b][s][p] = (g & 1) == 0 ? bits(value) : bits(rest);
            } else {
              qf[0][b][s][p] = bits(value);
              qf[1][b][s][p] = bits(rest);
            }
          }
    }
    float o[2 * NB][4];
    float sub[MINE], weight[MINE];  // what weights' exponents are less than scores, by the reference; this thread's sum of weights
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      sub[m] = kNoReference;
      weight[m] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    // this run's positions of the unit, and the pages of it without a masked token
    const int end_of_run = min(run.span.end, run.page1 * kPage), inner0 = (run.span.begin + kPage - 1) / kPage, inner1 = end_of_run / kPage;

    // while the copies are in this unit too, and whole, the next numbers are in its table
    const bool together = more && ahead.lane == run.lane && ahead.unit == run.unit;
    const int close = uniform(together ? run.page0 + run.page1 - (2 * PAGES - 1) - ahead_page : run.page0);
    const int* table = a.tables + run.table;
    for (int page = run.page0; page < run.page1; page += PAGES) {
      if (page < close) {
        copy(fill);
#pragma unroll
        for (int u = 0; u < PAGES; ++u) ahead_number[u] = (unsigned)table[ahead_page + u];
        asm volatile("cp.async.commit_group;" ::: "memory");
      } else {
        issue(fill);
      }
      step(fill);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const unsigned char *codes = ring + at + g * (D / 2) + t * (4 * NB), *scales = ring + at + Cfg::kCodes + g * (2 * NB);

      // scores of tokens g and g + 8 of each page
      float s_lo[PAGES][MINE], s_hi[PAGES][MINE];
      __align__(8) uint32_t dv_lo[PAGES][NB / 2], dv_hi[PAGES][NB / 2];
#pragma unroll
      for (int u = 0; u < PAGES; ++u) {
#pragma unroll
        for (int m = 0; m < MINE; ++m) s_lo[u][m] = s_hi[u][m] = 0.0f;
        __align__(16) uint32_t w_lo[NB], w_hi[NB];
        __align__(8) uint32_t d_lo[NB / 2], d_hi[NB / 2];
        load_words<NB>(w_lo, codes + u * Cfg::kBoth);
        load_words<NB>(w_hi, codes + u * Cfg::kBoth + 8 * (D / 2));
        load_words<NB / 2>(d_lo, scales + u * Cfg::kBoth);
        load_words<NB / 2>(d_hi, scales + u * Cfg::kBoth + 8 * (2 * NB));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t x = w_lo[b], y = w_hi[b], x8 = x >> 8, y8 = y >> 8;
          const uint32_t a00 = widen.get<true>(x), a01 = widen.get<true>(y), a02 = widen.get<false>(x), a03 = widen.get<false>(y);
          const uint32_t a10 = widen.get<true>(x8), a11 = widen.get<true>(y8), a12 = widen.get<false>(x8), a13 = widen.get<false>(y8);
          const float2 dl = __half22float2(halves(d_lo[b / 2])), dh = __half22float2(halves(d_hi[b / 2]));
          const float d0 = b & 1 ? dl.y : dl.x, d1 = b & 1 ? dh.y : dh.x;
          float c[4];
          mma_first(c, a00, a01, a02, a03, qf[0][b][0][0], qf[0][b][0][1]);
          mma(c, a10, a11, a12, a13, qf[0][b][1][0], qf[0][b][1][1]);
          if constexpr (PAIRS) {
            s_lo[u][0] = fmaf(d0, c[0] + c[1], s_lo[u][0]);
            s_hi[u][0] = fmaf(d1, c[2] + c[3], s_hi[u][0]);
          } else {
            mma(c, a00, a01, a02, a03, qf[1][b][0][0], qf[1][b][0][1]);
            mma(c, a10, a11, a12, a13, qf[1][b][1][0], qf[1][b][1][1]);
#pragma unroll
            for (int m = 0; m < MINE; ++m) {
              s_lo[u][m] = fmaf(d0, c[m], s_lo[u][m]);
              s_hi[u][m] = fmaf(d1, c[2 + m], s_hi[u][m]);
            }
          }
        }
        load_words<NB / 2>(dv_lo[u], scales + u * Cfg::kBoth + Cfg::kRecord);
        load_words<NB / 2>(dv_hi[u], scales + u * Cfg::kBoth + Cfg::kRecord + 8 * (2 * NB));
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
          s_lo[u][m] *= unscale[m];
          s_hi[u][m] *= unscale[m];
        }
      }
      if (page < inner0 || page + PAGES > inner1) {
        // a masked token's rows may hold anything: neither its score nor its scales are looked at
#pragma unroll
        for (int u = 0; u < PAGES; ++u) {
          const int pos_lo = (page + u) * kPage + g, pos_hi = pos_lo + 8;
          const bool live_lo = pos_lo >= run.span.begin && pos_lo < end_of_run, live_hi = pos_hi >= run.span.begin && pos_hi < end_of_run;
#pragma unroll
          for (int m = 0; m < MINE; ++m) {
            if (!live_lo) s_lo[u][m] = -INFINITY;
            if (!live_hi) s_hi[u][m] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < NB / 2; ++i) {
            if (!live_lo) dv_lo[u][i] = 0u;
            if (!live_hi) dv_hi[u][i] = 0u;
          }
        }
      }
      // The size of a token: its largest |dv| of any block, as a logarithm.
      auto sizes_of = [&](int u, auto&& of, float& lo, float& hi) {
        __half2 most_lo = of(__habs2(halves(dv_lo[u][0]))), most_hi = of(__habs2(halves(dv_hi[u][0])));
        if constexpr (NB == 4) {
          most_lo = __hmax2(most_lo, of(__habs2(halves(dv_lo[u][1]))));
          most_hi = __hmax2(most_hi, of(__habs2(halves(dv_hi[u][1]))));
        }
        const uint32_t both = bits(__hmax2(__lows2half2(most_lo, most_hi), __highs2half2(most_lo, most_hi)));
        lo = size_of(both, 0x7410u);
        hi = size_of(both, 0x7432u);
      };
      constexpr float kMost = kProductBits + kSizeZero + kSlack;  // of a weight's exponent and its token's size together
      bool rises = false;
#pragma unroll
      for (int u = 0; u < PAGES; ++u) {
        float lo, hi;
        sizes_of(u, [](__half2 d) { return d; }, lo, hi);
#pragma unroll
        for (int m = 0; m < MINE; ++m) rises = rises || !(s_lo[u][m] - sub[m] + lo <= kMost) || !(s_hi[u][m] - sub[m] + hi <= kMost);
      }
      if (__any_sync(0xffffffffu, rises)) {
        float f[MINE];
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
          float most = -INFINITY;
#pragma unroll
          for (int u = 0; u < PAGES; ++u) {
            // an infinite scale spoils the columns of its block, and nothing else: it takes no part in the token's size
            float lo, hi;
            sizes_of(u, [](__half2 d) { return __halves2half2(__hisinf(__low2half(d)) ? __half() : __low2half(d), __hisinf(__high2half(d)) ? __half() : __high2half(d)); }, lo, hi);
            most = fmaxf(most, fmaxf(s_lo[u][m] + lo, s_hi[u][m] + hi));
          }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
          f[m] = 1.0f;
          if (most - sub[m] > kMost) {  // each head for itself: its result does not depend on the others
            float to = most - (kProductBits + kSizeZero);
            if (most - to > kProductBits + kSizeZero + 0.5f) to = most;  // scores so large that f32 does not resolve the difference
            f[m] = exp2_flushed(sub[m] - to);
            sub[m] = to;
          }
          weight[m] *= f[m];
        }
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          o[i][0] *= f[0]; o[i][1] *= f[MINE - 1]; o[i][2] *= f[0]; o[i][3] *= f[MINE - 1];
        }
      }
#pragma unroll
      for (int u = 0; u < PAGES; ++u) {
        // Weights, and their products with the V scales as value and rest, transposed into operand order.
        uint32_t pf[PAIRS ? 1 : 2][NB][2];
        float p_lo[MINE], p_hi[MINE];
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
          p_lo[m] = exp2_flushed(s_lo[u][m] - sub[m]);
          p_hi[m] = exp2_flushed(s_hi[u][m] - sub[m]);
          weight[m] += p_lo[m] + p_hi[m];
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float2 lo = __half22float2(halves(dv_lo[u][b / 2])), hi = __half22float2(halves(dv_hi[u][b / 2]));
          const float d0 = b & 1 ? lo.y : lo.x, d1 = b & 1 ? hi.y : hi.x;
          if constexpr (PAIRS) {
            auto both = [](float x) {
              const float value = __half2float(__float2half_rn(x));
              return transpose8(bits(__floats2half2_rn(value, (x - value) * kRest)));
            };
            pf[0][b][0] = both(p_lo[0] * d0);
            pf[0][b][1] = both(p_hi[0] * d1);
          } else {
            auto both = [&](float x0, float x1, int i) {  // of two heads
              const __half2 value = __floats2half2_rn(x0, x1);
              pf[0][b][i] = transpose8(bits(value));
              pf[1][b][i] = transpose8(bits(__floats2half2_rn(x0 - __low2float(value), x1 - __high2float(value))));
            };
            both(p_lo[0] * d0, p_lo[1] * d0, 0);
            both(p_hi[0] * d1, p_hi[1] * d1, 1);
          }
        }
        __align__(16) uint32_t w[2][NB];  // of tokens 2 t and 2 t + 1, and of those eight further
        const unsigned char* v_codes = ring + at + u * Cfg::kBoth + Cfg::kRecord + t * D + g * (4 * NB);
        load_words<NB>(w[0], v_codes);
        load_words<NB>(w[1], v_codes + 4 * D);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t x = w[0][b], y = w[1][b], x8 = x >> 8, y8 = y >> 8;
          const uint32_t a00 = widen.get<true>(x), a01 = widen.get<false>(x), a02 = widen.get<true>(y), a03 = widen.get<false>(y);
          const uint32_t a10 = widen.get<true>(x8), a11 = widen.get<false>(x8), a12 = widen.get<true>(y8), a13 = widen.get<false>(y8);
#pragma unroll
          for (int p = 0; p < (PAIRS ? 1 : 2); ++p) {
            mma(o[2 * b], a00, a01, a02, a03, pf[p][b][0], pf[p][b][1]);
            mma(o[2 * b + 1], a10, a11, a12, a13, pf[p][b][0], pf[p][b][1]);
          }
        }
      }
      __syncwarp();
      step(at);
    }

    // a whole unit is written, a part of one kept for the end
    const bool begins = run.page0 == run.span.first, ends = run.page1 == run.span.first + run.span.pages;
    const int record = 2 * warp + (begins ? 1 : 0);
    if (lane == 0 && !(begins && ends)) records[record] = Record{1, ends, run.lane, head0, live_heads, run.stop + (run.span.first + run.span.pages - run.page1)};
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) weight[m] += __shfl_xor_sync(0xffffffffu, weight[m], off);
      const int h = PAIRS ? t : 2 * t + m;
      const float f = begins && ends ? (weight[m] == 0.0f ? 0.0f : 1.0f / weight[m]) : 1.0f;  // the powers of two in both cancel
      float* dst = sums + (record * Cfg::kHeads + h) * Cfg::kPitch + g;
#pragma unroll
      for (int i = 0; i < 4 * NB; ++i) {  // columns 8 i + g
        const float val = (PAIRS ? fmaf(o[i / 2][2 * (i & 1) + 1], 1.0f / kRest, o[i / 2][2 * (i & 1)]) : o[i / 2][2 * (i & 1) + m]) * f;
        if (!(begins && ends)) dst[8 * i] = val;
        else if (h < live_heads) store_out(a, D, run.lane, (head0 + h) * D + 8 * i + g, val);
      }
      if (g == 0) {
        refs[record * Cfg::kHeads + h] = sub[m];
        weights[record * Cfg::kHeads + h] = weight[m];
      }
    }
    works = advance(run);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // Units that more than one warp has: a record of a unit that begins in this CTA, or the first of one that began before it, and the records
  // behind it up to the unit's end.
  const bool mine = lane < 2 * kWarps && records[lane % (2 * kWarps)].valid;
  unsigned left = __ballot_sync(0xffffffffu, mine);
  const unsigned last = __ballot_sync(0xffffffffu, mine && records[lane % (2 * kWarps)].ends);
  Ends mine_of = {};
  while (left) {
    const int k = __ffs(left) - 1, end = __ffs(left & last);  // 0: the unit goes on behind this CTA
    const bool open = (k & 1) == 0;                           // it began in an earlier one
    const unsigned members = end ? left & (0xffffffffu >> (32 - end)) : left;
    left &= ~members;
    const Record first = records[k];
    if (open) {
      mine_of.open = 1;
    } else if (!end) {
      mine_of.tail = 1;
      mine_of.row = first.row;
      mine_of.head0 = first.head0;
      mine_of.heads = first.heads;
      // a run holds the places from total * run / runs on
      const long long place = records[31 - __clz(members)].end - 1;
      mine_of.last = (int)(((place + 1) * ((int)gridDim.x * kWarps) - 1) / total_places) / kWarps;
    }
    for (int i = threadIdx.x; i < first.heads * D; i += kWarps * 32) {
      const int h = i / D, d = i - h * D;
      float ref[kWarps], m = -INFINITY, acc = 0.0f, l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int r = w == k / 2 ? k : 2 * w;
        ref[w] = members >> r & 1 ? refs[r * Cfg::kHeads + h] : -INFINITY;
        m = fmaxf(m, ref[w]);
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int r = w == k / 2 ? k : 2 * w;
        const float f = ref[w] == -INFINITY ? 0.0f : exp2_flushed(ref[w] - m);
        if (members >> r & 1) {
          acc = fmaf(f, sums[(r * Cfg::kHeads + h) * Cfg::kPitch + d], acc);
          l = fmaf(f, weights[r * Cfg::kHeads + h], l);
        }
      }
      if (!open && end) {
        store_out(a, D, first.row, (first.head0 + h) * D + d, l == 0.0f ? 0.0f : acc / l);
      } else {
        float* dst = a.partial + ((size_t)(2 * blockIdx.x + (open ? 0 : 1)) * a.heads + h) * (D + kPartPad);
        dst[d] = acc;
        if (d == 0) { dst[D] = m; dst[D + 1] = l; }
      }
    }
  }
  if (!a.direct && threadIdx.x == 0) a.ends[blockIdx.x] = mine_of;
}

// Adds up the parts of units that were cut: grid (heads of a unit, CTAs of the attention kernel), a CTA for the unit that goes on behind
// its namesake, if there is one. Latency-bound: four warps take the parts in turn, four at a time, a thread D / 32 columns of them; a
// reference is fetched with its part. (One CTA per unit, a part after the other: 150 of 182 us for one lane in 37 parts; a CTA for every unit and
// head, which worked out by 64-bit divisions whether its unit was cut: 14 us for 64 lanes.)
constexpr int kMergeWarps = 4, kMergeParts = 4;
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) attention_q4_merge_kernel(Q4Args a) {
  __shared__ __align__(16) float sums[kMergeWarps][D];
  __shared__ float refs[kMergeWarps], weights[kMergeWarps];
  constexpr int COLUMNS = D / 32;  // of a thread
  chain_release();
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.x, c0 = blockIdx.y;
  const Ends own = a.ends[c0];
  if (!own.tail || h >= own.heads) return;
  float m = -INFINITY, l = 0.0f, acc[COLUMNS] = {};
  for (int first = c0 + warp; first <= own.last; first += kMergeWarps * kMergeParts) {
    float x[kMergeParts][COLUMNS], r[kMergeParts], w[kMergeParts];
    bool there[kMergeParts];  // with more CTAs than places some have no part
#pragma unroll
    for (int u = 0; u < kMergeParts; ++u) {
      const int c = min(first + u * kMergeWarps, own.last);
      const float* part = a.partial + ((size_t)(2 * c + (c == c0 ? 1 : 0)) * a.heads + h) * (D + kPartPad);
#pragma unroll
      for (int j = 0; j < COLUMNS; ++j) x[u][j] = part[lane + 32 * j];
      r[u] = part[D];
      w[u] = part[D + 1];
      there[u] = first + u * kMergeWarps <= own.last && (c == c0 || a.ends[c].open);
    }
#pragma unroll
    for (int u = 0; u < kMergeParts; ++u) {
      if (!there[u]) continue;
      const float to = fmaxf(m, r[u]), old = m == -INFINITY ? 0.0f : exp2_flushed(m - to), f = r[u] == -INFINITY ? 0.0f : exp2_flushed(r[u] - to);
      m = to;
      l = l * old + w[u] * f;
#pragma unroll
      for (int j = 0; j < COLUMNS; ++j) acc[j] = acc[j] * old + x[u][j] * f;
    }
  }
#pragma unroll
  for (int j = 0; j < COLUMNS; ++j) sums[warp][lane + 32 * j] = acc[j];
  if (lane == 0) { refs[warp] = m; weights[warp] = l; }
  __syncthreads();
  if (threadIdx.x >= D) return;
  float most = -INFINITY, sum = 0.0f, weight = 0.0f;
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) most = fmaxf(most, refs[w]);
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) {
    const float f = refs[w] == -INFINITY ? 0.0f : exp2_flushed(refs[w] - most);
    sum += f * sums[w][threadIdx.x];
    weight += f * weights[w];
  }
  store_out(a, D, own.row, (own.head0 + h) * D + threadIdx.x, weight == 0.0f ? 0.0f : sum / weight);
}

// Query heads of a KV head in groups of at most eight: with more the accumulators of a warp do not fit its registers.
int head_groups(int q_heads, int kv_heads) { return (q_heads / kv_heads + 7) / 8; }

template <int D, bool PAIRS>
cudaError_t launch_t(const Q4Args& a, unsigned ctas, cudaStream_t stream) {
  auto kernel = attention_q4_kernel<D, PAIRS>;
  constexpr size_t smem = Q4Cfg<D, PAIRS>::kSmem;
  const cudaError_t e = opt_in_shared_memory(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, dim3(ctas), dim3(kWarps * 32), smem, stream, a);
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
  p.direct = max_pages <= kDirectPages;
  // as many CTAs as are resident at once, but two pages for every warp where the tables are short
  p.ctas = p.direct ? units : std::min<int64_t>((int64_t)kResident * sm_count, (units * max_pages + 2 * kWarps - 1) / (2 * kWarps));
  p.scratch_bytes = p.direct ? 0 : (size_t)p.ctas * (2 * heads * (head_dim + kPartPad) * sizeof(float) + sizeof(Ends));
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
  a.batch = batch;
  a.q_heads = q_heads;
  a.kv_heads = pool.kv_heads;
  a.groups = head_groups(q_heads, pool.kv_heads);
  a.heads = (q_heads / pool.kv_heads + a.groups - 1) / a.groups;
  a.partial = scratch;
  a.ends = reinterpret_cast<Ends*>(scratch + (size_t)plan.ctas * 2 * a.heads * (pool.head_dim + kPartPad));
  a.direct = plan.direct;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.op_window = op_window;
  const unsigned ctas = (unsigned)plan.ctas;
  cudaError_t e;
  if (a.heads <= 4) e = pool.head_dim == 128 ? launch_t<128, true>(a, ctas, stream) : launch_t<64, true>(a, ctas, stream);
  else e = pool.head_dim == 128 ? launch_t<128, false>(a, ctas, stream) : launch_t<64, false>(a, ctas, stream);
  if (e != cudaSuccess) return e;
  if (launches) ++*launches;
  if (plan.direct) return cudaSuccess;
  e = launch_chained(pool.head_dim == 128 ? attention_q4_merge_kernel<128> : attention_q4_merge_kernel<64>, dim3((unsigned)a.heads, ctas), dim3(kMergeWarps * 32), 0,
                     stream, a);
  if (e == cudaSuccess && launches) ++*launches;
  return e;
}

}  // namespace etc
