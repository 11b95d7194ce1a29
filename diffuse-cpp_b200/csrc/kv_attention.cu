// kv_attention.cu — dmoe_kv_attention: softmax attention over a paged key/value cache.
//
// Reference: src/diffuse-moe-graph.cpp:163-175 under the block-causal mask :38-52. For a query row at
// position p, o = sum_j w_j v_j / sum_j w_j over the positions j < min(kv_len, (p / block + 1) block),
// w_j = exp(scale q.k_j). The rows of the query heads that share a key/value head (n_head / n_head_kv
// heads x the sequence's queries) read the same keys: they form one matrix, so that a page is read once
// for all of them.
//
// One pass with a running maximum. In 8-bit pages k = 2^ek kc, v = 2^ev vc with e4m3 kc, vc, one ek and ev
// for every 32 positions; e4m3 is exact in f16, so the products run in f16 on the codes:
//   t_j = log2(e) scale 2^ek (q.kc_j) + ev,  M = max t_j,  p_j = 2^(t_j - M),
//   o = sum p_j vc_j / sum p_j 2^-ev.
// The value scale rides in the exponent, so p is rounded to f16 relative to the largest weight times value
// scale. f16 has 30 binades of whole precision: M is held below the true maximum (kLift), so that the largest
// weights are near f16's top and those of positions beside one that takes nearly all the weight (an attention
// sink, whose value is often next to zero) are not rounded to a few bits. Queries are brought into [-1, 1] by a
// power of two per row (exact). M and both sums are 32-bit; p is rounded once, to the products' type.
//
// Work split: the tiles of all (sequence, row tile, key/value head) items are numbered through, and every
// CTA takes an equal run of them, whatever the lengths: a long sequence spreads over the GPU and short
// ones share a CTA. An item that spans CTAs leaves partial (o, M, sum) triples in the workspace, which
// kv_combine_kernel adds in a fixed order (results do not depend on timing).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>

#include "dmoe_internal.h"
#include "kv_common.cuh"
#include "sm100.cuh"

namespace dmoe {

namespace {

constexpr int kMaxGrid = 148;  // one CTA an SM
// The least factor of a score. Operands are at most 4 (queries) and 65504, so below it no score counts
constexpr float kTinyFactor = 0x1p-126f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// An item that a CTA begins and does not end
struct Spanning {
  int last;  // CTA that ends it; -1: there is none
  int row0, row_lo, rows, head;  // the sequence's first row, the item's rows [row_lo, row_lo + rows) of q_len * group
  int pad[3];
};

// Weights of f16 products are 2^kLift times what they are of the maximum's: up to 2^15. The tiles let them grow to that
// before their reference follows the maximum, so it begins 2^8 lower. bf16 has the range as it is.
template <int KV>
struct Lift {
  static constexpr float kRows = KV == KV_BF16 ? 0.f : 15.f;
  static constexpr float kTiles = KV == KV_BF16 ? 0.f : 7.f, kGrown = kTiles + 8.f;
};

struct AttnParams {
  KvPages pg;
  KvBatch b;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int64_t q_stride, out_stride;
  int is_bf16;       // type of q and out
  int n_head, group;
  uint32_t group_magic;  // ceil(2^28 / group): x / group for x < 2^13 and group <= 2^12 (x * error < 2^28)
  int block_length;
  int n_qt;          // row tiles a sequence can have (max_q_len)
  int whole;         // items are not split: no partial triples, no second kernel
  int vec_q, vec_q16, vec_out16;  // q rows allow 8-byte, 16-byte loads; out rows 16-byte stores
  float scale_log2;  // scale * log2(e)
  uint32_t* wait_err;  // word that bounded waits report to
  float* part;       // partial triples, slot = 2 * CTA + (the item begins in this CTA)
  struct Spanning* desc;  // [CTA]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the largest of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// two floats as one 64-bit operand of the packed fma and add
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^e for |e| <= 126
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// ---------------------------------------------------------------------------------------------
// schedule
// ---------------------------------------------------------------------------------------------
struct Item {
  KvSeq q;
  int seq, row_lo, rows;  // rows [row_lo, row_lo + rows) of the sequence's q_len * group
  int tiles;              // 0: no such item
};

__device__ __forceinline__ int row_limit(const AttnParams& p, const KvSeq& q, int row) {
  const int pos = q.kv_len - q.q_len + row / p.group;
  if (pos < 0) return 0;
  return (int)min((int64_t)q.kv_len, ((int64_t)(pos / p.block_length) + 1) * p.block_length);
}

template <int R, int TILE>
__device__ __forceinline__ Item item_of(const AttnParams& p, int u) {
  Item it;
  it.seq = p.n_qt == 1 ? u : u / p.n_qt;
  it.q = kv_sequence(p.b, p.pg, it.seq);
  it.row_lo = (u - it.seq * p.n_qt) * R;
  it.rows = min(R, it.q.q_len * p.group - it.row_lo);
  it.tiles = 0;
  if (it.rows > 0) it.tiles = max(1, (row_limit(p, it.q, it.row_lo + it.rows - 1) + TILE - 1) / TILE);
  return it;
}

// Beginning and ending an item costs about as much as OV tiles. An item of t tiles is OV + t units long, and
// the units of all items are numbered through; its tiles are the last t. With p.whole an item is one unit.
// The host refuses calls whose units could number 2^31 or more; sequences that overlap (a broken q_start) could still
// have more, which find_run reports.
struct Run {   // a CTA's run of units
  Item it;     // first item
  int u, head;
  int unit;    // first unit within it
  int left;    // units of the run
  int chunk;   // units of every run but the last
  int first;   // number of the first unit
};

// The whole CTA: finds its run. sums: THREADS / 32 elements of shared memory.
template <int R, int TILE, int OV, int THREADS>
__device__ __forceinline__ Run find_run(const AttnParams& p, uint2* sums, Run* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_u = p.b.n_seq * p.n_qt;
  const int per = (n_u + THREADS - 1) / THREADS;
  const int u0 = min((int64_t)n_u, (int64_t)per * tid), u1 = min((int64_t)n_u, (int64_t)u0 + per);
  int64_t own = 0;
  for (int u = u0; u < u1; ++u) {
    const int t = item_of<R, TILE>(p, u).tiles;
    if (t) own += p.whole ? 1 : t + OV;
  }
  const uint32_t mine = (uint32_t)own;
  uint32_t incl = mine;  // sums modulo 2^32, and beside them the sum of what lies above 16 bits
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  const uint32_t above = __reduce_add_sync(0xffffffffu, (uint32_t)min(own >> 16, (int64_t)1 << 20));
  if (lane == 31) sums[warp] = make_uint2(incl, above);
  if (tid == 0) found->left = 0;
  __syncthreads();
  uint32_t before_u = incl - mine, all = 0, high = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    const uint2 v = sums[w];
    if (w < warp) before_u += v.x;
    all += v.x;
    high += v.y;
  }
  const int heads = p.pg.n_head_kv;
  // high < 2^15: the sum is below 2^31 + THREADS * 2^16, so `all` is exact
  if (high >> 15 || (uint64_t)all * heads > INT32_MAX) {  // the whole grid alike: no runs
    if (tid == 0) kv_report(p.pg.err, DMOE_KV_ERR_BATCH);
    all = 0;
  }
  const int total = (int)(all * heads);
  int before = (int)(before_u * heads);  // in range wherever there is a run
  const int chunk = (int)(((uint32_t)total + gridDim.x - 1) / gridDim.x);
  const int first = (int)min((int64_t)chunk * blockIdx.x, (int64_t)total);
  if (first < total && first >= before && first < before + (int)mine * heads) {
    for (int u = u0; u < u1; ++u) {
      const Item it = item_of<R, TILE>(p, u);
      const int w = !it.tiles ? 0 : p.whole ? 1 : it.tiles + OV;
      if (first < before + w * heads) {
        found->it = it;
        found->u = u;
        found->head = (first - before) / w;
        found->unit = (first - before) % w;
        found->left = min(chunk, total - first);
        break;
      }
      before += w * heads;
    }
  }
  __syncthreads();
  Run r = *found;
  r.chunk = chunk;
  r.first = first;
  return r;
}

// Walks a CTA's run, item by item: every warp role does it on its own. The segment at hand is the tiles
// [t0, t1) of `it`; an item of which the run only holds units before its tiles is left to the next CTA.
template <int R, int TILE, int OV>
struct Walk {
  const AttnParams& p;
  Item it;
  int u, head, seg = -1, t0 = 0, t1 = 0;
  int unit, left, chunk, at;
  __device__ __forceinline__ Walk(const AttnParams& p_, const Run& r)
      : p(p_), it(r.it), u(r.u), head(r.head), unit(r.unit), left(r.left), chunk(r.chunk), at(r.first) {
    settle();
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == it.tiles; }
  // for an item that this CTA begins and does not end
  __device__ __forceinline__ Spanning begun() const {
    return {(at - unit + OV + it.tiles - 1) / chunk, it.q.row0, it.row_lo, it.rows, head, {0, 0, 0}};
  }
  __device__ __forceinline__ void next() {
    advance();
    settle();
  }

 private:
  __device__ __forceinline__ void advance() {
    const int n = p.whole ? 1 : min(left, OV + it.tiles - unit);
    left -= n;
    at += n;
    unit = 0;
    if (left > 0 && ++head == p.pg.n_head_kv) {
      head = 0;
      do it = item_of<R, TILE>(p, ++u);
      while (it.tiles == 0);
    }
  }
  __device__ __forceinline__ void settle() {
    while (left > 0) {
      t0 = p.whole ? 0 : max(0, unit - OV);
      t1 = p.whole ? it.tiles : min(it.tiles, unit + left - OV);
      if (t1 > t0) break;
      advance();
    }
    ++seg;
  }
};

// 16 bytes that are used once: not kept in L1, whose data path the products' operands share
__device__ __forceinline__ uint4 load_past_l1(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// mbar_wait by a whole warp, with one answer: after a timeout no lane goes on alone
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t bit) {
  const bool ok = mbar_wait(bar, parity, err, bit);
  return __all_sync(0xffffffffu, ok);
}

// `bytes` (a multiple of 16, both addresses 16-byte aligned) into this CTA's shared memory
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ---------------------------------------------------------------------------------------------
// 16-bit warp products
// ---------------------------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// whether a word of a value row holds an infinity or NaN
template <int KV>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  if (KV == KV_E4M3) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
  const uint32_t e = KV == KV_BF16 ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & e, e) != 0;
}

// the i-th element of a word of a value row (a code's value in 8-bit pages)
template <int KV>
__device__ __forceinline__ float element(uint32_t w, int i) {
  if (KV == KV_E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(w >> (8 * i)), __NV_E4M3);
    return __half2float(__half(h));
  }
  const uint16_t h = (uint16_t)(w >> (16 * i));
  return KV == KV_BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}

// two e4m3 codes (the low or the high half of w) as f16
template <int HALF>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  uint32_t r;
  const uint16_t h = (uint16_t)(HALF ? w >> 16 : w);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  return r;
}

// 4 consecutive query elements as floats
__device__ __forceinline__ void load_q4(const AttnParams& p, int64_t at, float (&x)[4]) {
  uint32_t w[2];
  if (p.vec_q) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p.q + at));
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = p.q[at + 2 * i] | ((uint32_t)p.q[at + 2 * i + 1] << 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (p.is_bf16) {
      x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

__device__ __forceinline__ void store_out(const AttnParams& p, int row0, int row, int head, int d, int hd, float x) {
  const int64_t at = (int64_t)(row0 + row / p.group) * p.out_stride + (int64_t)(head * p.group + row % p.group) * hd + d;
  if (p.is_bf16)
    p.out[at] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
  else
    p.out[at] = __half_as_ushort(__float2half_rn(x));
}

__device__ __forceinline__ void store_lse(const AttnParams& p, int row0, int row, int head, float m, float l) {
  if (p.lse)
    p.lse[(int64_t)(row0 + row / p.group) * p.n_head + head * p.group + row % p.group] =
        l == 0.f ? -INFINITY : kLn2 * (m + log2f(l));
}

// ---------------------------------------------------------------------------------------------
// Few rows (single tokens): warp-level products, keys and values from global memory to registers.
//
// A tile of NT * 8 rows. s^T = K q^T with the keys as the 16-row operand and the queries as the 8-column
// one, then o^T = V^T p^T: with few rows this wastes nothing, and both operands come straight from
// 16-byte loads. The order of the elements within a product's k is free as long as both sides agree:
// for s it is the 16-byte chunk of a key row that a lane loads, for o the lane's value rows are joined
// pairwise by byte permutations. p^T goes from accumulator to operand layout by an 8 x 8 transpose.
// Bound by HBM: the bytes of the pages. A step's keys lie side by side in a page, and so do its values: each warp
// has them brought into shared memory by one bulk copy each, one or two steps ahead (no barrier but the copies' own), so
// that the latency of HBM does not show. A step's chain of dependent instructions is long, and only other warps
// hide it: as many as registers and the ring leave room for. Measured: 64 tokens over 545 K positions of e4m3
// pages (558 MB) 108 us = 5.2 TB/s, 80 % of the copy rate; one token over 131072 positions 37 us with the second kernel.
// ---------------------------------------------------------------------------------------------
template <int HD, int KV, int NT>
struct RowsCfg {
  static constexpr int kWarps = NT == 1 ? 12 : 8;  // registers: 168 or 255 a thread
  static constexpr int R = 8 * NT;
  static constexpr int MT = KV == KV_E4M3 ? 2 : 1;  // 16-position product tiles a step
  static constexpr int STEP = 16 * MT;
  static constexpr int TILE = kWarps * STEP;
  static constexpr int OV = 3;
  static constexpr int ES = KV == KV_E4M3 ? 1 : 2;
  static constexpr int kStages = kWarps == 8 ? 3 : 2;
  static constexpr int kHalf = STEP * HD * ES;  // bytes of a step's keys, and of its values
  static constexpr size_t kRing = (size_t)kWarps * kStages * 2 * kHalf;
  static constexpr size_t kJoin = (size_t)kWarps * R * (HD + 2) * 4;
  static constexpr size_t kSmem = kRing > kJoin ? kRing : kJoin;  // the ring is idle when the warps are joined
  static constexpr int kPart = R * (HD + 2);  // floats of a partial triple
};

template <int HD, int KV, int NT>
__global__ void __launch_bounds__(32 * RowsCfg<HD, KV, NT>::kWarps, 1) kv_rows_kernel(const __grid_constant__ AttnParams p) {
  using C = RowsCfg<HD, KV, NT>;
  constexpr bool kBf = KV == KV_BF16;
  constexpr int R = C::R, MT = C::MT, STEP = C::STEP, TILE = C::TILE, ES = C::ES;
  constexpr int KCH = HD * ES / 64;        // 16-byte loads of a key row by each of 4 lanes
  constexpr int VB = HD * ES / 8;          // bytes of a value row by each of 8 lanes: 8, 16 or 32
  constexpr int VW = VB / 4;
  constexpr int JT = HD / 16;              // 16-row tiles of o^T
  extern __shared__ __align__(128) float smem_f[];
  __shared__ uint2 sums[C::kWarps];
  __shared__ Run found;
  __shared__ uint64_t bar[C::kWarps][C::kStages];  // a stage's copies have arrived
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  if (lane < C::kStages) mbar_init(&bar[warp][lane], 1);
  fence_mbar_init();
  uint32_t done = 0;  // steps of the items before
  bool ok = true;     // no wait has run out
  pdl_wait();
  Spanning begun = {-1, 0, 0, 0, 0, {0, 0, 0}};
  for (Walk<R, TILE, C::OV> w(p, find_run<R, TILE, C::OV, 32 * C::kWarps>(p, sums, &found)); w.more(); w.next()) {
    const Item& it = w.it;
    const int head = w.head;
    const int lim_min = row_limit(p, it.q, it.row_lo), lim_max = row_limit(p, it.q, it.row_lo + it.rows - 1);
    float o[NT][JT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][j][i] = 0.f;
    }

    const int end = (int)min((int64_t)lim_max, (int64_t)w.t1 * TILE);  // positions of this segment
    int pos = w.t0 * TILE + warp * STEP;
    const int32_t* table = p.b.table + it.seq * p.b.max_pages;
    // first row and scales of the warp's next 32 steps, one a lane (a step lies in one scale block, so in one page)
    const int steps = pos < end && ok ? (end - pos - 1) / (C::kWarps * STEP) + 1 : 0, pos_first = pos;
    int64_t held_row = 0;
    int held_scale = 0;
    auto get_rows = [&](int first) {
      const int at_pos = pos_first + (first + lane) * (C::kWarps * STEP);
      if (first + lane < steps) {
        const uint32_t blk = (uint32_t)at_pos / kScaleBlock, slot = kv_slot(p.pg, blk);
        int64_t page = table[slot];
        if (page < 0 || page >= p.pg.n_pages) {
          kv_report(p.pg.err, DMOE_KV_ERR_PAGE);
          page = 0;
        }
        held_row = kv_row(p.pg, page, head, (int)(blk - slot * p.pg.page_blocks) * kScaleBlock + at_pos % kScaleBlock);
        if (KV == KV_E4M3) held_scale = p.pg.k_scale[held_row / kScaleBlock] | p.pg.v_scale[held_row / kScaleBlock] << 8;
      }
    };
    uint8_t* const ring = reinterpret_cast<uint8_t*>(smem_f) + warp * (C::kStages * 2 * C::kHalf);
    constexpr int VN = VB == 8 ? 1 : VB / 16;  // 16-byte pieces of a value row a lane
    // Starts step n's copies; its scale bytes: key's, value's << 8.
    auto issue = [&](int n) {
      if (n >= steps) return 0;
      if (n % 32 == 0) get_rows(n);
      const int64_t row = __shfl_sync(0xffffffffu, held_row, n % 32);
      if (lane == 0) {
        const uint32_t s = (done + n) % C::kStages;
        uint8_t* const to = ring + s * 2 * C::kHalf;
        mbar_arrive_expect_tx(&bar[warp][s], 2 * C::kHalf);
        bulk_load(to, static_cast<const uint8_t*>(p.pg.k) + row * (HD * ES), C::kHalf, &bar[warp][s]);
        bulk_load(to + C::kHalf, static_cast<const uint8_t*>(p.pg.v) + row * (HD * ES), C::kHalf, &bar[warp][s]);
      }
      return KV == KV_E4M3 ? __shfl_sync(0xffffffffu, held_scale, n % 32) : 0;
    };
    fence_proxy_async_smem();  // the ring was last written by the warps' joining
    constexpr int kAhead = C::kStages - 1;
    int scales[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) scales[i + 1] = issue(i);
    int issued = min(steps, kAhead);
    // queries: lane (g, t) holds row g of each 8-row tile, at the elements its key chunks cover
    uint32_t qf[NT][HD / 16][2];
    float cq[NT][2];  // score factor and limit of the rows 2t, 2t + 1 of each tile
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = it.row_lo + n * 8 + g;
      const bool live = n * 8 + g < it.rows;
      float x[HD / 16][4];
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const int d = ES == 1 ? 16 * (t + 4 * (k / 4)) + 4 * (k % 4) : 8 * (t + 4 * (k / 2)) + 4 * (k % 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] = 0.f;
        if (live)
          load_q4(p, (int64_t)(it.q.row0 + row / p.group) * p.q_stride + (int64_t)(head * p.group + row % p.group) * HD + d, x[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[k][i]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // f16 products: rows scaled into [-1, 1] (past 2^126, where 2^e must stay a float, into [-4, 4])
      const int e = kBf ? 0 : min(max((int)(__float_as_uint(amax) >> 23) - 126, -100), 126);
      const float inv = pow2i(-e);
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qf[n][k][0] = pack2<kBf>(x[k][0] * inv, x[k][1] * inv);
        qf[n][k][1] = pack2<kBf>(x[k][2] * inv, x[k][3] * inv);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = n * 8 + 2 * t + i;
        cq[n][i] = p.scale_log2 * pow2i(__shfl_sync(0xffffffffu, e, (2 * t + i) * 4));
        lim[n][i] = r < it.rows ? row_limit(p, it.q, it.row_lo + r) : 0;
      }
    }
    for (int n = 0; n < steps; ++n, pos += C::kWarps * STEP) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) scales[i] = scales[i + 1];
      const int sc = scales[0];
      __syncwarp();  // no lane needs anything of the step before
      scales[kAhead] = issue(n + kAhead);
      issued = min(steps, n + C::kStages);
      const uint32_t stage = (done + n) % C::kStages;
      ok = warp_wait(&bar[warp][stage], (done + n) / C::kStages & 1, p.wait_err, DMOE_KV_ERR_TIMEOUT);
      if (!ok) break;
      const uint32_t kat = smem_u32(ring + stage * 2 * C::kHalf) + g * (HD * ES) + 16 * t;
      const uint32_t vat = smem_u32(ring + stage * 2 * C::kHalf + C::kHalf) + 2 * t * (HD * ES) + (VB == 8 ? 8 : 16) * g;
      uint32_t kr[MT][2][KCH][4];
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < KCH; ++c) {
            const uint4 v = lds128(kat + (16 * a + 8 * h) * (HD * ES) + 64 * c);
            kr[a][h][c][0] = v.x, kr[a][h][c][1] = v.y, kr[a][h][c][2] = v.z, kr[a][h][c][3] = v.w;
          }
      // s^T
      float s[NT][MT][4];
#pragma unroll
      for (int a = 0; a < MT; ++a) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][a][0] = s[n][a][1] = s[n][a][2] = s[n][a][3] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t af[4];
          if (KV == KV_E4M3) {
            const uint32_t x = kr[a][0][k / 4][k % 4], y = kr[a][1][k / 4][k % 4];
            af[0] = e4m3_pair<0>(x), af[1] = e4m3_pair<0>(y), af[2] = e4m3_pair<1>(x), af[3] = e4m3_pair<1>(y);
          } else {
            af[0] = kr[a][0][k / 2][2 * (k % 2)], af[1] = kr[a][1][k / 2][2 * (k % 2)];
            af[2] = kr[a][0][k / 2][2 * (k % 2) + 1], af[3] = kr[a][1][k / 2][2 * (k % 2) + 1];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<kBf>(s[n][a], af, qf[n][k][0], qf[n][k][1]);
        }
      }
      const int ev = KV == KV_E4M3 ? (sc >> 8) - 127 : 0;
      const float sk = KV == KV_E4M3 ? pow2i((sc & 255) - 127) : 1.f, evf = (float)ev;
      const float unv = KV == KV_E4M3 ? pow2i(-ev) : 1.f;
      const int here = pos;
      const bool edge = here + STEP > lim_min;

      // scores -> weights. Lane (g, t): positions 16a + g and 16a + 8 + g, rows 2t and 2t + 1
      uint32_t pf[NT][MT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][a][i] = fmaf(s[n][a][i], cq[n][i & 1] * sk, evf);
        if (edge) {
          asm volatile("" ::: "memory");  // stay a branch
#pragma unroll
          for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (here + 16 * a + 8 * (i >> 1) + g >= lim[n][i & 1]) s[n][a][i] = -INFINITY;
        }
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i & 1] = fmaxf(mx[i & 1], s[n][a][i]);
        float base[2], shrink[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], off));
          const float mn = fmaxf(m[n][i], __fsub_ru(mx[i], Lift<KV>::kRows));  // no weight is past 2^15, however large mx
          base[i] = mn == -INFINITY ? 0.f : mn;
          shrink[i] = ex2(m[n][i] - base[i]);
          m[n][i] = mn;
          l[n][i] *= shrink[i];
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int a = 0; a < MT; ++a) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][a][i] = ex2(s[n][a][i] - base[i & 1]);
            sum[i & 1] += s[n][a][i];
          }
          pf[n][a][0] = transpose8x8(pack2<kBf>(s[n][a][0], s[n][a][1]));
          pf[n][a][1] = transpose8x8(pack2<kBf>(s[n][a][2], s[n][a][3]));
        }
        l[n][0] = fmaf(sum[0], unv, l[n][0]);
        l[n][1] = fmaf(sum[1], unv, l[n][1]);
        if (__any_sync(0xffffffffu, shrink[0] != 1.f || shrink[1] != 1.f)) {
#pragma unroll
          for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][j][i] *= shrink[i & 1];
        }
      }
      uint32_t vr[MT][4][VW];
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t at = vat + (16 * a + (k & 1) + 8 * (k >> 1)) * (HD * ES);
          if (VB == 8) {
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(vr[a][k][0]), "=r"(vr[a][k][1]) : "r"(at));
          } else {
#pragma unroll
            for (int c = 0; c < VN; ++c) {
              const uint4 v = lds128(at + 128 * c);
              vr[a][k][4 * c] = v.x, vr[a][k][4 * c + 1] = v.y, vr[a][k][4 * c + 2] = v.z, vr[a][k][4 * c + 3] = v.w;
            }
          }
        }
      if (edge) {
        // positions past the sequence's end hold anything: their weights are zero, so must be the values
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool gone = here + 16 * a + 2 * t + (k & 1) + 8 * (k >> 1) >= lim_max;
#pragma unroll
            for (int c = 0; c < VW; ++c) vr[a][k][c] = gone ? 0u : vr[a][k][c];
          }
      }
      bool apart = false;  // a value that is not finite, at a position that only some rows see
      if (edge && lim_min < lim_max) {
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int c = 0; c < VW; ++c) apart |= not_finite<KV>(vr[a][k][c]);
        apart = __any_sync(0xffffffffu, apart);
      }
      if (apart) {
        // element by element, for the rows that see the position: zero times NaN must not reach the others
        constexpr int PER = 4 / ES;
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll 1
            for (int tt = 0; tt < 4; ++tt) {
              const int off = 2 * tt + (k & 1);  // position 16a + 8 (k >> 1) + off
#pragma unroll
              for (int c = 0; c < VW; ++c) {
                const uint32_t w = __shfl_sync(0xffffffffu, vr[a][k][c], g * 4 + tt);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const float pr = __shfl_sync(0xffffffffu, s[n][a][2 * (k >> 1) + i], off * 4 + t);
                    if (here + 16 * a + 8 * (k >> 1) + off < lim[n][i]) {
#pragma unroll
                      for (int e = 0; e < PER; ++e) {
                        float& acc = o[n][(PER * c + e) / 2][(e & 1) * 2 + i];
                        acc = fmaf(pr, element<KV>(w, e), acc);
                      }
                    }
                  }
              }
            }
        continue;
      }
      // o^T += V^T p^T
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          uint32_t af[4];
          if (KV == KV_E4M3) {
            const uint32_t sel = j & 1 ? 0x7362u : 0x5140u;
            const uint32_t x = __byte_perm(vr[a][0][j / 2], vr[a][1][j / 2], sel);
            const uint32_t y = __byte_perm(vr[a][2][j / 2], vr[a][3][j / 2], sel);
            af[0] = e4m3_pair<0>(x), af[1] = e4m3_pair<1>(x), af[2] = e4m3_pair<0>(y), af[3] = e4m3_pair<1>(y);
          } else {
            af[0] = __byte_perm(vr[a][0][j], vr[a][1][j], 0x5410u);
            af[1] = __byte_perm(vr[a][0][j], vr[a][1][j], 0x7632u);
            af[2] = __byte_perm(vr[a][2][j], vr[a][3][j], 0x5410u);
            af[3] = __byte_perm(vr[a][2][j], vr[a][3][j], 0x7632u);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<kBf>(o[n][j], af, pf[n][a][0], pf[n][a][1]);
        }
    }

    // after a timeout: what is still on its way (with the same limit), then on to the end
    if (!ok)
      for (int n = 0; n < issued; ++n) warp_wait(&bar[warp][(done + n) % C::kStages], (done + n) / C::kStages & 1, p.wait_err, DMOE_KV_ERR_TIMEOUT);
    done += steps;

    // join the warps: o, M and the sum of each row
    __syncthreads();  // every warp has left the ring
    float* os = smem_f;                           // [warp][row][d]
    float* ml = smem_f + C::kWarps * R * HD;      // [warp][row][2]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], off);
        if (g == 0) {
          ml[(warp * R + n * 8 + 2 * t + i) * 2] = m[n][i];
          ml[(warp * R + n * 8 + 2 * t + i) * 2 + 1] = l[n][i];
        }
      }
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = (ES == 1 || HD == 64 ? HD / 8 * g + 2 * j : 8 * (g + 8 * (j / 4)) + 2 * (j % 4)) + (i >> 1);
          os[(warp * R + n * 8 + 2 * t + (i & 1)) * HD + d] = o[n][j][i];
        }
    }
    __syncthreads();
    const bool whole = w.whole();
    float* part = p.part + (int64_t)(2 * blockIdx.x + (w.t0 == 0 ? 1 : 0)) * C::kPart;
    for (int i = tid; i < it.rows * HD; i += 32 * C::kWarps) {
      const int r = i / HD, d = i % HD;
      float mm = -INFINITY;
#pragma unroll
      for (int k = 0; k < C::kWarps; ++k) mm = fmaxf(mm, ml[(k * R + r) * 2]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float acc = 0.f, ll = 0.f;
#pragma unroll
      for (int k = 0; k < C::kWarps; ++k) {
        const float f = ex2(ml[(k * R + r) * 2] - base);
        acc = fmaf(os[(k * R + r) * HD + d], f, acc);
        ll = fmaf(ml[(k * R + r) * 2 + 1], f, ll);
      }
      if (whole) {
        store_out(p, it.q.row0, it.row_lo + r, head, d, HD, ll == 0.f ? 0.f : acc / ll);
        if (d == 0) store_lse(p, it.q.row0, it.row_lo + r, head, mm, ll);
      } else {
        part[r * HD + d] = acc;
        if (d == 0) part[R * HD + 2 * r] = mm, part[R * HD + 2 * r + 1] = ll;
      }
    }
    if (!whole && w.t0 == 0) begun = w.begun();
    __syncthreads();  // os and ml are free again
  }
  if (tid == 0) p.desc[blockIdx.x] = begun;
  pdl_trigger();
}

// ---------------------------------------------------------------------------------------------
// Many rows (denoising blocks, prompts): tensor-core tiles of 2 x 128 rows by 128 positions.
//
// One persistent CTA per SM. Warps 0-3 and 4-7: softmax of the two 128-row halves, a thread a row; warps
// 8-11: keys, 12-15: values, from the pages into shared memory as 16-bit operands in the 128-byte swizzle; a
// thread of warp 16 issues the products. TMEM: two score tiles (f32, 128 columns each; a half's weights
// overwrite its scores as the 16-bit A operand of the second product) and two outputs. The products of one
// half run while the other half's softmax does. The reference of a row's weights (Lift) follows
// the running maximum only when that is 2^8 ahead of where it was set, so an output is rescaled in TMEM only
// then.
// Bound by a half's chain of scores (512 cycles of the tensor pipe), exponentials (128 a thread, 8 cycles a warp:
// 1024 at least) and products (512), of which two are in flight: about 3800 cycles for two tiles. Measured: 2048 rows
// over 16384 positions of bf16 pages 535 us = 0.97 PFLOP/s (tensor pipe 54 % active, exponential unit 54 %); 16
// blocks of 32 rows over 0.5-16 K positions of e4m3 pages 117 us; a prompt of 4096 230 us. The registers of every
// role spill (1.4 KB of stores a thread): run, walk and item are carried by all of them.
// ---------------------------------------------------------------------------------------------
template <int HD, int KV>
struct TileCfg {
  static constexpr int R = 256, TILE = 128;
  static constexpr int ES = KV == KV_E4M3 ? 1 : 2;
  static constexpr int OV = 4;
  static constexpr int kThreads = 640, kLoaders = 128;
  // registers a thread: 256 * 160 + 256 * 64 + 128 * 32 = the 640 * 96 of the launch
  static constexpr int kSoftmaxRegs = 160, kLoadRegs = 64, kIssueRegs = 32;
  static constexpr int kPlane = 128 * 128;             // 64 elements of 128 rows
  static constexpr int kOperand = HD / 64 * kPlane;    // bytes of a 128-row operand
  static constexpr int kStages = 2;
  static constexpr int kOutWarp = 32 * 64;             // staging of 32 columns of a warp's 32 output rows
  static constexpr size_t kSmem = 1024 + (2 + 2 * kStages) * (size_t)kOperand + 8 * kOutWarp;
  static constexpr int kPart = R * (HD + 2);
};

struct TileBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_part[2], p_full[2], o_full[2], read[4], reset, done;
};


template <int HD, int KV>
__global__ void __launch_bounds__(640, 1) kv_tile_kernel(const __grid_constant__ AttnParams p) {
  using C = TileCfg<HD, KV>;
  constexpr bool kBf = KV == KV_BF16;
  constexpr int R = C::R, TILE = C::TILE, ES = C::ES;
  constexpr uint32_t kIdescS = idesc_16b_f32(128, 128, kBf, false), kIdescO = idesc_16b_f32(128, HD, kBf, true);
  extern __shared__ uint8_t smem_raw[];
  __shared__ TileBars bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ uint2 sums[C::kThreads / 32];
  __shared__ Run found;
  // [item of the run & 3][sign][d]: first position whose value is +inf, or -inf; both for NaN
  __shared__ int not_finite_from[4][2][HD];
  __shared__ int any_not_finite[4];
  // scales of keys, exponents of values and their reciprocal scales [..][tile of the run & 3][32-position block].
  // Written with the keys, before their arrival; the slot is free again when the tile two on has been multiplied by
  // the queries of both halves
  __shared__ __align__(16) float scale_s[3][4][4];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                                 // [half] operands
  uint8_t* k_s = q_s + 2 * C::kOperand;                // [stage]
  uint8_t* v_s = k_s + C::kStages * C::kOperand;       // [stage]
  uint8_t* out_s = v_s + C::kStages * C::kOperand;     // [softmax warp]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // tensor memory only after the kernel before has ended: one that still had to allocate its own would wait for
  // this one, which waits for it
  pdl_wait();
  if (warp == 16) {
    tmem_alloc(&tmem_base_s, 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], C::kLoaders);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], C::kLoaders);
      mbar_init(&bar.v_empty[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_part[i], 128);
      mbar_init(&bar.p_full[i], 128);
      mbar_init(&bar.o_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar.read[i], 256);
    mbar_init(&bar.reset, C::kLoaders);
    mbar_init(&bar.q_full, 256);
    mbar_init(&bar.done, 1);
    fence_mbar_init();
  }
  if (tid < 4) any_not_finite[tid] = 0;
  tc_fence_before();
  const Run run = find_run<R, TILE, C::OV, C::kThreads>(p, sums, &found);  // ends with a barrier of the CTA
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  uint32_t* err = p.wait_err;
  constexpr uint32_t kTimeout = DMOE_KV_ERR_TIMEOUT;

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kIssueRegs));
    Walk<R, TILE, C::OV> w(p, run);
    if (warp == 16) {
      // ---- products: one thread waits and issues, so that nothing but the waits lies between them
      if (elect_one()) {
        uint32_t n = 0;  // tiles whose keys were used
        uint32_t ph_p[2] = {0, 0};
        bool ok = true;
        auto wait = [&](uint64_t* b, uint32_t parity) { return mbar_wait(b, parity, err, kTimeout); };
        const uint64_t q_desc = sdesc_sw128(smem_u32(q_s), 1024), k_desc = sdesc_sw128(smem_u32(k_s), 1024),
                       v_desc = sdesc_sw128_mn(smem_u32(v_s), C::kPlane);
        auto scores = [&](int half, int stage) {
          const uint64_t qd = q_desc + half * (C::kOperand / 16), kd = k_desc + stage * (C::kOperand / 16);
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const int off = ((k / 4) * C::kPlane + (k % 4) * 32) / 16;
            mma_f16_ss(tmem + half * 128, qd + off, kd + off, kIdescS, k > 0);
          }
          mma_commit(&bar.s_full[half]);
        };
        auto outputs = [&](int half, int stage, int part, bool first) {
          const uint64_t vd = v_desc + stage * (C::kOperand / 16) + part * 4 * (2048 / 16);
          const uint32_t pa = tmem + half * 128 + part * 32;
          mma_f16_ts(tmem + 256 + half * 128, pa, vd, kIdescO, !first);
#pragma unroll
          for (int k = 1; k < TILE / 32; ++k) mma_f16_ts(tmem + 256 + half * 128, pa + 8 * k, vd + k * (2048 / 16), kIdescO, 1);
        };
        for (; ok && w.more(); w.next()) {
          const int halves = w.it.rows > 128 ? 2 : 1, tiles = w.t1 - w.t0;
          ok = wait(&bar.q_full, w.seg & 1) && wait(&bar.k_full[n & 1], (n >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          for (int h = 0; h < halves; ++h) scores(h, n & 1);
          mma_commit(&bar.k_empty[n & 1]);
          for (int j = 0; ok && j < tiles; ++j, ++n) {
            const int stage = n & 1, next = (n + 1) & 1;
            ok = wait(&bar.v_full[stage], (n >> 1) & 1);
            for (int h = 0; ok && h < halves; ++h) {
              ok = wait(&bar.p_part[h], ph_p[h]);
              if (!ok) break;
              tc_fence_after();
              outputs(h, stage, 0, j == 0);
              ok = wait(&bar.p_full[h], ph_p[h]);
              if (!ok) break;
              ph_p[h] ^= 1;
              tc_fence_after();
              outputs(h, stage, 1, false);
              if (h == halves - 1) mma_commit(&bar.v_empty[stage]);
              if (j + 1 < tiles) {
                if (h == 0) {
                  ok = wait(&bar.k_full[next], ((n + 1) >> 1) & 1);
                  if (!ok) break;
                  tc_fence_after();
                }
                scores(h, next);
                if (h == halves - 1) mma_commit(&bar.k_empty[next]);
              } else {
                mma_commit(&bar.o_full[h]);
              }
            }
          }
        }
        mma_commit(&bar.done);  // every product that was issued has ended before TMEM is freed
        wait(&bar.done, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ---- keys (warps 8-11) and values (12-15)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kLoadRegs));
    Walk<R, TILE, C::OV> w(p, run);
    const bool is_v = warp >= 12;
    const int lt = tid & 127;
    uint64_t* const full = is_v ? bar.v_full : bar.k_full;
    uint64_t* const empty = is_v ? bar.v_empty : bar.k_empty;
    uint8_t* const ring = is_v ? v_s : k_s;
    const uint8_t* const base = static_cast<const uint8_t*>(is_v ? p.pg.v : p.pg.k);
    constexpr int LPR = HD * ES / 16;             // lanes a row, 16 bytes each
    constexpr int RPI = C::kLoaders / LPR;        // rows an instruction of all loaders covers
    constexpr int N = TILE / RPI;                 // 16-byte pieces a thread loads of a tile
    const int c = lt % LPR, r0 = lt / LPR;
    bool ok = true;
    // first row of each of the tile's 32-position blocks in the pages. The page numbers of eight tiles
    // are read at once, one a lane
    const uint8_t* block_at[4];  // this thread's piece of its first row in each block
    int64_t scale_at = 0;         // scale of block `lane` of the tile (lanes 0-3)
    int held = 0, held_from = 0;  // blocks [held_from, held_from + 32) of the item
    auto get_pages = [&](int tile, int lim, bool new_item) {
      const int b0 = tile * (TILE / 32);
      if (new_item || b0 >= held_from + 32) {
        held_from = b0;
        held = 0;
        if ((b0 + lane) * 32 < lim) {
          held = p.b.table[w.it.seq * p.b.max_pages + kv_slot(p.pg, b0 + lane)];
          if (held < 0 || held >= p.pg.n_pages) {
            kv_report(p.pg.err, DMOE_KV_ERR_PAGE);
            held = 0;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int page = __shfl_sync(0xffffffffu, held, b0 + i - held_from);
        const uint32_t b = b0 + i;
        const int64_t blk = ((int64_t)page * p.pg.n_head_kv + w.head) * p.pg.page_blocks + (b - kv_slot(p.pg, b) * p.pg.page_blocks);
        block_at[i] = base + blk * (32 * HD * ES) + r0 * (HD * ES) + 16 * c;
        if (KV == KV_E4M3 && lane == i) scale_at = blk;
      }
    };
    // this thread's i-th piece of the tile; its row is r0 + i * RPI
    auto source = [&](int i) { return block_at[i * RPI / 32] + (i * RPI % 32) * (HD * ES); };
    // Values at positions that only some rows see, where they are not finite: their products with a zero
    // weight would reach the other rows. They are set to zero, and their element marked for the rows that see them
    auto mark = [&](int seg, int pos, int d, bool plus, bool minus) {
      if (plus) atomicMin(&not_finite_from[seg & 3][0][d], pos);
      if (minus) atomicMin(&not_finite_from[seg & 3][1][d], pos);
      any_not_finite[seg & 3] = 1;
    };
    auto reset_marks = [&](int seg) {
      // once both halves have read the buffer's last use, four items back
      if (!warp_wait(&bar.read[seg & 3], ((seg >> 2) & 1) ^ 1, err, kTimeout)) return false;
      if (lt < HD) not_finite_from[seg & 3][0][lt] = not_finite_from[seg & 3][1][lt] = INT32_MAX;
      if (lt == 0) any_not_finite[seg & 3] = 0;
      mbar_arrive(&bar.reset);
      return warp_wait(&bar.reset, seg & 1, err, kTimeout);
    };
    auto limit = [&]() { return row_limit(p, w.it.q, w.it.row_lo + w.it.rows - 1); };
    uint4 x[KV == KV_E4M3 ? N : 1];  // 8-bit pages: the next tile, on its way
    int scale = 0;                   // and the scale bytes of its block `lane`: key's, value's << 8 (key loaders 0-3)
    auto fetch = [&](int tile, int lim) {
      if constexpr (KV == KV_E4M3) {
        scale = 127 | 127 << 8;
        if (!is_v && lt < 4 && tile * TILE + 32 * lt < lim) scale = p.pg.k_scale[scale_at] | p.pg.v_scale[scale_at] << 8;
        if ((tile + 1) * TILE <= lim) {
#pragma unroll
          for (int i = 0; i < N; ++i) x[i] = load_past_l1(source(i));
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            x[i] = make_uint4(0, 0, 0, 0);
            if (tile * TILE + r0 + i * RPI < lim) x[i] = load_past_l1(source(i));
          }
        }
      }
    };
    uint32_t n = 0;
    if (w.more()) {
      const int lim = limit();
      get_pages(w.t0, lim, true);
      fetch(w.t0, lim);
    }
    while (ok && w.more()) {
      const int lim_min = row_limit(p, w.it.q, w.it.row_lo), lim_max = limit();
      const int seg = w.seg, t0 = w.t0, t1 = w.t1;
      for (int t = t0; t < t1; ++t, ++n) {
        const int stage = n & 1;
        uint8_t* const dst = ring + stage * C::kOperand;
        ok = warp_wait(&empty[stage], ((n >> 1) & 1) ^ 1, err, kTimeout);
        if (ok && is_v && t == t0) ok = reset_marks(seg);
        if (!ok) break;
        const bool edge = is_v && lim_min < lim_max && (t + 1) * TILE > lim_min;
        if constexpr (KV == KV_E4M3) {
          // the values' scales too: the softmax needs them with the scores, before the values need be here
          if (!is_v && lt < 4) {
            const int ev = (scale >> 8) - 127;
            scale_s[0][n & 3][lt] = pow2i((scale & 255) - 127), scale_s[1][n & 3][lt] = (float)ev, scale_s[2][n & 3][lt] = pow2i(-ev);
          }
          if (edge) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const int pos = t * TILE + r0 + i * RPI;
              uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t bad = __vcmpeq4(v[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                if (bad && pos >= lim_min) {
                  for (int b = 0; b < 4; ++b)
                    if ((bad >> (8 * b)) & 1u) mark(seg, pos, 16 * c + 4 * e + b, true, true);
                  v[e] &= ~bad;
                }
              }
              x[i] = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
          const int first = (c / 4) & 1;  // lanes of the two planes take turns: no bank twice
          uint8_t* const row0 = dst + (c / 4) * C::kPlane + r0 * 128;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[2 * e] = e4m3_pair<0>(v[e]), h[2 * e + 1] = e4m3_pair<1>(v[e]);
            const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
            uint8_t* const row = row0 + i * RPI * 128;
            static_assert(RPI % 8 == 0, "the swizzle of a thread's rows is one");
            const int ca = (2 * (c % 4)) ^ (r0 & 7), cb = (2 * (c % 4) + 1) ^ (r0 & 7);
            *reinterpret_cast<uint4*>(row + 16 * (first ? cb : ca)) = first ? b : a;
            *reinterpret_cast<uint4*>(row + 16 * (first ? ca : cb)) = first ? a : b;
          }
        } else {
          // 16-bit pages need no conversion
          uint8_t* const mine = dst + (c / 8) * C::kPlane + r0 * 128 + 16 * ((c % 8) ^ (r0 & 7));
          static_assert(RPI % 8 == 0, "the swizzle of a thread's rows is one");
          const uint32_t to = smem_u32(mine);
          if ((t + 1) * TILE <= lim_max) {
#pragma unroll
            for (int i = 0; i < N; ++i)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * RPI * 128), "l"(source(i)) : "memory");
          } else {
#pragma unroll 4
            for (int i = 0; i < N; ++i) {
              const bool in = t * TILE + r0 + i * RPI < lim_max;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * RPI * 128), "l"(in ? source(i) : base),
                           "r"(in ? 16 : 0)
                           : "memory");
            }
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          if (edge) {
#pragma unroll 1
            for (int i = 0; i < N; ++i) {
              const int pos = t * TILE + r0 + i * RPI;
              uint4* const at = reinterpret_cast<uint4*>(mine + i * RPI * 128);  // this thread's own copy
              uint32_t v[4] = {at->x, at->y, at->z, at->w};
              bool any = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                constexpr uint32_t kExp = kBf ? 0x7f807f80u : 0x7c007c00u;
                const uint32_t bad = __vcmpeq2(v[e] & kExp, kExp);
                if (bad && pos >= lim_min) {
                  for (int b = 0; b < 2; ++b) {
                    if (!((bad >> (16 * b)) & 1u)) continue;
                    const uint32_t h = v[e] >> (16 * b) & 0xffffu;
                    const bool nan = (h & ~kExp & 0x7fffu) != 0;
                    mark(seg, pos, 8 * c + 2 * e + b, nan || !(h & 0x8000u), nan || (h & 0x8000u));
                  }
                  v[e] &= ~bad;
                  any = true;
                }
              }
              if (any) *at = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(&full[stage]);
        // the next tile of this item, or the next item's first
        const bool same = t + 1 < t1;
        if (!same) w.next();
        if (same || w.more()) {
          const int next = same ? t + 1 : w.t0, lim = same ? lim_max : limit();
          get_pages(next, lim, !same);
          fetch(next, lim);
        }
      }
    }
  } else {
    // ---- softmax of one half
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    Walk<R, TILE, C::OV> w(p, run);
    const int half = warp >> 2, quarter = warp & 3;
    const int my = half * 128 + quarter * 32 + lane;  // row of the item
    const uint32_t s_addr = tmem_addr(tmem, quarter * 32, half * 128), o_addr = tmem_addr(tmem, quarter * 32, 256 + half * 128);
    uint32_t ph_s = 0, ph_o = 0;
    bool ok = true;
    Spanning begun = {-1, 0, 0, 0, 0, {0, 0, 0}};
    // the warp's 32 rows of queries, HD / 8 lanes a row, copied into the operand as they are
    constexpr int LPQ = HD / 8, RPL = 32 / LPQ;
    uint8_t* const q_warp = q_s + half * C::kOperand + quarter * 32 * 128;
    auto fetch_queries = [&]() {
      if (!w.more() || half * 128 >= w.it.rows) return;
      const int tok0 = w.it.row_lo / p.group, g0 = w.it.row_lo - tok0 * p.group, sub = lane % LPQ;
      const uint16_t* const q0 = p.q + (int64_t)(w.it.q.row0 + tok0) * p.q_stride + (int64_t)w.head * p.group * HD + 8 * sub;
#pragma unroll 2
      for (int r = lane / LPQ; r < 32; r += RPL) {
        const int row = g0 + half * 128 + quarter * 32 + r;
        const int tok = (int)((row * (uint64_t)p.group_magic) >> 28);  // row / group
        const bool in = half * 128 + quarter * 32 + r < w.it.rows;
        const uint16_t* const src = in ? q0 + tok * p.q_stride + (row - tok * p.group) * HD : p.q;
        uint8_t* const dst = q_warp + (sub / 8) * C::kPlane + r * 128 + 16 * ((sub % 8) ^ (r & 7));
        if (p.vec_q16) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
        } else {
          uint16_t h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = in ? src[e] : (uint16_t)0;
          *reinterpret_cast<uint4*>(dst) = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16,
                                                      h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
        }
      }
    };
    // a thread turns its row into the products' type; f16 products: scaled into [-1, 1] by a power of two. The factor
    // that turns the row's products into scores
    auto ready_queries = [&]() {
      float factor = p.scale_log2;
      if (!w.more()) return factor;
      if (half * 128 < w.it.rows) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        if (!(kBf && p.is_bf16)) {
          uint8_t* const mine = q_warp + lane * 128;
          auto piece = [&](int i) { return reinterpret_cast<uint4*>(mine + (i / 8) * C::kPlane + 16 * ((i % 8) ^ (lane & 7))); };
          float inv = 1.f;
          if (!kBf) {
            uint32_t a = 0;  // magnitudes compare as integers
#pragma unroll 4
            for (int i = 0; i < HD / 8; ++i) {
              const uint4 v = *piece(i);
              a = __vmaxu2(a, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
            }
            a = max(a & 0xffffu, a >> 16);
            const float amax = p.is_bf16 ? __uint_as_float(a << 16) : __half2float(__ushort_as_half((uint16_t)a));
            const int e = min(max((int)(__float_as_uint(amax) >> 23) - 126, -100), 126);
            inv = pow2i(-e);
            factor *= pow2i(e);
            if (KV != KV_E4M3) factor = fmaxf(factor, kTinyFactor);  // 8-bit pages: when the keys' scale is in it
          }
#pragma unroll 2
          for (int i = 0; i < HD / 8; ++i) {
            const uint4 x = *piece(i);
            uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = p.is_bf16 ? make_float2(__uint_as_float(v[k] << 16), __uint_as_float(v[k] & 0xffff0000u))
                                         : __half22float2(*reinterpret_cast<const __half2*>(&v[k]));
              v[k] = pack2<kBf>(f.x * inv, f.y * inv);
            }
            *piece(i) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        fence_proxy_async_smem();
      }
      mbar_arrive(&bar.q_full);
      return factor;
    };
    fetch_queries();
    float next_factor = ready_queries();
    uint32_t n = 0;  // tiles
    while (ok && w.more()) {
      const int seg = w.seg, rows = w.it.rows;
      const bool active = half * 128 < rows, live = my < rows, whole = w.whole();
      const float factor = next_factor;
      if (!whole && w.t0 == 0) begun = w.begun();
      if (!active) {
        // not ahead of the other half: an arrival for the next item would count for this one's queries
        ok = warp_wait(&bar.q_full, seg & 1, err, kTimeout);
        if (!ok) break;
        mbar_arrive(&bar.read[seg & 3]);
        n += w.t1 - w.t0;
        w.next();
        fetch_queries();
        next_factor = ready_queries();
        continue;
      }
      const int row = w.it.row_lo + my;
      const int lim_all = row_limit(p, w.it.q, w.it.row_lo + rows - 1);
      const int lim = live ? row_limit(p, w.it.q, row) : lim_all;
      const int lim_warp = row_limit(p, w.it.q, w.it.row_lo + min(rows - 1, half * 128 + quarter * 32));
      float m = -INFINITY, l = 0.f;  // reference of the weights, sum
      const int t0 = w.t0, t1 = w.t1;
      for (int t = t0; t < t1; ++t, ++n) {
        ok = warp_wait(&bar.s_full[half], ph_s, err, kTimeout);
        if (!ok) break;
        ph_s ^= 1;
        tc_fence_after();
        // 32 scores at a time, the next ones on their way; they are read twice, since a row of 128 in registers
        // leaves none to overlap the exponentials with
        uint32_t x[2][32];
        tmem_ld32(s_addr, x[0]);
        float c[4], ev[4], un[4];  // score factors, exponents of the values' scales, their reciprocals
        if (KV == KV_E4M3) {
          const float4 k = *reinterpret_cast<const float4*>(scale_s[0][n & 3]), v = *reinterpret_cast<const float4*>(scale_s[1][n & 3]),
                       u = *reinterpret_cast<const float4*>(scale_s[2][n & 3]);
          // not down to zero (tiny queries over zero keys): masked scores are -inf when they are multiplied
          c[0] = fmaxf(factor * k.x, kTinyFactor), c[1] = fmaxf(factor * k.y, kTinyFactor);
          c[2] = fmaxf(factor * k.z, kTinyFactor), c[3] = fmaxf(factor * k.w, kTinyFactor);
          ev[0] = v.x, ev[1] = v.y, ev[2] = v.z, ev[3] = v.w;
          un[0] = u.x, un[1] = u.y, un[2] = u.z, un[3] = u.w;
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b) c[b] = factor, ev[b] = 0.f, un[b] = 1.f;
        }
        const bool edge = (t + 1) * TILE > lim_warp;
        const int valid = lim - t * TILE;  // columns this row sees
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t(&y)[32] = x[b & 1];
          tmem_wait_ld();
          if (b < 3) tmem_ld32(s_addr + 32 * (b + 1), x[(b + 1) & 1]);
          if (edge) {  // scores that the row does not see, here and (a store keeps this a branch) in TMEM
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = 32 * b + i < valid ? y[i] : 0xff800000u;
            tmem_st16(s_addr + 32 * b, reinterpret_cast<uint32_t(&)[16]>(y[0]));
            tmem_st16(s_addr + 32 * b + 16, reinterpret_cast<uint32_t(&)[16]>(y[16]));
          }
          float top[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3(__uint_as_float(y[8 * i]), __uint_as_float(y[8 * i + 1]), __uint_as_float(y[8 * i + 2]));
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3(top[i], __uint_as_float(y[8 * i + 3]), __uint_as_float(y[8 * i + 4]));
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3(top[i], __uint_as_float(y[8 * i + 5]), __uint_as_float(y[8 * i + 6]));
          top[0] = max3(top[0], __uint_as_float(y[7]), top[1]);
          top[2] = max3(top[2], __uint_as_float(y[15]), top[3]);
          top[0] = max3(top[0], __uint_as_float(y[23]), top[2]);
          top[0] = max3(top[0], __uint_as_float(y[31]), top[0]);
          mx = max3(mx, fmaf(top[0], c[b], ev[b]), mx);
        }
        if (edge) tmem_wait_st();
        tmem_ld32(s_addr, x[0]);
        if (!(mx < INFINITY)) {  // a score that is NaN or infinite: so is the row, whatever the weights become
          l = __int_as_float(0x7fc00000);
          mx = m;
        }
        float shrink = 1.f;
        // at least the largest score as the weights' fma has it, exact: mx was rounded, by far more than 1 where it is huge
        const float most = fmaf(fabsf(mx), 0x1p-23f, mx);
        if (most - m > Lift<KV>::kGrown || m == -INFINITY) {
          const float to = fmaxf(m, __fsub_ru(most, Lift<KV>::kTiles));
          shrink = to == -INFINITY ? 1.f : ex2(m - to);
          m = to;
          l *= shrink;
        }
        if (t > t0 && __any_sync(0xffffffffu, shrink != 1.f)) {
          // the products of the tile before have ended: the scores' arrival counts them
#pragma unroll 1
          for (int d = 0; d < HD; d += 16) {
            uint32_t y[16];
            tmem_ld16(o_addr + d, y);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * shrink);
            tmem_st16(o_addr + d, y);
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t(&y)[32] = x[b & 1];
          tmem_wait_ld();
          if (b < 3) tmem_ld32(s_addr + 32 * (b + 1), x[(b + 1) & 1]);
          const uint64_t c2 = pair(c[b], c[b]), off2 = pair(ev[b] - base, ev[b] - base);
          uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float a, d;
            const uint64_t e = fma2(pair(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), c2, off2);
            unpair(e, a, d);
            a = ex2(a), d = ex2(d);
            sum[i / 2 & 1] = add2(sum[i / 2 & 1], pair(a, d));
            pk[i / 2] = pack2<kBf>(a, d);
          }
          tmem_st16(s_addr + 16 * b, pk);
          float a, d;
          unpair(add2(sum[0], sum[1]), a, d);
          l = fmaf(a + d, un[b], l);
          if (b == 1) {  // the products of the first half of the columns need not wait
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bar.p_part[half]);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bar.p_full[half]);
      }
      if (!ok) break;
      const Item it = w.it;
      const int head = w.head;
      w.next();
      // the scores' last arrival: the operand is free. The next item's scores are computed while this one's
      // output is written
      fetch_queries();
      next_factor = ready_queries();
      ok = warp_wait(&bar.o_full[half], ph_o, err, kTimeout);
      if (!ok) break;
      ph_o ^= 1;
      tc_fence_after();
      const bool marked = *const_cast<volatile int*>(&any_not_finite[seg & 3]) != 0;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // a warp's rows lie side by side in a partial, [d][row]; rows of the output go through shared memory, 32
      // columns at a time, so that either is written in whole sectors
      float* const part = p.part + (int64_t)(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * C::kPart + my;
      uint8_t* const stage = out_s + warp * C::kOutWarp;
      uint16_t* out_row[4];  // lane's rows 8 i + lane / 4, at its eight columns
      {
        const int tok0 = it.row_lo / p.group, g0 = it.row_lo - tok0 * p.group;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = g0 + half * 128 + quarter * 32 + 8 * i + lane / 4, tok = (int)((r * (uint64_t)p.group_magic) >> 28);
          out_row[i] = p.out + (int64_t)(it.q.row0 + tok0 + tok) * p.out_stride + (int64_t)(head * p.group + r - tok * p.group) * HD + 8 * (lane % 4);
        }
      }
#pragma unroll 1
      for (int d0 = 0; d0 < HD; d0 += 32) {
        uint32_t x[32];
        tmem_ld32(o_addr + d0, x);
        tmem_wait_ld();
        if (marked) {
#pragma unroll 1
          for (int i = 0; i < 32; ++i) {
            const float plus = *const_cast<volatile int*>(&not_finite_from[seg & 3][0][d0 + i]) < lim ? INFINITY : 0.f;
            const float minus = *const_cast<volatile int*>(&not_finite_from[seg & 3][1][d0 + i]) < lim ? INFINITY : 0.f;
            if (plus + minus != 0.f) {
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = e == i ? __float_as_uint(__uint_as_float(x[e]) + (plus - minus)) : x[e];
            }
          }
        }
        if (!whole) {
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; ++i) part[(d0 + i) * R] = __uint_as_float(x[i]);
          }
          continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = l == 0.f ? 0.f : __uint_as_float(x[8 * i + 2 * e]) * inv, b = l == 0.f ? 0.f : __uint_as_float(x[8 * i + 2 * e + 1]) * inv;
            h[e] = p.is_bf16 ? pack2<true>(a, b) : pack2<false>(a, b);
          }
          *reinterpret_cast<uint4*>(stage + lane * 64 + 16 * (i ^ ((lane >> 1) & 3))) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + lane / 4, of = half * 128 + quarter * 32 + r;
          const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + 16 * ((lane % 4) ^ ((r >> 1) & 3)));
          if (of < rows) {
            uint16_t* const o = out_row[i] + d0;
            if (p.vec_out16) {
              *reinterpret_cast<uint4*>(o) = v;
            } else {
              const uint32_t h[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = (uint16_t)(h[e / 2] >> (16 * (e & 1)));
            }
          }
        }
        __syncwarp();
      }
      if (live) {
        if (!whole)
          part[HD * R] = m, part[(HD + 1) * R] = l;
        else
          store_lse(p, it.q.row0, row, head, m, l);
      }
      tc_fence_before();
      mbar_arrive(&bar.read[seg & 3]);
    }
    if (tid == 0) p.desc[blockIdx.x] = begun;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tmem, 512);
  pdl_trigger();
}

// Adds the partial triples of the items that the CTAs of the first kernel began and did not end: for CTA c's,
// those of slots 2c + 1, 2(c + 1), .. 2 last. The pieces of all such items (PIECES each) are shared out over the
// grid: every CTA reads all descriptors and takes every gridDim.x-th piece. Eight teams of threads take every
// eighth triple with a running maximum each, and are joined in order.
template <int PIECES, typename F>
__device__ __forceinline__ void for_pieces(const AttnParams& p, int n_cta, F&& f) {
  __shared__ Spanning begun_s[kMaxGrid];
  __shared__ int from_s[kMaxGrid];
  __shared__ int count_s[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Spanning d{};
  d.last = -1;
  if (tid < n_cta) d = p.desc[tid];
  const bool has = d.last >= 0;
  const uint32_t mask = __ballot_sync(0xffffffffu, has);
  if (lane == 0) count_s[warp] = __popc(mask);
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < 8; ++w) {
    if (w < warp) before += count_s[w];
    total += count_s[w];
  }
  if (has) {
    const int i = before + __popc(mask & ((1u << lane) - 1));
    begun_s[i] = d;
    from_s[i] = tid;
  }
  __syncthreads();
  for (int i = blockIdx.x; i < total * PIECES; i += gridDim.x) {
    const int piece = i / total, at = i - piece * total;  // first pieces first: an item may have fewer
    f(begun_s[at], from_s[at], piece);
  }
}

// Adds triple (mk, lk, x) to (m, l, acc).
template <int D>
__device__ __forceinline__ void join(float& m, float& l, float (&acc)[D], float mk, float lk, const float (&x)[D]) {
  const float to = fmaxf(m, mk), base = to == -INFINITY ? 0.f : to, f0 = ex2(m - base), f1 = ex2(mk - base);
  m = to;
  l = l * f0 + lk * f1;
#pragma unroll
  for (int i = 0; i < D; ++i) acc[i] = acc[i] * f0 + x[i] * f1;
}

// Few rows, triples [row][d]: a piece is a row.
template <int HD, int R>
__global__ void __launch_bounds__(256) kv_combine_kernel(const __grid_constant__ AttnParams p, int n_cta) {
  constexpr int D = HD / 32;  // columns a lane
  __shared__ float acc_s[8][HD];
  __shared__ float m_s[8], l_s[8];
  pdl_wait();
  const int lane = threadIdx.x & 31, team = threadIdx.x >> 5;
  for_pieces<R>(p, n_cta, [&](const Spanning& b, int c, int r) {
    if (r >= b.rows) return;
    const int n = b.last - c + 1;
    auto slot = [&](int k) { return p.part + (int64_t)(2 * (c + k) + (k == 0 ? 1 : 0)) * (R * (HD + 2)); };
    float acc[D] = {}, l = 0.f, m = -INFINITY;
#pragma unroll 4
    for (int k = team; k < n; k += 8) {
      const float* s = slot(k);
      float x[D];
#pragma unroll
      for (int i = 0; i < D; ++i) x[i] = s[r * HD + 32 * i + lane];
      join(m, l, acc, s[R * HD + 2 * r], s[R * HD + 2 * r + 1], x);
    }
#pragma unroll
    for (int i = 0; i < D; ++i) acc_s[team][32 * i + lane] = acc[i];
    if (lane == 0) m_s[team] = m, l_s[team] = l;
    __syncthreads();
    if (threadIdx.x < HD) {
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, m_s[k]);
      const float base = top == -INFINITY ? 0.f : top;
      float a = 0.f, sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = ex2(m_s[k] - base);
        a = fmaf(acc_s[k][threadIdx.x], f, a);
        sum = fmaf(l_s[k], f, sum);
      }
      store_out(p, b.row0, b.row_lo + r, b.head, threadIdx.x, HD, sum == 0.f ? 0.f : a / sum);
      if (threadIdx.x == 0) store_lse(p, b.row0, b.row_lo + r, b.head, top, sum);
    }
    __syncthreads();
  });
}

// Row tiles, triples [d][row]. Up to 8 triples: a piece is 32 rows, a lane a row and a warp an eighth of the
// columns, all triples' loads on their way at once. More (a few items over the whole GPU): a piece is 32 rows by 16
// columns and the warps share the triples.
template <int HD, int R>
__global__ void __launch_bounds__(256) kv_combine_tiles_kernel(const __grid_constant__ AttnParams p, int n_cta) {
  constexpr int D = 16, PD = HD / D, DW = HD / 8;
  __shared__ float acc_s[8][D][33];
  __shared__ float m_s[8][32], l_s[8][32];
  uint16_t(*const out_s)[HD + 8] = reinterpret_cast<uint16_t(*)[HD + 8]>(&acc_s[0][0][0]);
  static_assert(sizeof(acc_s) >= 32 * (HD + 8) * 2, "the output of 32 rows fits");
  pdl_wait();
  const int lane = threadIdx.x & 31, team = threadIdx.x >> 5;
  for_pieces<R / 32 * PD>(p, n_cta, [&](const Spanning& b, int c, int piece) {
    const int n = b.last - c + 1;
    const bool few = n <= 8;
    const int r0 = (few ? piece : piece / PD) * 32, d0 = few ? 0 : piece % PD * D;
    if (r0 >= b.rows) return;
    const int r = min(r0 + lane, b.rows - 1);
    auto slot = [&](int k) { return p.part + (int64_t)(2 * (c + k) + (k == 0 ? 1 : 0)) * (R * (HD + 2)) + r; };
    float l = 0.f, m = -INFINITY;
    if (few) {
      float acc[DW] = {};
#pragma unroll 2
      for (int k = 0; k < n; ++k) {
        const float* s = slot(k);
        float x[DW];
#pragma unroll
        for (int i = 0; i < DW; ++i) x[i] = s[(team * DW + i) * R];
        join(m, l, acc, s[HD * R], s[(HD + 1) * R], x);
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int i = 0; i < DW; i += 2) {
        const float x = l == 0.f ? 0.f : acc[i] * inv, y = l == 0.f ? 0.f : acc[i + 1] * inv;
        *reinterpret_cast<uint32_t*>(&out_s[lane][team * DW + i]) = p.is_bf16 ? pack2<true>(x, y) : pack2<false>(x, y);
      }
      if (team == 0 && r0 + lane < b.rows) store_lse(p, b.row0, b.row_lo + r, b.head, m, l);
      __syncthreads();
      for (int i = threadIdx.x; i < 32 * HD / 8; i += 256) {
        const int row = i / (HD / 8), d = 8 * (i % (HD / 8)), of = b.row_lo + r0 + row, tok = of / p.group;
        if (r0 + row >= b.rows) break;
        uint16_t* const o = p.out + (int64_t)(b.row0 + tok) * p.out_stride + (int64_t)(b.head * p.group + of - tok * p.group) * HD + d;
        if (p.vec_out16) {
          *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(&out_s[row][d]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = out_s[row][d + e];
        }
      }
      __syncthreads();
      return;
    }
    float acc[D] = {};
#pragma unroll 2
    for (int k = team; k < n; k += 8) {
      const float* s = slot(k);
      float x[D];
#pragma unroll
      for (int i = 0; i < D; ++i) x[i] = s[(d0 + i) * R];
      join(m, l, acc, s[HD * R], s[(HD + 1) * R], x);
    }
#pragma unroll
    for (int i = 0; i < D; ++i) acc_s[team][i][lane] = acc[i];
    m_s[team][lane] = m, l_s[team][lane] = l;
    __syncthreads();
    // thread: row tid / 8, columns 2 (tid % 8) and the next
    const int row = threadIdx.x / 8, d = 2 * (threadIdx.x % 8);
    float top = -INFINITY, x = 0.f, y = 0.f, sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, m_s[k][row]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = ex2(m_s[k][row] - base);
      x = fmaf(acc_s[k][d][row], f, x);
      y = fmaf(acc_s[k][d + 1][row], f, y);
      sum = fmaf(l_s[k][row], f, sum);
    }
    if (r0 + row < b.rows) {
      store_out(p, b.row0, b.row_lo + r0 + row, b.head, d0 + d, HD, sum == 0.f ? 0.f : x / sum);
      store_out(p, b.row0, b.row_lo + r0 + row, b.head, d0 + d + 1, HD, sum == 0.f ? 0.f : y / sum);
      if (d0 == 0 && d == 0) store_lse(p, b.row0, b.row_lo + r0 + row, b.head, top, sum);
    }
    __syncthreads();
  });
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
constexpr int kRowsGrid = kMaxGrid;
constexpr int kTileGrid = kMaxGrid;
constexpr int kCombineGrid = 8 * kMaxGrid;
// Items are not split over CTAs, which saves the partial triples and the second kernel, where an item can have at
// most kWholeTiles tiles (one sequence, 500 positions: 12.0 us against 13.8 split; at 6 tiles 19.7 against 13.8), or
// kWholeTilesMany where there are kMany items or more (64 sequences of 2200 positions: 43.7 against 48.6 us).
constexpr int kWholeTiles = 3, kWholeTilesMany = 8, kMany = 64;
// Rows of a sequence and key/value head that the few-rows kernel takes. With 16 rows it is ahead of the tiles, whose
// second half idles: 64 sequences of 8 K positions 140 against 316 us (e4m3), 189 against 225 us (bf16).
constexpr int kRowsMax = 16;

// The shared memory limit of a kernel, raised once on each device.
template <typename F>
cudaError_t allow_smem(F kernel, size_t bytes, std::atomic<uint64_t>& seen) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (seen.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < 64) seen.fetch_or(uint64_t{1} << dev, std::memory_order_relaxed);
  return e;
}

template <int HD, int KV, int NT>
cudaError_t launch_rows(AttnParams p, int max_rows, cudaStream_t st) {
  using C = RowsCfg<HD, KV, NT>;
  static std::atomic<uint64_t> seen{0};
  p.n_qt = (max_rows + C::R - 1) / C::R;
  p.whole = p.b.max_pages * p.pg.page_size <= (p.b.n_seq * p.pg.n_head_kv >= kMany ? kWholeTilesMany : kWholeTiles) * C::TILE;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  cudaError_t e = allow_smem(kv_rows_kernel<HD, KV, NT>, C::kSmem, seen);
  if (e == cudaSuccess) e = launch_pdl(kv_rows_kernel<HD, KV, NT>, dim3(kRowsGrid), dim3(32 * C::kWarps), C::kSmem, st, p);
  if (e == cudaSuccess && !p.whole) e = launch_pdl(kv_combine_kernel<HD, C::R>, dim3(kCombineGrid), dim3(256), 0, st, p, kRowsGrid);
  return e;
}

template <int HD, int KV>
cudaError_t launch_tiles(AttnParams p, int max_rows, cudaStream_t st) {
  using C = TileCfg<HD, KV>;
  static std::atomic<uint64_t> seen{0};
  p.n_qt = (max_rows + C::R - 1) / C::R;
  p.whole = p.b.max_pages * p.pg.page_size <= (p.b.n_seq * p.pg.n_head_kv >= kMany ? kWholeTilesMany : kWholeTiles) * C::TILE;
  static_assert(C::kSmem <= 220 * 1024, "shared memory");
  cudaError_t e = allow_smem(kv_tile_kernel<HD, KV>, C::kSmem, seen);
  if (e == cudaSuccess) e = launch_pdl(kv_tile_kernel<HD, KV>, dim3(kTileGrid), dim3(C::kThreads), C::kSmem, st, p);
  if (e == cudaSuccess && !p.whole) e = launch_pdl(kv_combine_tiles_kernel<HD, C::R>, dim3(kCombineGrid), dim3(256), 0, st, p, kTileGrid);
  return e;
}

template <int HD, int KV>
cudaError_t launch_kv(const AttnParams& p, int max_rows, cudaStream_t st) {
  return max_rows <= 8          ? launch_rows<HD, KV, 1>(p, max_rows, st)
         : max_rows <= kRowsMax ? launch_rows<HD, KV, 2>(p, max_rows, st)
                                : launch_tiles<HD, KV>(p, max_rows, st);
}

// desc, the waits' error word, partial triples (two a CTA) of the larger row tile that max_rows can need
constexpr size_t kWsHead = kMaxGrid * sizeof(Spanning) + 16;
size_t workspace_bytes_of(int hd, int64_t max_rows) {
  const int64_t rows = max_rows <= kRowsMax ? kRowsMax : 256;
  return kWsHead + (size_t)kMaxGrid * 2 * rows * (hd + 2) * 4;
}
int64_t max_rows_of(const dmoe_kv_cache* c, const dmoe_kv_batch* b, const dmoe_kv_attention_args* a) {
  return std::min<int64_t>(b->max_q_len, a->n_tokens) * (a->n_head / std::max(1, c->n_head_kv));
}

}  // namespace

}  // namespace dmoe

using namespace dmoe;

extern "C" size_t dmoe_kv_attention_workspace(const dmoe_kv_cache* cache, const dmoe_kv_batch* batch,
                                              const dmoe_kv_attention_args* a) {
  if (!cache || !batch || !a || (cache->head_dim != 64 && cache->head_dim != 128)) return 0;
  return workspace_bytes_of(cache->head_dim, max_rows_of(cache, batch, a));
}

extern "C" dmoe_status dmoe_kv_attention(const dmoe_kv_cache* cache, const dmoe_kv_batch* batch,
                                         const dmoe_kv_attention_args* a, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  auto fail = [](dmoe_status st, const char* what) {
    char msg[320];
    snprintf(msg, sizeof(msg), "dmoe_kv_attention: %s", what);
    set_last_error(msg);
    return st;
  };
  if (!a) return fail(DMOE_ERR_INVALID_ARG, "null pointer");
  if (const dmoe_status st = kv_check("dmoe_kv_attention", cache, batch, a->n_tokens, a->n_head)) return st;
  const int hd = cache->head_dim;
  if (a->type != DMOE_TYPE_F16 && a->type != DMOE_TYPE_BF16)
    return fail(DMOE_ERR_UNSUPPORTED, "q and out are f16 or bf16");
  if (a->block_length <= 0) return fail(DMOE_ERR_INVALID_ARG, "block_length must be positive");
  if (!(a->scale > 0.f && a->scale < INFINITY)) return fail(DMOE_ERR_INVALID_ARG, "scale must be positive and finite");
  if (a->q_stride < (int64_t)a->n_head * hd || a->out_stride < (int64_t)a->n_head * hd)
    return fail(DMOE_ERR_INVALID_ARG, "q_stride or out_stride is shorter than a row");
  const int group = a->n_head / cache->n_head_kv;
  if (((int64_t)std::min<int64_t>(batch->max_q_len, a->n_tokens) * group + 7) * std::max(1, batch->n_seq) > INT32_MAX)
    return fail(DMOE_ERR_UNSUPPORTED, "n_seq * max_q_len * n_head / n_head_kv must be below 2^31");
  {
    // units of work, at most: row tiles of 8 or 256 rows, by tiles of 128 positions at least (the last one partly filled)
    const int64_t rows = max_rows_of(cache, batch, a), tile = rows <= kRowsMax ? 8 : 256;
    const double items = std::min((double)batch->n_seq * ((rows + tile - 1) / tile), (double)a->n_tokens * group / tile + batch->n_seq);
    if (items * (std::ceil((double)batch->max_pages * cache->page_size / 128) + 4) * cache->n_head_kv >= 2147483648.0)
      return fail(DMOE_ERR_UNSUPPORTED, "rows times positions of the page table too many for one call");
  }
  if (a->n_tokens == 0 || batch->n_seq == 0 || batch->max_q_len == 0) return DMOE_OK;
  if (!a->q || !a->out || !workspace) return fail(DMOE_ERR_INVALID_ARG, "null pointer");
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 1u ||
      reinterpret_cast<uintptr_t>(a->lse) & 3u)
    return fail(DMOE_ERR_INVALID_ARG, "q, out or lse is not aligned to its elements");
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return fail(DMOE_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
  if (workspace_bytes < dmoe_kv_attention_workspace(cache, batch, a)) return fail(DMOE_ERR_INVALID_ARG, "workspace is too small");

  const NvtxRange nvtx_call("dmoe_kv_attention");
  AttnParams p{};
  p.pg = kv_pages(cache);
  p.b = kv_batch(batch, a->n_tokens);
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  p.q_stride = a->q_stride;
  p.out_stride = a->out_stride;
  p.is_bf16 = a->type == DMOE_TYPE_BF16;
  p.n_head = a->n_head;
  p.group = group;
  p.group_magic = (uint32_t)(((1u << 28) + group - 1) / group);
  p.block_length = a->block_length;
  p.vec_q = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(2 * a->q_stride)) & 7u) == 0;
  p.vec_q16 = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(2 * a->q_stride)) & 15u) == 0;
  p.vec_out16 = ((reinterpret_cast<uintptr_t>(a->out) | (uintptr_t)(2 * a->out_stride)) & 15u) == 0;
  p.scale_log2 = a->scale * kLog2e;
  p.desc = static_cast<Spanning*>(workspace);
  p.wait_err = cache->err ? cache->err : reinterpret_cast<uint32_t*>(p.desc + kMaxGrid);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kWsHead);
  const int max_rows = (int)max_rows_of(cache, batch, a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const KvType kv = kv_type_of(cache->type);
  cudaError_t e;
  set_pdl_for_call(true);
  if (hd == 128)
    e = kv == KV_BF16 ? launch_kv<128, KV_BF16>(p, max_rows, st) : kv == KV_F16 ? launch_kv<128, KV_F16>(p, max_rows, st) : launch_kv<128, KV_E4M3>(p, max_rows, st);
  else
    e = kv == KV_BF16 ? launch_kv<64, KV_BF16>(p, max_rows, st) : kv == KV_F16 ? launch_kv<64, KV_F16>(p, max_rows, st) : launch_kv<64, KV_E4M3>(p, max_rows, st);
  set_pdl_for_call(false);
  if (e != cudaSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "launch failed: %s", cudaGetErrorString(e));
    return fail(DMOE_ERR_CUDA, msg);
  }
  return DMOE_OK;
}
