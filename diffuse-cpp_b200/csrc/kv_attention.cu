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
// The value scale rides in the exponent, so p <= 1 is rounded to f16 relative to the largest weight
// times value scale and neither factor can leave f16's range. Queries are brought into [-1, 1] by a
// power of two per row (exact). M and both sums are 32-bit; p is rounded once, to the products' type.
//
// Work split: the tiles of all (sequence, row tile, key/value head) items are numbered through, and every
// CTA takes an equal run of them, whatever the lengths: a long sequence spreads over the GPU and short
// ones share a CTA. An item that spans CTAs leaves partial (o, M, sum) triples in the workspace, which
// kv_combine_kernel adds in a fixed order (results do not depend on timing).
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "dmoe_internal.h"
#include "kv_common.cuh"
#include "sm100.cuh"

namespace dmoe {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnParams {
  KvPages pg;
  KvBatch b;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int64_t q_stride, out_stride;
  int is_bf16;       // type of q and out
  int n_head, group;
  int block_length;
  int n_qt;          // row tiles a sequence can have (max_q_len)
  int vec_q;         // q rows allow 8-byte loads
  float scale_log2;  // scale * log2(e)
  float* part;       // partial triples, slot = 2 * CTA + (the item begins in this CTA)
  int4* desc;        // [CTA] {item, head, last CTA, 1} of the item this CTA begins and does not end
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  it.seq = u / p.n_qt;
  it.q = kv_sequence(p.b, p.pg, it.seq);
  it.row_lo = (u % p.n_qt) * R;
  it.rows = min(R, it.q.q_len * p.group - it.row_lo);
  it.tiles = 0;
  if (it.rows > 0) it.tiles = max(1, (row_limit(p, it.q, it.row_lo + it.rows - 1) + TILE - 1) / TILE);
  return it;
}

struct Run {       // a CTA's run of tiles
  int u, head;     // first item
  int64_t tile;    // first tile within it
  int64_t left;    // tiles of the run
  int64_t chunk;   // tiles of every run but the last
  int64_t first;   // number of the first tile
};

// The whole CTA: finds its run. smem: scratch of THREADS / 32 + 1 words and one Run.
template <int R, int TILE, int THREADS>
__device__ __forceinline__ Run find_run(const AttnParams& p, int64_t* sums, Run* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t n_u = (int64_t)p.b.n_seq * p.n_qt;
  const int64_t per = (n_u + THREADS - 1) / THREADS;
  const int64_t u0 = min(n_u, per * tid), u1 = min(n_u, u0 + per);
  int64_t mine = 0;
  for (int64_t u = u0; u < u1; ++u) mine += item_of<R, TILE>(p, (int)u).tiles;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sums[warp] = incl;
  if (tid == 0) found->left = 0;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const int heads = p.pg.n_head_kv;
  total *= heads;
  const int64_t chunk = (total + gridDim.x - 1) / gridDim.x;
  const int64_t first = chunk * blockIdx.x;
  before *= heads;
  if (first < total && first >= before && first < before + mine * heads) {
    for (int64_t u = u0; u < u1; ++u) {
      const int64_t w = item_of<R, TILE>(p, (int)u).tiles;
      if (first < before + w * heads) {
        found->u = (int)u;
        found->head = (int)((first - before) / w);
        found->tile = (first - before) % w;
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

__device__ __forceinline__ void store_out(const AttnParams& p, const KvSeq& q, int row, int head, int d, int hd, float x) {
  const int64_t at = (int64_t)(q.row0 + row / p.group) * p.out_stride + (int64_t)(head * p.group + row % p.group) * hd + d;
  if (p.is_bf16)
    p.out[at] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
  else
    p.out[at] = __half_as_ushort(__float2half_rn(x));
}

__device__ __forceinline__ void store_lse(const AttnParams& p, const KvSeq& q, int row, int head, float m, float l) {
  if (p.lse)
    p.lse[(int64_t)(q.row0 + row / p.group) * p.n_head + head * p.group + row % p.group] =
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
// Bound by HBM: the bytes of the pages; each warp loads the next keys while it works on the values.
// ---------------------------------------------------------------------------------------------
template <int HD, int KV, int NT>
struct RowsCfg {
  static constexpr int kWarps = 8;
  static constexpr int R = 8 * NT;
  static constexpr int MT = KV == KV_E4M3 ? 2 : 1;  // 16-position product tiles a step
  static constexpr int STEP = 16 * MT;
  static constexpr int TILE = kWarps * STEP;
  static constexpr int ES = KV == KV_E4M3 ? 1 : 2;
  static constexpr size_t kSmem = (size_t)kWarps * R * (HD + 2) * 4;
  static constexpr int kPart = R * (HD + 2);  // floats of a partial triple
};

template <int HD, int KV, int NT>
__global__ void __launch_bounds__(256, 1) kv_rows_kernel(const __grid_constant__ AttnParams p) {
  using C = RowsCfg<HD, KV, NT>;
  constexpr bool kBf = KV == KV_BF16;
  constexpr int R = C::R, MT = C::MT, STEP = C::STEP, TILE = C::TILE, ES = C::ES;
  constexpr int KCH = HD * ES / 64;        // 16-byte loads of a key row by each of 4 lanes
  constexpr int VB = HD * ES / 8;          // bytes of a value row by each of 8 lanes: 8, 16 or 32
  constexpr int VW = VB / 4;
  constexpr int JT = HD / 16;              // 16-row tiles of o^T
  extern __shared__ float smem_f[];
  __shared__ int64_t sums[C::kWarps];
  __shared__ Run found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  Run run = find_run<R, TILE, 256>(p, sums, &found);
  int4 begun = make_int4(0, 0, 0, 0);
  int64_t at = run.first;
  int u = run.u, head = run.head;
  int64_t tile0 = run.tile;
  Item it{};
  if (run.left > 0) it = item_of<R, TILE>(p, u);
  while (run.left > 0) {
    const int64_t tile1 = min((int64_t)it.tiles, tile0 + run.left);
    // queries: lane (g, t) holds row g of each 8-row tile, at the elements its key chunks cover
    uint32_t qf[NT][HD / 16][2];
    float cq[NT][2];  // score factor and limit of the rows 2t, 2t + 1 of each tile
    int lim[NT][2];
    int lim_min = INT32_MAX, lim_max = 0;
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
      // f16 products: rows scaled into [-1, 1]
      const int e = kBf ? 0 : min(max((int)(__float_as_uint(amax) >> 23) - 126, -100), 100);
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
    lim_min = row_limit(p, it.q, it.row_lo);
    lim_max = row_limit(p, it.q, it.row_lo + it.rows - 1);

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

    const int end = (int)min((int64_t)lim_max, tile1 * TILE);  // positions of this segment
    int pos = (int)(tile0 * TILE) + warp * STEP;
    const int32_t* table = p.b.table + it.seq * p.b.max_pages;
    uint32_t kr[MT][2][KCH][4];
    int64_t row = 0;
    int ek = 0, ev = 0;
    // page of a step's positions (a step lies in one scale block, so in one page), scales and keys
    auto load_keys = [&](int at_pos) {
      int64_t page = table[at_pos / p.pg.page_size];
      if (page < 0 || page >= p.pg.n_pages) {
        kv_report(p.pg.err, DMOE_KV_ERR_PAGE);
        page = 0;
      }
      row = kv_row(p.pg, page, head, at_pos % p.pg.page_size);
      if (KV == KV_E4M3) {
        ek = (int)p.pg.k_scale[row / kScaleBlock] - 127;
        ev = (int)p.pg.v_scale[row / kScaleBlock] - 127;
      }
      const uint8_t* base = static_cast<const uint8_t*>(p.pg.k) + row * (HD * ES);
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < KCH; ++c) {
            const uint4 v = __ldcs(reinterpret_cast<const uint4*>(base + (16 * a + 8 * h + g) * (HD * ES) + 16 * (t + 4 * c)));
            kr[a][h][c][0] = v.x, kr[a][h][c][1] = v.y, kr[a][h][c][2] = v.z, kr[a][h][c][3] = v.w;
          }
    };
    if (pos < end) load_keys(pos);
    for (; pos < end; pos += C::kWarps * STEP) {
      // this step's values
      uint32_t vr[MT][4][VW];
      const uint8_t* vbase = static_cast<const uint8_t*>(p.pg.v) + row * (HD * ES);
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint8_t* src = vbase + (16 * a + 2 * t + (k & 1) + 8 * (k >> 1)) * (HD * ES);
          if (VB == 8) {
            const uint2 v = __ldcs(reinterpret_cast<const uint2*>(src + 8 * g));
            vr[a][k][0] = v.x, vr[a][k][1] = v.y;
          } else {
#pragma unroll
            for (int c = 0; c < VB / 16; ++c) {
              const uint4 v = __ldcs(reinterpret_cast<const uint4*>(src + 16 * (g + 8 * c)));
              vr[a][k][4 * c] = v.x, vr[a][k][4 * c + 1] = v.y, vr[a][k][4 * c + 2] = v.z, vr[a][k][4 * c + 3] = v.w;
            }
          }
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
      const float sk = KV == KV_E4M3 ? pow2i(ek) : 1.f, evf = KV == KV_E4M3 ? (float)ev : 0.f;
      const float unv = KV == KV_E4M3 ? pow2i(-ev) : 1.f;
      const int here = pos;
      const bool edge = here + STEP > lim_min;
      if (pos + C::kWarps * STEP < end) load_keys(pos + C::kWarps * STEP);  // the next step's keys

      // scores -> weights. Lane (g, t): positions 16a + g and 16a + 8 + g, rows 2t and 2t + 1
      uint32_t pf[NT][MT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = fmaf(s[n][a][i], cq[n][i & 1] * sk, evf);
            if (edge && here + 16 * a + 8 * (i >> 1) + g >= lim[n][i & 1]) x = -INFINITY;
            s[n][a][i] = x;
            mx[i & 1] = fmaxf(mx[i & 1], x);
          }
        float base[2], shrink[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], off));
          const float mn = fmaxf(m[n][i], mx[i]);
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

    // join the warps: o, M and the sum of each row
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
    const bool whole = tile0 == 0 && tile1 == it.tiles;
    float* part = p.part + (int64_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * C::kPart;
    for (int i = tid; i < it.rows * HD; i += 256) {
      const int r = i / HD, d = i % HD;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) mm = fmaxf(mm, ml[(w * R + r) * 2]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float acc = 0.f, ll = 0.f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float f = ex2(ml[(w * R + r) * 2] - base);
        acc = fmaf(os[(w * R + r) * HD + d], f, acc);
        ll = fmaf(ml[(w * R + r) * 2 + 1], f, ll);
      }
      if (whole) {
        store_out(p, it.q, it.row_lo + r, head, d, HD, ll == 0.f ? 0.f : acc / ll);
        if (d == 0) store_lse(p, it.q, it.row_lo + r, head, mm, ll);
      } else {
        part[r * HD + d] = acc;
        if (d == 0) part[R * HD + 2 * r] = mm, part[R * HD + 2 * r + 1] = ll;
      }
    }
    if (!whole && tile0 == 0)
      begun = make_int4(u, head, (int)((at + it.tiles - 1) / run.chunk), 1);
    __syncthreads();  // os and ml are free again
    run.left -= tile1 - tile0;
    at += tile1 - tile0;
    tile0 = 0;
    if (run.left > 0 && ++head == p.pg.n_head_kv) {
      head = 0;
      do it = item_of<R, TILE>(p, ++u);
      while (it.tiles == 0);
    }
  }
  if (tid == 0) p.desc[blockIdx.x] = begun;
  pdl_trigger();
}

// Adds the partial triples of the item that CTA blockIdx.x of the first kernel began: those of
// slots 2c + 1, 2(c + 1), .. 2 last, in that order. One CTA a row: 8 groups of HD / 4 threads.. take every
// eighth triple, then their sums are added in order.
template <int HD, int R, int TILE>
__global__ void __launch_bounds__(8 * HD / 4) kv_combine_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kLanes = HD / 4;
  __shared__ float4 acc_s[8][kLanes];
  __shared__ float l_s[8];
  pdl_wait();
  const int c = blockIdx.x, r = blockIdx.y;
  const int4 begun = p.desc[c];
  if (begun.w == 0) return;
  const Item it = item_of<R, TILE>(p, begun.x);
  if (r >= it.rows) return;
  const int n = begun.z - c + 1;
  const int sub = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  auto slot = [&](int k) { return p.part + (int64_t)(2 * (c + k) + (k == 0 ? 1 : 0)) * (R * (HD + 2)); };
  float m = -INFINITY;
  for (int k = 0; k < n; ++k) m = fmaxf(m, slot(k)[R * HD + 2 * r]);
  const float base = m == -INFINITY ? 0.f : m;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int k = grp; k < n; k += 8) {
    const float* s = slot(k);
    const float f = ex2(s[R * HD + 2 * r] - base);
    const float4 v = reinterpret_cast<const float4*>(s + r * HD)[sub];
    acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
    l = fmaf(s[R * HD + 2 * r + 1], f, l);
  }
  acc_s[grp][sub] = acc;
  if (sub == 0) l_s[grp] = l;
  __syncthreads();
  if (grp != 0) return;
  for (int k = 1; k < 8; ++k) {
    const float4 v = acc_s[k][sub];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    l += l_s[k];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float x[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
  for (int i = 0; i < 4; ++i) store_out(p, it.q, it.row_lo + r, begun.y, 4 * sub + i, HD, l == 0.f ? 0.f : x[i]);
  if (sub == 0) store_lse(p, it.q, it.row_lo + r, begun.y, m, l);
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
constexpr int kRowsGrid = 148;
constexpr int kMaxGrid = 148;

template <int HD, int KV, int NT>
cudaError_t launch_rows(AttnParams p, int max_rows, cudaStream_t st) {
  using C = RowsCfg<HD, KV, NT>;
  p.n_qt = (max_rows + C::R - 1) / C::R;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(kv_rows_kernel<HD, KV, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
  if (e != cudaSuccess) return e;
  kv_rows_kernel<HD, KV, NT><<<kRowsGrid, 256, C::kSmem, st>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  set_pdl_for_call(true);
  e = launch_pdl(kv_combine_kernel<HD, C::R, C::TILE>, dim3(kRowsGrid, C::R), dim3(8 * HD / 4), 0, st, p);
  set_pdl_for_call(false);
  return e;
}

template <int HD, int KV>
cudaError_t launch_kv(const AttnParams& p, int max_rows, cudaStream_t st) {
  return max_rows <= 8 ? launch_rows<HD, KV, 1>(p, max_rows, st) : launch_rows<HD, KV, 2>(p, max_rows, st);
}

size_t workspace_bytes_of(int hd) { return (size_t)kMaxGrid * (2 * 16 * (hd + 2) * 4 + sizeof(int4)); }

}  // namespace

}  // namespace dmoe

using namespace dmoe;

extern "C" size_t dmoe_kv_attention_workspace(const dmoe_kv_cache* cache, const dmoe_kv_batch* batch,
                                              const dmoe_kv_attention_args* a) {
  if (!cache || !batch || !a || (cache->head_dim != 64 && cache->head_dim != 128)) return 0;
  return workspace_bytes_of(cache->head_dim);
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
  p.block_length = a->block_length;
  p.vec_q = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(2 * a->q_stride)) & 7u) == 0;
  p.scale_log2 = a->scale * kLog2e;
  p.desc = static_cast<int4*>(workspace);
  p.part = reinterpret_cast<float*>(p.desc + kMaxGrid);
  const int max_rows = (int)std::min<int64_t>(batch->max_q_len, a->n_tokens) * group;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const KvType kv = kv_type_of(cache->type);
  cudaError_t e;
  if (hd == 128)
    e = kv == KV_BF16 ? launch_kv<128, KV_BF16>(p, max_rows, st) : kv == KV_F16 ? launch_kv<128, KV_F16>(p, max_rows, st) : launch_kv<128, KV_E4M3>(p, max_rows, st);
  else
    e = kv == KV_BF16 ? launch_kv<64, KV_BF16>(p, max_rows, st) : kv == KV_F16 ? launch_kv<64, KV_F16>(p, max_rows, st) : launch_kv<64, KV_E4M3>(p, max_rows, st);
  if (e != cudaSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "launch failed: %s", cudaGetErrorString(e));
    return fail(DMOE_ERR_CUDA, msg);
  }
  return DMOE_OK;
}
