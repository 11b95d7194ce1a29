// kv_append.cu — dmoe_kv_append: QK norm, rotation and the write of keys and values into a paged
// cache, with the rotated queries as output.
//
// Reference: the fused QKV's split, QK norm and RoPE of src/diffuse-moe-graph.cpp:126-161. For a
// row x of a query or key head: y = x / sqrt(mean x^2 + eps) * w, then (y_i, y_{i + r/2}) turns by
// theta_i = position * base^(-2i / r) for i < r / 2. The angle is taken in turns in 64 bits (at position 131072 a
// 32-bit angle is already 0.004 off); sine and cosine of its fraction in 32, with what the rounding left added.
//
// Pages of 8 bits: for each (32-position block, head) e = the smallest exponent with amax <= 448 * 2^e,
// and e4m3(x * 2^-e) is stored, as it follows from x in 64 bits (a 32-bit x turns a code in ten million, and a scale
// now and then; keys are few beside the queries). A power of two as scale loses nothing against any other scale (e4m3
// keeps 4 significant bits at every size) and makes the move of kept values to a new scale exact.
//
// Work unit: a 32-position block of one sequence that gains rows (the grid is an upper bound of their
// number, and every warp finds its unit by a scan of the batch). gridDim.y divides the heads: first the
// groups of heads whose rows are independent (queries; keys and values too in 16-bit pages), then, for
// 8-bit pages, the groups of key / value heads, where the CTA holds a block of one head in registers
// until its amax is known. 16 lanes (head_dim 128) or 8 (64) share a row, 8 elements each: 16-byte
// loads of 16-bit rows, two or four rows a warp at once, and half the shuffles of a warp per row.
//
// Measured on B200 (32 + 4 + 4 heads of 128, rotary_dim 64, e4m3): a 16384-token prompt, 318.8 MB, 120 us = 2.7 TB/s, 41 %
// of the copy rate (17 us less with keys in 32 bits). Instruction issue bounds it, not HBM: norm, rotation and conversion
// take about 150 instructions per 8 elements. One block of 32 positions: 10 us a call, most of it the launch and
// the host. Many single tokens: every warp scans the batch for its unit, which takes most of the time beyond some hundreds
// of sequences (1024: 102 us, 4096: 786 us).
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "dmoe_internal.h"
#include "kv_common.cuh"
#include "sm100.cuh"

namespace dmoe {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxHalf = 64;  // rotary_dim / 2 at head_dim 128
constexpr int kWantedHeld = 148 * 3;  // of them for the keys of 8-bit pages, whose table is dearer (prompt: 123 us at 6 an SM)
// CTAs of a large call (16384-token prompt: 119 us at 4 or 6 an SM, 128 at 12, 139 at 24; 24 x 64 rows into bf16 pages:
// 21.2, 20.7, 23.0, 32.8)
constexpr int kWanted = 148 * 6;

struct AppendParams {
  KvPages pg;
  KvBatch b;
  const void* qkv;
  void* q_out;
  const float* q_norm;
  const float* k_norm;
  int64_t qkv_stride, q_stride;
  int q_type;
  int n_head;
  int half;          // rotary_dim / 2
  uint32_t half_magic;  // ceil(2^18 / half): i / half for i < 2^11 (i * error < 2^11 * 2^6)
  int flat_slots;    // heads of the independent rows: [0, flat_slots)
  int flat_per_cta, flat_groups;  // heads a CTA takes of them, and how many such groups
  int held_per_cta, held_groups;  // the same of the key heads, and of the value heads, of 8-bit pages
  int vec_in, vec_out;  // rows are 16-byte aligned
  float eps;
  double turns[kMaxHalf];  // base^(-2i / rotary_dim) / 2 pi
};

// 8 consecutive elements as they are, by 16-byte loads when `vec`, and as floats.
template <int IN>
struct Raw8 {
  uint32_t w[IN == DMOE_TYPE_F32 ? 8 : 4];
  __device__ __forceinline__ void load(const void* p, int64_t at, int vec) {
    constexpr int N = IN == DMOE_TYPE_F32 ? 2 : 1;
    if (vec) {
      const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (IN == DMOE_TYPE_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint4 v = __ldcs(s + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if (IN == DMOE_TYPE_F32) {
#pragma unroll
      for (int i = 0; i < 4 * N; ++i) w[i] = __ldcs(static_cast<const uint32_t*>(p) + at + i);
    } else {
      const uint16_t* h = static_cast<const uint16_t*>(p) + at;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __ldcs(h + 2 * i) | ((uint32_t)__ldcs(h + 2 * i + 1) << 16);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (IN == DMOE_TYPE_F32 ? 8 : 4); ++i) w[i] = 0;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (IN == DMOE_TYPE_F32) {
        x[2 * i] = __uint_as_float(w[2 * i]), x[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
      } else if constexpr (IN == DMOE_TYPE_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

__device__ __forceinline__ uint4 pack8(const float (&x)[8], int type) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (type == DMOE_TYPE_F16) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void store8(void* p, int64_t at, int type, int vec, const float (&x)[8]) {
  if (type == DMOE_TYPE_F32) {
    float* f = static_cast<float*>(p) + at;
    if (vec) {
      reinterpret_cast<float4*>(f)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(f)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = x[i];
    }
    return;
  }
  const uint4 w = pack8(x, type);
  uint16_t* h = static_cast<uint16_t*>(p) + at;
  if (vec) {
    *reinterpret_cast<uint4*>(h) = w;
  } else {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
  }
}

// A lane's 8 weights of a norm; ones where there is none.
__device__ __forceinline__ void load_weights(const float* w, int sub, float (&g)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 v = w ? __ldg(reinterpret_cast<const float4*>(w) + 2 * sub + i) : make_float4(1.f, 1.f, 1.f, 1.f);
    g[4 * i] = v.x, g[4 * i + 1] = v.y, g[4 * i + 2] = v.z, g[4 * i + 3] = v.w;
  }
}

// y = norm(x) * w, then the rotation; every lane of the warp takes part (LPR lanes hold one row).
// cs: the row's (cos, sin) pairs.
template <int LPR>
__device__ __forceinline__ void norm_rotate(float (&x)[8], const float (&w)[8], bool norm, float eps, int sub, int half,
                                            const float2* cs) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  float m = fmaf(ss, 1.0f / (8 * LPR), eps), r = rsqrtf(m);
  // a root outside [2^-50, 2^50]: its squares may have left the range of 32 bits. The row times a power of two
  const bool far = norm && __float_as_uint(r) - __float_as_uint(0x1p-50f) > __float_as_uint(0x1p50f) - __float_as_uint(0x1p-50f);
  if (__any_sync(0xffffffffu, far)) {
    const float s = !far ? 1.0f : m > 1.0f ? 0x1p-100f : 0x1p100f;
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= s, ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    m = fmaf(ss, 1.0f / (8 * LPR), eps * s * s);
    r = rsqrtf(m);
    if (m == INFINITY) m = 0.f;  // r is 0 and stays it
  }
  r = norm ? fmaf(0.5f * r, fmaf(-m * r, r, 1.0f), r) : 1.0f;  // a Newton step: two units in the last place become one half
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
  if (half == 0) return;
  const int hl = half / 8;
  const bool lo = sub < hl, in = sub < 2 * hl;
  const int lane = threadIdx.x & 31, from = lane + (lo ? hl : in ? -hl : 0);
  const float4* c = reinterpret_cast<const float4*>(cs + 8 * (lo ? sub : in ? sub - hl : 0));
  const float sign = lo ? -1.f : 1.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float y0 = __shfl_sync(0xffffffffu, x[i], from), y1 = __shfl_sync(0xffffffffu, x[i + 1], from);
    const float4 t = c[i / 2];
    if (in) {
      x[i] = fmaf(x[i], t.x, sign * (y0 * t.y));
      x[i + 1] = fmaf(x[i + 1], t.z, sign * (y1 * t.w));
    }
  }
}

__device__ __forceinline__ double shfl_double(double x, int from) {
  return __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(x), from), __shfl_sync(0xffffffffu, __double2loint(x), from));
}

// norm_rotate in 64 bits, for values that 3 bits are cut from next: each result is rounded to odd (cut to 32 bits, the
// last bit set if anything was cut off), so that the second rounding, and the comparison with a scale's border,
// come out as for the exact value.
template <int LPR>
__device__ __forceinline__ void norm_rotate_exact(float (&x)[8], const float (&w)[8], bool norm, float eps, int sub, int half,
                                                  const double2* cs) {
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fma((double)x[i], (double)x[i], ss);
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) ss += shfl_double(ss, (threadIdx.x & 31) ^ o);
  const double r = norm ? rsqrt(ss * (1.0 / (8 * LPR)) + (double)eps) : 1.0;
  const int hl = half / 8;
  const bool lo = sub < hl, in = sub < 2 * hl;
  const int lane = threadIdx.x & 31, from = lane + (lo ? hl : in ? -hl : 0);
  const double2* c = cs + 8 * (lo ? sub : in ? sub - hl : 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double y = (double)x[i] * r * (double)w[i];
    if (half) {
      const double z = shfl_double(y, from);
      if (in) {
        const double2 t = c[i];
        y = lo ? y * t.x - z * t.y : y * t.x + z * t.y;
      }
    }
    const float f = __double2float_rz(y);
    x[i] = (double)f == y ? f : __int_as_float(__float_as_int(f) | 1);
  }
}

// Scale exponent of a block: amax = f 2^x with 1 <= f < 2, and 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kExpMin), kExpMax);  // zero and subnormal amax: the smallest
}

__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = make_float2(x[4 * j + 2 * i] * inv, x[4 * j + 2 * i + 1] * inv);
      uint32_t h = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);  // round to nearest even
      if (!(fabsf(f.x) < INFINITY)) h = (h & 0xff00u) | 0x7fu;  // no infinity in e4m3: NaN
      if (!(fabsf(f.y) < INFINITY)) h = (h & 0x00ffu) | 0x7f00u;
      o |= h << (16 * i);
    }
    w[j] = o;
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void dequantise8(uint2 w, float scale, float (&x)[8]) {
  const uint32_t v[2] = {w.x, w.y};
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v[j] >> (16 * i)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[4 * j + 2 * i] = f.x * scale, x[4 * j + 2 * i + 1] = f.y * scale;
    }
}

template <int HD, int KV, int IN>
__global__ void __launch_bounds__(kThreads, 4) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LPR = HD / 8;     // lanes a row
  constexpr int RPW = 32 / LPR;   // rows a warp holds at once
  constexpr int PASSES = kScaleBlock / (kWarps * RPW);
  // (cos, sin) of the block's positions: [position][i] float2, or double2 for the keys of 8-bit pages
  __shared__ __align__(16) uint8_t table[kScaleBlock * kMaxHalf * (KV == KV_E4M3 ? 16 : 8)];
  float2* const cs = reinterpret_cast<float2*>(table);
  double2* const cs64 = reinterpret_cast<double2*>(table);
  __shared__ float amax_s[2][kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LPR;

  pdl_wait();
  // this CTA's unit: block `rel` among those of sequence `s` that gain rows
  int s = -1, rel = (int)blockIdx.x;
  KvSeq q{};
  for (int base = 0; base < p.b.n_seq; base += 32) {
    KvSeq t{};
    int nb = 0;
    if (base + lane < p.b.n_seq) {
      t = kv_sequence(p.b, p.pg, base + lane);
      const int p0 = max(0, t.kv_len - t.q_len);
      if (t.q_len > 0) nb = t.kv_len > p0 ? (t.kv_len - 1) / kScaleBlock - p0 / kScaleBlock + 1 : 1;
    }
    int sum = nb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, sum > rel);
    if (hit) {
      const int l = __ffs(hit) - 1;
      rel -= __shfl_sync(0xffffffffu, sum - nb, l);
      q.row0 = __shfl_sync(0xffffffffu, t.row0, l);
      q.q_len = __shfl_sync(0xffffffffu, t.q_len, l);
      q.kv_len = __shfl_sync(0xffffffffu, t.kv_len, l);
      s = base + l;
      break;
    }
    rel -= __shfl_sync(0xffffffffu, sum, 31);
  }
  if (s < 0) return;
  const int pos0 = q.kv_len - q.q_len;  // position of the sequence's first row; negative: padding rows
  const int b0 = (max(0, pos0) / kScaleBlock + rel) * kScaleBlock;
  const int lo = max(b0, pos0), hi = min(b0 + kScaleBlock, q.kv_len);  // positions that are written
  const int fresh = max(0, hi - lo);
  int64_t page = -1;
  if (fresh > 0) {
    page = p.b.table[s * p.b.max_pages + b0 / p.pg.page_size];
    if (page < 0 || page >= p.pg.n_pages) {
      kv_report(p.pg.err, DMOE_KV_ERR_PAGE);
      page = -1;
    }
  }
  const int off0 = b0 % p.pg.page_size;
  const int64_t row_lo = (int64_t)q.row0 + (lo - pos0);  // row of position lo
  const int group = (int)blockIdx.y;

  // (cos, sin) of the block's new positions, once for all heads of the CTA; values are not rotated
  const bool values = group >= p.flat_groups + p.held_groups;
  for (int i = tid; i < (values ? 0 : fresh * p.half); i += kThreads) {
    const int t = (int)((i * p.half_magic) >> 18), f = i - t * p.half;
    const double a = (double)(lo + t) * p.turns[f];
    const double turn = a - rint(a);
    if (KV == KV_E4M3 && group >= p.flat_groups) {
      double sn, c;
      sincospi(2.0 * turn, &sn, &c);
      cs64[(lo - b0 + t) * kMaxHalf + f] = make_double2(c, sn);
      continue;
    }
    const float hi = (float)turn, rest = 6.2831853f * (float)(turn - hi);  // what 24 bits leave of the angle
    float sn, c;
    sincospif(2.0f * hi, &sn, &c);
    cs[(lo - b0 + t) * kMaxHalf + f] = make_float2(fmaf(-sn, rest, c), fmaf(c, rest, sn));
  }
  __syncthreads();

  if (group < p.flat_groups) {
    const int h0 = group * p.flat_per_cta, nh = min(p.flat_per_cta, p.flat_slots - h0);
    if (rel == 0 && pos0 < 0) {  // padding rows: zero queries
      const int pad = min(-pos0, q.q_len);
      const float zero[8] = {};
      constexpr int kSome = 1 << 16;  // rows at a time, so that 8-element pieces are numbered in 31 bits
      for (int first = 0; first < pad; first += min(kSome, pad - first))
        for (int r = tid; r < min(kSome, pad - first) * nh * LPR; r += kThreads) {
          const int h = h0 + (r / LPR) % nh;
          if (h < p.n_head)
            store8(p.q_out, (int64_t)(q.row0 + first + r / LPR / nh) * p.q_stride + (int64_t)h * HD + 8 * (r % LPR), p.q_type,
                   p.vec_out, zero);
        }
    }
    float wq[8], wk[8];
    load_weights(p.q_norm, sub, wq);
    load_weights(KV == KV_E4M3 ? p.q_norm : p.k_norm, sub, wk);
    // r / fresh for r < 2^13 (at most 128 heads a CTA) and fresh <= 32: r * (magic * fresh - 2^18) < 2^18
    const uint32_t magic = fresh ? ((1u << 18) + fresh - 1) / fresh : 0;
    // four rows a lane on their way at once
    constexpr int U = IN == DMOE_TYPE_F32 ? 2 : 4;
    for (int r0 = warp * RPW; r0 < fresh * nh; r0 += kWarps * RPW * U) {
      Raw8<IN> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * kWarps * RPW + lane / LPR;
        raw[u].zero();
        if (r < fresh * nh) {
          const int h = (int)((r * magic) >> 18);
          raw[u].load(p.qkv, (row_lo + r - h * fresh) * p.qkv_stride + (int64_t)(h0 + h) * HD + 8 * sub, p.vec_in);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * kWarps * RPW + lane / LPR;
        if (r0 + u * kWarps * RPW >= fresh * nh) break;  // the whole warp
        const bool live = r < fresh * nh;
        const int hr = live ? (int)((r * magic) >> 18) : 0, t = live ? r - hr * fresh : 0, h = h0 + hr;
        const bool is_q = h < p.n_head, is_v = h >= p.n_head + p.pg.n_head_kv;
        float x[8], y[8];
        raw[u].get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
        const float2* const c = cs + (lo - b0 + t) * kMaxHalf;
        if (KV == KV_E4M3) {
          norm_rotate<LPR>(y, wq, p.q_norm != nullptr, p.eps, sub, p.half, c);
        } else if (!__all_sync(0xffffffffu, is_v || !live)) {
          float w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = is_q ? wq[i] : wk[i];
          norm_rotate<LPR>(y, w, (is_q ? p.q_norm : p.k_norm) != nullptr, p.eps, sub, p.half, c);
        }
        if (!live) continue;
        if (KV == KV_E4M3 || is_q) {
          store8(p.q_out, (row_lo + t) * p.q_stride + (int64_t)h * HD + 8 * sub, p.q_type, p.vec_out, y);
        } else if (page >= 0) {
          const int hk = is_v ? h - p.n_head - p.pg.n_head_kv : h - p.n_head;
          const int64_t at = kv_row(p.pg, page, hk, off0 + (lo - b0) + t) * HD + 8 * sub;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = is_v ? x[i] : y[i];
          store8(is_v ? p.pg.v : p.pg.k, at, KV == KV_BF16 ? DMOE_TYPE_BF16 : DMOE_TYPE_F16, 1, y);
        }
      }
    }
    return;
  }
  if (KV != KV_E4M3 || fresh == 0 || page < 0) return;

  const bool is_v = values;
  float wk[8];
  load_weights(is_v ? nullptr : p.k_norm, sub, wk);
  const int hk0 = (group - p.flat_groups - (values ? p.held_groups : 0)) * p.held_per_cta, hk1 = min(hk0 + p.held_per_cta, p.pg.n_head_kv);
  for (int hk = hk0; hk < hk1; ++hk) {
    const int hs = (is_v ? p.pg.n_head_kv : 0) + hk;
    uint8_t* codes = static_cast<uint8_t*>(is_v ? p.pg.v : p.pg.k);
    uint8_t* sc = (is_v ? p.pg.v_scale : p.pg.k_scale) +
                  ((page * p.pg.n_head_kv + hk) * p.pg.page_size + off0) / kScaleBlock;
    const int e_old = lo > b0 ? (int)*sc - 127 : kExpMin;
    float x[PASSES][8];
    float amax = 0.f;
    {
      Raw8<IN> raw[PASSES];
      uint2 kept[PASSES];
#pragma unroll
      for (int j = 0; j < PASSES; ++j) {
        const int t = (j * kWarps + warp) * RPW + lane / LPR, pos = b0 + t;
        raw[j].zero();
        if (pos >= lo && pos < hi)
          raw[j].load(p.qkv, (row_lo + (pos - lo)) * p.qkv_stride + (int64_t)(p.n_head + hs) * HD + 8 * sub, p.vec_in);
        else if (pos < lo)
          kept[j] = *reinterpret_cast<const uint2*>(codes + kv_row(p.pg, page, hk, off0 + t) * HD + 8 * sub);
      }
#pragma unroll
      for (int j = 0; j < PASSES; ++j) {
        raw[j].get(x[j]);
        if (b0 + (j * kWarps + warp) * RPW + lane / LPR < lo) dequantise8(kept[j], exp2f((float)e_old), x[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int t = (j * kWarps + warp) * RPW + lane / LPR;
      if (!is_v) {  // uniform over the CTA; rows that are kept pass through
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[j][i];
        const bool now = b0 + t >= lo && b0 + t < hi;
        norm_rotate_exact<LPR>(y, wk, p.k_norm != nullptr, p.eps, sub, p.half, cs64 + (now ? t : lo - b0) * kMaxHalf);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = now ? y[i] : x[j][i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x[j][i]);
        amax = fmaxf(amax, a < INFINITY ? a : 0.f);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) amax_s[hk & 1][warp] = amax;
    __syncthreads();  // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < kWarps; ++w) amax = fmaxf(amax, amax_s[hk & 1][w]);
    const int e = scale_exponent(amax);
    const float inv = exp2f((float)-e);
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int t = (j * kWarps + warp) * RPW + lane / LPR, pos = b0 + t;
      if (pos < hi && (pos >= lo || e != e_old))
        *reinterpret_cast<uint2*>(codes + kv_row(p.pg, page, hk, off0 + t) * HD + 8 * sub) = quantise8(x[j], inv);
    }
    if (tid == 0) *sc = (uint8_t)(e + 127);
  }
}

template <int IN>
cudaError_t launch_append(const AppendParams& p, int hd, KvType kv, dim3 grid, cudaStream_t st) {
  void (*k)(AppendParams);
  if (hd == 128)
    k = kv == KV_BF16 ? kv_append_kernel<128, KV_BF16, IN> : kv == KV_F16 ? kv_append_kernel<128, KV_F16, IN> : kv_append_kernel<128, KV_E4M3, IN>;
  else
    k = kv == KV_BF16 ? kv_append_kernel<64, KV_BF16, IN> : kv == KV_F16 ? kv_append_kernel<64, KV_F16, IN> : kv_append_kernel<64, KV_E4M3, IN>;
  return launch_pdl(k, grid, dim3(kThreads), 0, st, p);
}

bool is_float_type(int t) { return t == DMOE_TYPE_F32 || t == DMOE_TYPE_F16 || t == DMOE_TYPE_BF16; }
int64_t size_of(int t) { return t == DMOE_TYPE_F32 ? 4 : 2; }
bool aligned16(const void* p, int64_t stride_bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)stride_bytes) & 15u) == 0;
}

}  // namespace

dmoe_status kv_check(const char* call, const dmoe_kv_cache* c, const dmoe_kv_batch* b, int64_t n_tokens, int n_head) {
  char msg[256];
  auto fail = [&](dmoe_status st, const char* what) {
    snprintf(msg, sizeof(msg), "%s: %s", call, what);
    set_last_error(msg);
    return st;
  };
  if (!c || !b) return fail(DMOE_ERR_INVALID_ARG, "null pointer");
  if (n_tokens < 0 || n_tokens > INT32_MAX || b->n_seq < 0 || b->max_q_len < 0 || b->max_pages < 0)
    return fail(DMOE_ERR_INVALID_ARG, "negative size, or 2^31 tokens or more");
  if (c->type != DMOE_TYPE_BF16 && c->type != DMOE_TYPE_F16 && c->type != DMOE_TYPE_E4M3)
    return fail(DMOE_ERR_UNSUPPORTED, "pages are bf16, f16 or e4m3");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(DMOE_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (c->n_head_kv <= 0 || n_head <= 0 || n_head % c->n_head_kv || n_head > 4096)
    return fail(DMOE_ERR_INVALID_ARG, "n_head must be a multiple of n_head_kv, at most 4096");
  if (c->page_size <= 0 || c->page_size % kScaleBlock || c->page_size > 65536)
    return fail(DMOE_ERR_UNSUPPORTED, "page_size must be a multiple of 32, at most 65536");
  if (c->n_pages <= 0 || c->n_pages > INT32_MAX) return fail(DMOE_ERR_INVALID_ARG, "n_pages must be in [1, 2^31)");
  if (b->max_pages > (1 << 30) / c->page_size)
    return fail(DMOE_ERR_UNSUPPORTED, "max_pages * page_size must be at most 2^30");
  if (!c->k || !c->v || (c->type == DMOE_TYPE_E4M3 && (!c->k_scale || !c->v_scale)))
    return fail(DMOE_ERR_INVALID_ARG, "null pointer in the cache");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u)
    return fail(DMOE_ERR_INVALID_ARG, "k and v must be 16-byte aligned");
  if (b->n_seq > 0 && n_tokens > 0 && (!b->q_start || !b->kv_len || (b->max_pages > 0 && !b->page_table)))
    return fail(DMOE_ERR_INVALID_ARG, "null pointer in the batch");
  if ((reinterpret_cast<uintptr_t>(b->q_start) | reinterpret_cast<uintptr_t>(b->kv_len) |
       reinterpret_cast<uintptr_t>(b->page_table) | reinterpret_cast<uintptr_t>(c->err)) & 3u)
    return fail(DMOE_ERR_INVALID_ARG, "q_start, kv_len, page_table and err must be 4-byte aligned");
  return DMOE_OK;
}

}  // namespace dmoe

using namespace dmoe;

extern "C" dmoe_status dmoe_kv_append(const dmoe_kv_cache* cache, const dmoe_kv_batch* batch,
                                      const dmoe_kv_append_args* a, void* stream) {
  auto fail = [](dmoe_status st, const char* what) {
    char msg[320];
    snprintf(msg, sizeof(msg), "dmoe_kv_append: %s", what);
    set_last_error(msg);
    return st;
  };
  if (!a) return fail(DMOE_ERR_INVALID_ARG, "null pointer");
  if (const dmoe_status st = kv_check("dmoe_kv_append", cache, batch, a->n_tokens, a->n_head)) return st;
  const int hd = cache->head_dim, nk = cache->n_head_kv;
  if (!is_float_type(a->qkv_type) || !is_float_type(a->q_type))
    return fail(DMOE_ERR_UNSUPPORTED, "qkv and q_out are f32, f16 or bf16");
  if (a->rotary_dim < 0 || a->rotary_dim > hd || a->rotary_dim % 16)
    return fail(DMOE_ERR_UNSUPPORTED, "rotary_dim must be a multiple of 16 up to head_dim");
  if (a->rotary_dim > 0 && !(a->rope_base > 0.0 && a->rope_base < INFINITY))
    return fail(DMOE_ERR_INVALID_ARG, "rope_base must be positive");
  if (a->qkv_stride < (int64_t)(a->n_head + 2 * nk) * hd || a->q_stride < (int64_t)a->n_head * hd)
    return fail(DMOE_ERR_INVALID_ARG, "qkv_stride or q_stride is shorter than a row");
  if (a->n_tokens == 0 || batch->n_seq == 0) return DMOE_OK;
  if (!a->qkv || !a->q_out) return fail(DMOE_ERR_INVALID_ARG, "null pointer");
  if ((reinterpret_cast<uintptr_t>(a->qkv) % size_of(a->qkv_type)) | (reinterpret_cast<uintptr_t>(a->q_out) % size_of(a->q_type)))
    return fail(DMOE_ERR_INVALID_ARG, "qkv or q_out is not aligned to its elements");
  if ((reinterpret_cast<uintptr_t>(a->q_norm) | reinterpret_cast<uintptr_t>(a->k_norm)) & 15u)
    return fail(DMOE_ERR_INVALID_ARG, "q_norm and k_norm must be 16-byte aligned");

  const NvtxRange nvtx_call("dmoe_kv_append");
  AppendParams p{};
  p.pg = kv_pages(cache);
  p.b = kv_batch(batch, a->n_tokens);
  p.qkv = a->qkv;
  p.q_out = a->q_out;
  p.q_norm = a->q_norm;
  p.k_norm = a->k_norm;
  p.qkv_stride = a->qkv_stride;
  p.q_stride = a->q_stride;
  p.q_type = a->q_type;
  p.n_head = a->n_head;
  p.half = a->rotary_dim / 2;
  p.eps = a->eps;
  p.vec_in = aligned16(a->qkv, a->qkv_stride * size_of(a->qkv_type));
  p.vec_out = aligned16(a->q_out, a->q_stride * size_of(a->q_type));
  if (p.half > 0) {
    p.half_magic = ((1u << 18) + p.half - 1) / p.half;
    // base^(-2i / r) as powers of one ratio: 63 products of 64 bits stay within 1e-14 of the power
    const double ratio = pow(a->rope_base, -2.0 / a->rotary_dim);
    double t = 0.15915494309189533577;  // 1 / 2 pi
    for (int i = 0; i < p.half; ++i, t *= ratio) p.turns[i] = t;
  }
  const KvType kv = kv_type_of(cache->type);
  // a sequence of f rows touches at most f blocks, at most f / 32 + 2, and at most (f + 62) / 32
  const int64_t units = std::min<int64_t>({a->n_tokens, a->n_tokens / kScaleBlock + 2ll * batch->n_seq,
                                  ((int64_t)batch->max_q_len + 2 * kScaleBlock - 2) / kScaleBlock * batch->n_seq});
  if (units == 0) return DMOE_OK;
  const bool held = kv == KV_E4M3;
  p.flat_slots = a->n_head + (held ? 0 : 2 * nk);
  // Heads a CTA takes: as many as leave about kWanted CTAs (the rotation's table is then made for several heads; one
  // head each below that, where latency counts), but at least the 16 rows that the warps hold at once
  const int64_t fresh = std::max<int64_t>(1, std::min<int64_t>(kScaleBlock, a->n_tokens / std::max<int64_t>(1, units)));
  auto share = [&](int64_t heads, int64_t least, int64_t wanted) {
    const int64_t per = std::min<int64_t>(128, std::max((units * heads + wanted - 1) / wanted, least)), groups = (heads + per - 1) / per;
    return (int)((heads + groups - 1) / groups);  // even groups
  };
  p.flat_per_cta = share(p.flat_slots, std::min<int64_t>(p.flat_slots, (16 + fresh - 1) / fresh), kWanted);
  p.flat_groups = (p.flat_slots + p.flat_per_cta - 1) / p.flat_per_cta;
  p.held_per_cta = held ? share(nk, 1, kWantedHeld) : 1;
  p.held_groups = held ? (nk + p.held_per_cta - 1) / p.held_per_cta : 0;
  const dim3 grid((unsigned)units, (unsigned)(p.flat_groups + 2 * p.held_groups));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  set_pdl_for_call(true);
  cudaError_t e;
  if (a->qkv_type == DMOE_TYPE_F32)
    e = launch_append<DMOE_TYPE_F32>(p, hd, kv, grid, st);
  else if (a->qkv_type == DMOE_TYPE_F16)
    e = launch_append<DMOE_TYPE_F16>(p, hd, kv, grid, st);
  else
    e = launch_append<DMOE_TYPE_BF16>(p, hd, kv, grid, st);
  set_pdl_for_call(false);
  if (e != cudaSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "launch failed: %s", cudaGetErrorString(e));
    return fail(DMOE_ERR_CUDA, msg);
  }
  return DMOE_OK;
}
