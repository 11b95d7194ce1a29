// kv_common.cuh — what the paged key/value cache's two kernels share: the parameter blocks, the
// checks of a sequence's entry in the device tables, conversions between the element types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "../../include/diffuse_moe.h"

namespace dmoe {

constexpr int kScaleBlock = DMOE_KV_SCALE_BLOCK;  // positions that share a scale
constexpr int kExpMin = -60, kExpMax = 120;       // exponents of a scale

enum KvType : int { KV_BF16 = 0, KV_F16 = 1, KV_E4M3 = 2 };

struct KvPages {
  void* k;
  void* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  uint32_t* err;
  int64_t n_pages;
  int n_head_kv, page_size;
  int page_blocks;       // page_size / 32
  uint64_t page_magic;   // ceil(2^36 / page_blocks)
};

// Page slot of 32-position block b, b < 2^25 (positions are below 2^30): b / page_blocks, exactly, since
// page_blocks <= 2^11 and b * (page_magic * page_blocks - 2^36) < 2^36.
__device__ __forceinline__ uint32_t kv_slot(const KvPages& pg, uint32_t b) {
  return (uint32_t)((b * pg.page_magic) >> 36);
}

struct KvBatch {
  const int32_t* table;
  const int32_t* q_start;
  const int32_t* kv_len;
  int64_t max_pages, n_tokens;
  int n_seq, max_q_len;
};

struct KvSeq {
  int row0, q_len, kv_len;
};

__device__ __forceinline__ void kv_report(uint32_t* err, uint32_t bit) {
  if (err) atomicOr(err, bit);
}

// Sequence s of the batch; an entry that breaks the batch's rules is reported and owns no rows.
__device__ __forceinline__ KvSeq kv_sequence(const KvBatch& b, const KvPages& pg, int s) {
  KvSeq q;
  q.row0 = b.q_start[s];
  const int end = b.q_start[s + 1];
  q.kv_len = b.kv_len[s];
  q.q_len = end - q.row0;
  if (q.row0 < 0 || end < q.row0 || end > b.n_tokens || q.kv_len < 0 || q.kv_len > b.max_pages * pg.page_size ||
      q.q_len > b.max_q_len) {
    kv_report(pg.err, DMOE_KV_ERR_BATCH);
    q.q_len = 0;
  }
  return q;
}

// First element of (page, head, offset) in the pages.
__device__ __forceinline__ int64_t kv_row(const KvPages& pg, int64_t page, int head, int offset) {
  return (page * pg.n_head_kv + head) * pg.page_size + offset;
}

// Host-side checks that both entry points make; returns DMOE_OK or sets the error message.
dmoe_status kv_check(const char* call, const dmoe_kv_cache* c, const dmoe_kv_batch* b, int64_t n_tokens, int n_head);
inline KvType kv_type_of(int type) {
  return type == DMOE_TYPE_BF16 ? KV_BF16 : type == DMOE_TYPE_F16 ? KV_F16 : KV_E4M3;
}
inline KvPages kv_pages(const dmoe_kv_cache* c) {
  const uint64_t blocks = (uint64_t)c->page_size / kScaleBlock;
  return {c->k, c->v, c->k_scale, c->v_scale, c->err, c->n_pages, c->n_head_kv, c->page_size, (int)blocks,
          ((uint64_t{1} << 36) + blocks - 1) / blocks};
}
inline KvBatch kv_batch(const dmoe_kv_batch* b, int64_t n_tokens) {
  return {b->page_table, b->q_start, b->kv_len, b->max_pages, n_tokens, b->n_seq, b->max_q_len};
}

}  // namespace dmoe
