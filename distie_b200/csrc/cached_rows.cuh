// What the kernels of an 8-bit cache and of drafted tokens share: the cache as they see it, the rows of a step, e4m3
// conversions.
//
// An 8-bit cache holds every key and value row (one token, one kv head) as e4m3 numbers n and one float32 scale s beside
// them, in arrays of the pages' shape: the row stands for n * s.  s is the row's largest magnitude over 448, the largest
// e4m3 number, so a row loses at most half an e4m3 step per element (2^-4 relative, 2^-10 s below 2^-6 s).  A row
// that held a number that is not finite has s = NaN and zeros, and reads back as NaN throughout.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

#define DISTIE_E4M3 2  // a cache's element type, beside DISTIE_F32 and DISTIE_BF16

namespace distie {

constexpr float kE4m3Most = 448.f;

// The pages of one cache slot: [num_pages, num_kv_heads, page_size, key_dim | value_dim] and, for e4m3, the rows' scales.
struct CachePages {
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
  const int* block_table;  // [seats, table_width]
  int table_width;
  int num_kv_heads;
  int key_dim, value_dim;
  int page_size;
  int page_shift;  // log2(page_size), or -1
  int num_pages;

  __device__ __forceinline__ int column_of(int key) const { return page_shift >= 0 ? key >> page_shift : key / page_size; }
  __device__ __forceinline__ int within(int key) const { return page_shift >= 0 ? key & (page_size - 1) : key % page_size; }
  // The row of `key` among all rows of the slot, or -1 when its page is missing.
  __device__ __forceinline__ long long row_of(const int* table, int key, int kv_head) const {
    const int column = column_of(key);
    const int page = column < table_width ? __ldg(table + column) : -1;
    if (page < 0 || page >= num_pages) return -1;
    return ((long long)page * num_kv_heads + kv_head) * page_size + within(key);
  }
};

__host__ inline CachePages make_pages(const void* k, const void* v, const float* k_scale, const float* v_scale, const int* block_table,
                                      int table_width, int num_kv_heads, int key_dim, int value_dim, int page_size, int num_pages) {
  CachePages c{k, v, k_scale, v_scale, block_table, table_width, num_kv_heads, key_dim, value_dim, page_size, -1, num_pages};
  if ((page_size & (page_size - 1)) == 0)
    for (c.page_shift = 0; (1 << c.page_shift) < page_size; ++c.page_shift) {
    }
  return c;
}

// The query rows of a step, request by request.  Request b has `nodes` new tokens, tokens first .. first + nodes - 1 of the
// step, whose keys and values stand behind its `past` cached ones (new token j at place past + j).  A new token sees the
// cached places that its window allows and new token j when bit j of its mask is set.  Tokens of no request are nobody's: nothing
// is written for them.  Without `seqs` every token is a request of its own: a single token behind positions[t] cached ones, which
// sees itself.
struct QueryRows {
  const int* positions;   // [tokens]
  const int* token_seq;   // [tokens]
  const int* seq_seat;    // [requests]
  const int* seqs;        // [requests, 3]: first, nodes, past; or null
  const int* bits;        // [tokens, words]
  int words;
  int tokens;             // of the step
  int requests;
  int most_nodes;         // new tokens of a request that the grid has tiles for
  int group;              // query heads per kv head
  int num_heads;
  int window, chunk, keep_first;
  float scale_log2;       // scale * log2(e)
  ScoreExtras extras;
};

struct Request {
  int first, nodes, past, seat;
};

__device__ __forceinline__ Request request_of(const QueryRows& rows, int b) {
  Request r;
  if (rows.seqs) {
    // (held to the step's tokens, the masks' words and the grid, whatever the rows say)
    r.first = min(max(rows.seqs[3 * b], 0), rows.tokens);
    r.nodes = min(min(max(rows.seqs[3 * b + 1], 0), min(rows.words * 32, rows.most_nodes)), rows.tokens - r.first);
    r.past = max(rows.seqs[3 * b + 2], 0);
    r.seat = rows.seq_seat[b];
  } else {
    r.first = b;
    r.nodes = 1;
    r.past = rows.positions[b];
    r.seat = rows.seq_seat[rows.token_seq[b]];
  }
  return r;
}

// Whether a token belongs to a request.
__device__ __forceinline__ bool token_is_somebodys(const QueryRows& rows, int token) {
  if (rows.seqs == nullptr) return true;
  const int b = rows.token_seq[token];
  if (b < 0 || b >= rows.requests) return false;
  const Request r = request_of(rows, b);
  return token >= r.first && token < r.first + r.nodes;
}

// Whether new token `node` of its request sees new token j (bit j of its mask).
__device__ __forceinline__ bool mask_bit(const QueryRows& rows, int token, int j) {
  return rows.seqs == nullptr || ((__ldg(rows.bits + (size_t)token * rows.words + (j >> 5)) >> (j & 31)) & 1);
}

__device__ __forceinline__ float score_log2(float dot, const QueryRows& rows) {
  return rows.extras.cap > 0.f ? 1.4426950408889634f * rows.extras.cap * tanhf(dot * rows.extras.cap_pre) : dot * rows.scale_log2;
}

// Two e4m3 numbers (the low 16 bits of x) as two float16, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t x) {
  uint32_t y;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(x));
  return y;
}
__device__ __forceinline__ void e4m3x4_to_float(uint32_t x, float (&out)[4]) {
  const uint32_t lo = e4m3x2_to_half2((uint16_t)(x & 0xffffu)), hi = e4m3x2_to_half2((uint16_t)(x >> 16));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
}
__device__ __forceinline__ float e4m3_to_float(uint8_t x) {
  const uint32_t h = e4m3x2_to_half2((uint16_t)x);
  return __half2float(__low2half(*reinterpret_cast<const __half2*>(&h)));
}

// An element as a float32 number (TYPE: its type), without its row's scale; through L2, for kernels that start early.
template <int TYPE>
__device__ __forceinline__ float value_cg(const void* rows, size_t at) {
  if (TYPE == DISTIE_E4M3) return e4m3_to_float(__ldcg(reinterpret_cast<const uint8_t*>(rows) + at));
  if (TYPE == DISTIE_BF16) return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(rows) + at) << 16);
  return __ldcg(reinterpret_cast<const float*>(rows) + at);
}

// The partial results of split key ranges: scratch holds o [tokens * heads * splits, value_dim] and behind it (maximum in
// base-2 units, sum) pairs.
struct Partials {
  float* o;
  float* ml;
  int splits;
};

// Joins the parts of every (token, head) into 16-bit rows (attention_rows.cu).
int rows_merge_bf16(const Partials& parts, const QueryRows& rows, void* out, int out_stride, int value_dim, cudaStream_t stream);

}  // namespace distie
