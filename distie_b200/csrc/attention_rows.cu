// Attention of few query rows per request over the paged cache, for any sizes and types: single tokens over an 8-bit cache,
// trees of drafted tokens over a cache in 8, 16 or 32 bits.  Float32 arithmetic throughout.
//
// The rows of a request that share a kv head, (new token, query head of the group), are packed: row r is head r % group of
// new token r / group.  A block takes up to 16 rows and walks its share of the keys in tiles of 32: keys and values come
// into shared memory as float32 once for all rows, a thread makes the scores of one key with four rows, a warp the softmax
// statistics of four rows (running maximum and sum), a thread the output columns of all rows.  With few rows the reads
// of the cache bound it; keys are then split over blocks and the parts merged.
#include <cuda_fp16.h>

#include "cached_rows.cuh"
#include "packed.h"

namespace distie {

constexpr int kRowsTile = 16;
constexpr int kRowsKeys = 32;
constexpr int kRowsThreads = 128;
constexpr int kRowsMostDim = 256;

template <typename T, int CACHE>
__global__ void __launch_bounds__(kRowsThreads)
attention_rows_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, int out_stride, QueryRows rows, CachePages cache,
                      Partials parts, int* __restrict__ error) {
  extern __shared__ __align__(16) float dyn[];
  const int dim = cache.key_dim, vdim = cache.value_dim;
  float* q_s = dyn;                                 // [16][dim]
  float* k_s = q_s + kRowsTile * dim;               // [32][dim + 1]
  float* v_s = k_s + kRowsKeys * (dim + 1);         // [32][vdim]
  __shared__ float p_s[kRowsKeys][kRowsTile + 4];   // weights, a key's rows side by side
  __shared__ float corr_s[kRowsTile], m_s[kRowsTile], l_s[kRowsTile];
  __shared__ int bad_s;                             // a value of this tile is not finite
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y, split = blockIdx.z;
  const Request request = request_of(rows, b);
  const int kv_head = blockIdx.x % cache.num_kv_heads, tile = blockIdx.x / cache.num_kv_heads;
  const int row0 = tile * kRowsTile, all_rows = request.nodes * rows.group;
  if (row0 >= all_rows) return;
  const int count = min(kRowsTile, all_rows - row0);
  const int* table = cache.block_table + (size_t)request.seat * cache.table_width;

  for (int i = threadIdx.x; i < kRowsTile * dim; i += kRowsThreads) {
    const int r = i / dim, e = i % dim;
    float x = 0.f;
    if (r < count) {
      const int token = request.first + (row0 + r) / rows.group, head = kv_head * rows.group + (row0 + r) % rows.group;
      x = to_float(q[(size_t)token * q_stride + (size_t)head * dim + e]);
    }
    q_s[i] = x;
  }
  if (threadIdx.x < kRowsTile) {
    m_s[threadIdx.x] = -INFINITY;
    l_s[threadIdx.x] = 0.f;
  }
  // The oldest cached key that any row of the tile sees inside its window (all new tokens' keys are walked); the keys
  // before it are walked up to keep_first only.
  int oldest = request.past;
  for (int r = 0; r < count; ++r)
    oldest = min(oldest, first_visible_key(rows.positions[request.first + (row0 + r) / rows.group], rows.window, rows.chunk));
  const int keys = request.past + request.nodes;
  const int kept = min(rows.keep_first, oldest);
  // Tiles of keys: those of the kept first keys, then those from the oldest one on; the splits share them out.
  const int kept_tiles = (kept + kRowsKeys - 1) / kRowsKeys;
  const int start = min(oldest, keys) / kRowsKeys * kRowsKeys;
  const int tiles = kept_tiles + (keys - start + kRowsKeys - 1) / kRowsKeys;
  const int share = (tiles + parts.splits - 1) / parts.splits;
  const int tile_end = min(tiles, (split + 1) * share);

  float acc[kRowsTile][2];
#pragma unroll
  for (int r = 0; r < kRowsTile; ++r) acc[r][0] = acc[r][1] = 0.f;

  for (int j = split * share; j < tile_end; ++j) {
    const int key0 = j < kept_tiles ? j * kRowsKeys : start + (j - kept_tiles) * kRowsKeys;
    // A key of the kept tiles that the window's tiles hold too is left to those.
    const int key_end = j < kept_tiles ? min(kept, start) : keys;
    __syncthreads();  // the tile before this one is done with
    if (threadIdx.x == 0) bad_s = 0;
    __syncthreads();
    for (int r = warp; r < kRowsKeys; r += kRowsThreads / 32) {
      const int key = key0 + r;
      long long at = -1;
      if (key < key_end && (key >= oldest || key < kept)) {
        at = cache.row_of(table, key, kv_head);
        if (at < 0 && lane == 0 && error) atomicExch(error, rows.seqs ? 8 : 4);
      }
      const float ks = CACHE == DISTIE_E4M3 && at >= 0 ? cache.k_scale[at] : 1.f, vs = CACHE == DISTIE_E4M3 && at >= 0 ? cache.v_scale[at] : 1.f;
      for (int e = lane; e < dim; e += 32) k_s[r * (dim + 1) + e] = at >= 0 ? cached_value<CACHE>(cache.k, (size_t)at * dim + e) * ks : 0.f;
      bool bad = false;
      for (int e = lane; e < vdim; e += 32) {
        const float x = at >= 0 ? cached_value<CACHE>(cache.v, (size_t)at * vdim + e) * vs : 0.f;
        bad |= !(fabsf(x) <= 3.402823466e38f);
        v_s[r * vdim + e] = x;
      }
      if (bad) bad_s = 1;
    }
    __syncthreads();
    {  // scores: key `lane`, rows 4 warp .. 4 warp + 3; then their softmax statistics over the warp
      const int key = key0 + lane;
      float dot[4] = {0.f, 0.f, 0.f, 0.f};
      const float* k_row = k_s + lane * (dim + 1);
      const float* q_row = q_s + warp * 4 * dim;
      for (int e = 0; e < dim; ++e) {
        const float x = k_row[e];
#pragma unroll
        for (int u = 0; u < 4; ++u) dot[u] += x * q_row[u * dim + e];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = warp * 4 + u;
        bool seen = r < count && key < key_end;
        if (seen) {
          const int token = request.first + (row0 + r) / rows.group;
          const int first = first_visible_key(rows.positions[token], rows.window, rows.chunk);
          int key_position = key;
          if (key >= request.past) {
            seen = mask_bit(rows, token, key - request.past);
            key_position = rows.positions[request.first + key - request.past];
          }
          seen = seen && (key_position >= first || key_position < rows.keep_first) && cache.row_of(table, key, kv_head) >= 0;
        }
        const float x = seen ? score_log2(dot[u], rows) : -INFINITY;
        const float m_old = m_s[r];
        const float m_new = fmaxf(m_old, warp_max(x));
        const float p = x == -INFINITY ? 0.f : exp2f(x - m_new);
        const float corr = m_old == -INFINITY ? 0.f : exp2f(m_old - m_new);
        const float sum = warp_sum(p);
        p_s[lane][r] = p;
        __syncwarp();
        if (lane == 0) {
          l_s[r] = l_s[r] * corr + sum;
          m_s[r] = m_new;
          corr_s[r] = corr;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = threadIdx.x + i * kRowsThreads;
      if (e < vdim) {
#pragma unroll
        for (int r = 0; r < kRowsTile; ++r) acc[r][i] *= corr_s[r];
        if (!bad_s) {
          for (int key = 0; key < kRowsKeys; ++key) {
            const float v = v_s[key * vdim + e];
#pragma unroll
            for (int r = 0; r < kRowsTile; r += 4) {
              const float4 p = *reinterpret_cast<const float4*>(&p_s[key][r]);
              acc[r][i] += p.x * v;
              acc[r + 1][i] += p.y * v;
              acc[r + 2][i] += p.z * v;
              acc[r + 3][i] += p.w * v;
            }
          }
        } else {  // 0 * NaN is not 0: a value that is not finite reaches the rows that see it alone
          for (int key = 0; key < kRowsKeys; ++key) {
            const float v = v_s[key * vdim + e];
#pragma unroll
            for (int r = 0; r < kRowsTile; ++r) acc[r][i] += p_s[key][r] != 0.f ? p_s[key][r] * v : 0.f;
          }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = threadIdx.x + i * kRowsThreads;
    if (e >= vdim) continue;
#pragma unroll
    for (int r = 0; r < kRowsTile; ++r) {
      if (r >= count) break;
      const int token = request.first + (row0 + r) / rows.group, head = kv_head * rows.group + (row0 + r) % rows.group;
      if (parts.splits == 1) {
        const float inv = rows.extras.sink ? sink_inverse_log2(m_s[r], l_s[r], rows.extras.sink[head]) : (l_s[r] == 0.f ? 0.f : 1.f / l_s[r]);
        out[(size_t)token * out_stride + (size_t)head * vdim + e] = from_float<T>(acc[r][i] * inv);
      } else {
        const size_t row = ((size_t)token * rows.num_heads + head) * parts.splits + split;
        parts.o[row * vdim + e] = acc[r][i];
        if (e == 0) {
          parts.ml[row * 2] = m_s[r];
          parts.ml[row * 2 + 1] = l_s[r];
        }
      }
    }
  }
}

// Joins the parts of a (token, head): a block each.  A row of parts takes a group of threads, four columns a thread, and
// the groups share out the splits, so that the loads of many of them are in flight together; the order of the additions
// follows from the number of splits alone.
constexpr int kMergeThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kMergeThreads)
attention_rows_merge_kernel(Partials parts, T* __restrict__ out, int out_stride, int value_dim, const float* __restrict__ sink) {
  __shared__ float sh_acc[kMergeThreads][4];
  __shared__ float sh_l[kMergeThreads];
  __shared__ float sh_max[kMergeThreads / 32];
  grid_dependency_release();
  grid_dependency_wait();
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row0 = ((size_t)token * gridDim.y + head) * parts.splits;
  const int per_row = (value_dim + 3) / 4, groups = kMergeThreads / per_row;  // up to 64 threads, at least 4 groups
  const int mine = threadIdx.x / per_row, column = threadIdx.x % per_row * 4;
  float m_all = -INFINITY;
  for (int s = threadIdx.x; s < parts.splits; s += kMergeThreads) m_all = fmaxf(m_all, __ldcg(parts.ml + (row0 + s) * 2));
  m_all = warp_max(m_all);
  if (lane == 0) sh_max[warp] = m_all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeThreads / 32; ++w) m_all = fmaxf(m_all, sh_max[w]);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, l_mine = 0.f;
  if (mine < groups) {
#pragma unroll 4
    for (int s = mine; s < parts.splits; s += groups) {
      const float m = __ldcg(parts.ml + (row0 + s) * 2), l = __ldcg(parts.ml + (row0 + s) * 2 + 1);
      // (a part without a key has a sum of 0, one whose scores are all NaN a sum of NaN; both have no maximum)
      const float weight = m == -INFINITY ? l : exp2f(m - m_all);
      l_mine += l * weight;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (column + e < value_dim) acc[e] += __ldcg(parts.o + (row0 + s) * value_dim + column + e) * weight;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sh_acc[threadIdx.x][e] = acc[e];
  if (column == 0) sh_l[mine] = l_mine;
  __syncthreads();
  if (threadIdx.x < per_row) {
    float l_all = 0.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < groups; ++r) {
      l_all += sh_l[r];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += sh_acc[r * per_row + threadIdx.x][e];
    }
    const float inv = sink ? sink_inverse_log2(m_all, l_all, sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (column + e < value_dim) out[(size_t)token * out_stride + (size_t)head * value_dim + column + e] = from_float<T>(sum[e] * inv);
  }
}

template <typename T>
static int rows_merge(const Partials& parts, void* out, int out_stride, int tokens, int num_heads, int value_dim, const float* sink,
                      cudaStream_t stream) {
  return (int)launch_dependent(attention_rows_merge_kernel<T>, dim3(tokens, num_heads), dim3(kMergeThreads), 0, stream, parts, (T*)out, out_stride,
                               value_dim, sink);
}

int rows_merge_bf16(const Partials& parts, void* out, int out_stride, int tokens, int num_heads, int value_dim, const float* sink,
                    cudaStream_t stream) {
  return rows_merge<__nv_bfloat16>(parts, out, out_stride, tokens, num_heads, value_dim, sink, stream);
}

}  // namespace distie

using namespace distie;

extern "C" long long distie_attention_rows_scratch_floats(int tokens, int num_heads, int value_dim, int splits) {
  return splits > 1 ? (long long)tokens * num_heads * splits * (value_dim + 2) : 0;
}

// q [tokens, >= heads * key_dim], out [tokens, heads * value_dim] of type `dtype`; seqs null: single tokens, `requests` of
// them, else [requests, 3] with at most most_nodes new tokens each.  scratch: distie_attention_rows_scratch_floats.
extern "C" int distie_attention_rows(const void* q, int q_stride, void* out, int out_stride, float* scratch, const int* positions,
                                     const int* token_seq, const int* seq_seat, const int* seqs, const int* bits, int words,
                                     int requests, int tokens, int most_nodes, const void* k_cache, const void* v_cache,
                                     const float* k_scale, const float* v_scale, const int* block_table, int table_width, int num_heads,
                                     int num_kv_heads, int key_dim, int value_dim, int page_size, int num_pages, int window, int chunk,
                                     int keep_first, float scale, float softcap, const float* sink, int splits, int dtype, int cache_type,
                                     int* error, cudaStream_t stream) {
  if (tokens <= 0 || requests <= 0) return 0;
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads != 0 || key_dim < 1 || key_dim > kRowsMostDim || value_dim < 1 ||
      value_dim > kRowsMostDim || page_size < 1 || table_width < 1 || most_nodes < 1 || words < 1 || keep_first < 0 || splits < 1 ||
      splits > 65535 || requests > 65535 || num_heads > 65535 || (splits > 1 && scratch == nullptr) || (seqs != nullptr && bits == nullptr) ||
      (cache_type == DISTIE_E4M3 && (k_scale == nullptr || v_scale == nullptr)))
    return DISTIE_ERR_ARG;
  const CachePages cache = make_pages(k_cache, v_cache, k_scale, v_scale, block_table, table_width, num_kv_heads, key_dim, value_dim,
                                      page_size, num_pages);
  const QueryRows rows{positions, token_seq, seq_seat, seqs, bits, words, tokens, num_heads / num_kv_heads, num_heads, window, chunk, keep_first,
                       scale * 1.4426950408889634f, make_score_extras(scale, softcap, sink)};
  const Partials parts{scratch, scratch ? scratch + (size_t)tokens * num_heads * splits * value_dim : nullptr, splits};
  const int tiles = (most_nodes * rows.group + kRowsTile - 1) / kRowsTile;
  const dim3 grid(tiles * num_kv_heads, requests, splits);
  const size_t shared = ((size_t)kRowsTile * key_dim + (size_t)kRowsKeys * (key_dim + 1 + value_dim)) * sizeof(float);
  cudaError_t err;
#define DISTIE_ROWS(T, CACHE)                                                                                                       \
  {                                                                                                                                 \
    if (shared > 48 * 1024 && (err = cudaFuncSetAttribute(attention_rows_kernel<T, CACHE>,                                           \
                                                          cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024)) != cudaSuccess)  \
      return (int)err;                                                                                        \
    attention_rows_kernel<T, CACHE><<<grid, kRowsThreads, shared, stream>>>((const T*)q, q_stride, (T*)out, out_stride, rows, cache,   \
                                                                            parts, error);                                          \
    DISTIE_LAUNCH_CHECK();                                                                                                          \
    if (splits > 1) return rows_merge<T>(parts, out, out_stride, tokens, num_heads, value_dim, sink, stream);                          \
    return 0;                                                                                                                       \
  }
  if (dtype == DISTIE_BF16 && cache_type == DISTIE_E4M3) DISTIE_ROWS(__nv_bfloat16, DISTIE_E4M3)
  if (dtype == DISTIE_BF16 && cache_type == DISTIE_BF16) DISTIE_ROWS(__nv_bfloat16, DISTIE_BF16)
  if (dtype == DISTIE_F32 && cache_type == DISTIE_E4M3) DISTIE_ROWS(float, DISTIE_E4M3)
  if (dtype == DISTIE_F32 && cache_type == DISTIE_F32) DISTIE_ROWS(float, DISTIE_F32)
#undef DISTIE_ROWS
  return DISTIE_ERR_UNSUPPORTED;
}

DISTIE_PACKED(distie_attention_rows)
