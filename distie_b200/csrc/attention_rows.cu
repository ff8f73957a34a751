// Attention of few query rows per request over the paged cache, for any sizes and types: single tokens over an 8-bit cache,
// trees of drafted tokens over a cache in 8, 16 or 32 bits.  Float32 arithmetic throughout.
//
// The rows of a request that share a kv head, (new token, query head of the group), are packed: row r is head r % group of
// new token r / group.  A block takes up to 16 rows and walks its share of the keys in tiles of 32: keys and values come
// into shared memory as float32 once for all rows, a thread makes the scores of one key with four rows, a warp the softmax
// statistics of four rows (running maximum and sum), a thread a column of the sums of 4, 8 or 16 rows, so that all threads have
// one.  Keys are split over blocks (rows_splits in kernels/cached.py) and the parts joined.
//
// What bounds it is latency: a block alone takes about 5,000 cycles a tile of 32 keys (its rows found 600, their loads 2,000,
// scores 800, weights 1,200, sums 600; 8,000 before loads, reductions and sums were laid side by side).  So registers go to loads
// in flight, two blocks an SM.  Two trees of 13 new tokens over 500 keys, 80 tiles of rows, heads of 32 in float32: 23 us with
// the joining kernel; over 5,000 keys 119.
#include <cuda_fp16.h>

#include "cached_rows.cuh"
#include "packed.h"

namespace distie {

constexpr int kRowsTile = 16;
constexpr int kRowsKeys = 32;
constexpr int kRowsThreads = 128;
constexpr int kRowsPitch = kRowsTile + 4;  // of a key's weights in shared memory
constexpr int kRowsMostDim = 256;

__host__ __device__ constexpr int rows_k_pitch(int dim) { return dim % 4 == 0 ? dim + 4 : dim + 1; }

// The sums of a column of values of ROWS rows (acc[..][i]), scaled down by `corr`, and a tile's weights times values joined to them.
template <int ROWS>
__device__ __forceinline__ void add_values(float (&acc)[kRowsTile][2], int i, const float* corr, const float* weights, const float* values,
                                           int vdim, int bad) {
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r][i] *= corr[r];
  if (!bad) {
#pragma unroll 8
    for (int j = 0; j < kRowsKeys; ++j) {
      const float v = values[j * vdim];
#pragma unroll
      for (int r = 0; r < ROWS; r += 4) {
        const float4 w = *reinterpret_cast<const float4*>(weights + j * kRowsPitch + r);
        acc[r][i] += w.x * v;
        acc[r + 1][i] += w.y * v;
        acc[r + 2][i] += w.z * v;
        acc[r + 3][i] += w.w * v;
      }
    }
  } else {  // 0 * NaN is not 0: a value that is not finite reaches the rows that see it (their weights are above 0), and no others
    for (int j = 0; j < kRowsKeys; ++j) {
      const float v = values[j * vdim];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float w = weights[j * kRowsPitch + r];
        acc[r][i] += w != 0.f ? w * v : 0.f;
      }
    }
  }
}

template <typename T, int CACHE>
__global__ void __launch_bounds__(kRowsThreads, 2)
attention_rows_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, int out_stride, QueryRows rows, CachePages cache,
                      Partials parts, int* __restrict__ error) {
  extern __shared__ __align__(16) float dyn[];
  const int dim = cache.key_dim, vdim = cache.value_dim;
  float* q_s = dyn;                                 // [16][dim]
  const int k_pitch = rows_k_pitch(dim);            // (free of bank conflicts, by one element or by four a lane)
  float* k_s = q_s + kRowsTile * dim;               // [32][k_pitch]
  float* v_s = k_s + kRowsKeys * k_pitch;           // [32][vdim]
  __shared__ alignas(16) float p_s[kRowsKeys][kRowsPitch];   // weights, a key's rows side by side
  __shared__ float corr_s[kRowsTile], m_s[kRowsTile], l_s[kRowsTile];
  __shared__ int bad_s;                             // a value of this tile is not finite
  __shared__ int first_s[kRowsTile], token_s[kRowsTile], head_s[kRowsTile];  // a row's oldest visible key, its token and head
  grid_dependency_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y, split = blockIdx.z;
  const Request request = request_of(rows, b);
  const int kv_head = blockIdx.x % cache.num_kv_heads, tile = blockIdx.x / cache.num_kv_heads;
  const int row0 = tile * kRowsTile, all_rows = request.nodes * rows.group;
  if (row0 >= all_rows) {
    if (blockIdx.x == 0 && b == 0 && split == 0) grid_dependency_wait();  // (some block of the grid always waits: kernels end in order)
    return;
  }
  const int count = min(kRowsTile, all_rows - row0);
  const int* table = cache.block_table + (size_t)request.seat * cache.table_width;

  if (threadIdx.x < kRowsTile) {  // (rows behind the last one are nobody's: copies of it, never written)
    const int row = row0 + min((int)threadIdx.x, count - 1), node = row / rows.group, token = request.first + node;
    token_s[threadIdx.x] = token;
    head_s[threadIdx.x] = kv_head * rows.group + row - node * rows.group;
    first_s[threadIdx.x] = first_visible_key(rows.positions[token], rows.window, rows.chunk);
  }
  __syncthreads();
  grid_dependency_wait();  // q and the newest rows come from the kernels before this one
  for (int e = lane; e < dim; e += 32)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = warp * 4 + u;
      q_s[r * dim + e] = value_cg<sizeof(T) == 4 ? DISTIE_F32 : DISTIE_BF16>(q, (size_t)token_s[r] * q_stride + (size_t)head_s[r] * dim + e);
    }
  // The oldest cached key that any row of the tile sees inside its window (all new tokens' keys are walked); the keys
  // before it are walked up to keep_first only.
  int oldest = request.past;
  for (int r = 0; r < count; ++r) oldest = min(oldest, first_s[r]);
  const int keys = request.past + request.nodes;
  const int kept = min(rows.keep_first, oldest);
  // Tiles of keys: those of the kept first keys, then those from the oldest one on; the splits share them out.
  const int kept_tiles = (kept + kRowsKeys - 1) / kRowsKeys;
  const int start = min(oldest, keys) / kRowsKeys * kRowsKeys;
  const int tiles = kept_tiles + (keys - start + kRowsKeys - 1) / kRowsKeys;
  const int share = (tiles + parts.splits - 1) / parts.splits;
  const int tile_end = min(tiles, (split + 1) * share);

  // A warp keeps the maxima and sums of its four rows; of the sums of values a thread keeps a column of all 16 rows (two of
  // values beyond 128), of 8 with up to 64 columns, of 4 with up to 32.
  float m_mine[4], l_mine[4], acc[kRowsTile][2];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    m_mine[u] = -INFINITY;
    l_mine[u] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < kRowsTile; ++r) acc[r][0] = acc[r][1] = 0.f;
  const int row_parts = vdim <= 32 ? 4 : vdim <= 64 ? 2 : 1, part_rows = kRowsTile / row_parts, part_threads = kRowsThreads / row_parts;
  const int column = threadIdx.x & (part_threads - 1), row_first = threadIdx.x / part_threads * part_rows;

  for (int j = split * share; j < tile_end; ++j) {
    const int key0 = j < kept_tiles ? j * kRowsKeys : start + (j - kept_tiles) * kRowsKeys;
    // A key of the kept tiles that the window's tiles hold too is left to those.
    const int key_end = j < kept_tiles ? min(kept, start) : keys;
    __syncthreads();  // the tile before this one is done with
    if (threadIdx.x == 0) bad_s = 0;
    __syncthreads();
    // Lane r of every warp finds key r's row; a warp then takes 8 rows, all their loads together (of no row: the cache's first,
    // not used).
    const int key = key0 + lane;
    long long at = -1;
    if (key < key_end && (key >= oldest || key < kept)) {
      at = cache.row_of(table, key, kv_head);
      if (at < 0 && warp == 0 && error) atomicExch(error, rows.seqs ? 8 : 4);
    }
    int key_position = key;
    if (rows.seqs && key >= request.past && key < keys) key_position = rows.positions[request.first + key - request.past];
    float k_scale = 1.f, v_scale = 1.f;
    if (CACHE == DISTIE_E4M3) {
      k_scale = __ldcg(cache.k_scale + max(at, 0ll));
      v_scale = __ldcg(cache.v_scale + max(at, 0ll));
    }
    constexpr int MINE = kRowsKeys / (kRowsThreads / 32);
    const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
    uint32_t from[MINE];  // (a cache has fewer than 2^32 rows)
    float ks[MINE], vs[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      from[i] = __shfl_sync(0xffffffffu, (uint32_t)max(at, 0ll), warp * MINE + i);
      ks[i] = __shfl_sync(0xffffffffu, k_scale, warp * MINE + i);
      vs[i] = __shfl_sync(0xffffffffu, v_scale, warp * MINE + i);
    }
    bool bad = false;
    for (int e = lane; e < max(dim, vdim); e += 32) {
      float kx[MINE], vx[MINE];
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        kx[i] = value_cg<CACHE>(cache.k, (size_t)from[i] * (uint32_t)dim + min(e, dim - 1));
        vx[i] = value_cg<CACHE>(cache.v, (size_t)from[i] * (uint32_t)vdim + min(e, vdim - 1));
      }
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int r = warp * MINE + i;
        const bool live = (there >> r) & 1;
        if (e < dim) k_s[r * k_pitch + e] = live ? kx[i] * ks[i] : 0.f;
        if (e < vdim) {
          const float x = live ? vx[i] * vs[i] : 0.f;
          bad |= !(fabsf(x) <= 3.402823466e38f);
          v_s[r * vdim + e] = x;
        }
      }
    }
    if (bad) bad_s = 1;
    __syncthreads();
    {  // scores: key `lane`, rows 4 warp .. 4 warp + 3; then their softmax statistics over the warp
      float dot[4] = {0.f, 0.f, 0.f, 0.f};
      const float* k_row = k_s + lane * k_pitch;
      const float* q_row = q_s + warp * 4 * dim;
      if (dim % 4 == 0) {
#pragma unroll 4
        for (int e = 0; e < dim; e += 4) {
          const float4 x = *reinterpret_cast<const float4*>(k_row + e);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float4 y = *reinterpret_cast<const float4*>(q_row + u * dim + e);
            dot[u] += x.x * y.x;
            dot[u] += x.y * y.y;
            dot[u] += x.z * y.z;
            dot[u] += x.w * y.w;
          }
        }
      } else {
        for (int e = 0; e < dim; ++e) {
          const float x = k_row[e];
#pragma unroll
          for (int u = 0; u < 4; ++u) dot[u] += x * q_row[u * dim + e];
        }
      }
      float x[4], most[4], p[4], sum[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = warp * 4 + u;
        bool seen = r < count && at >= 0 && (key_position >= first_s[r] || key_position < rows.keep_first);
        if (seen && key >= request.past) seen = mask_bit(rows, token_s[r], key - request.past);
        x[u] = most[u] = seen ? score_log2(dot[u], rows) : -INFINITY;
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1)  // (the four rows' chains side by side)
#pragma unroll
        for (int u = 0; u < 4; ++u) most[u] = fmaxf(most[u], __shfl_xor_sync(0xffffffffu, most[u], d));
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float m_old = m_mine[u], m_new = fmaxf(m_old, most[u]), corr = m_old == -INFINITY ? 0.f : exp2f(m_old - m_new);
        p[u] = x[u] == -INFINITY ? 0.f : exp2f(x[u] - m_new);
        if (bad_s && p[u] == 0.f && x[u] != -INFINITY) p[u] = 1.4e-45f;  // (the smallest number: whoever sees a value that is not finite gets it)
        sum[u] = p[u];
        m_mine[u] = m_new;
        l_mine[u] *= corr;
        if (lane == 0) corr_s[warp * 4 + u] = corr;
      }
      *reinterpret_cast<float4*>(&p_s[lane][warp * 4]) = make_float4(p[0], p[1], p[2], p[3]);
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1)
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], d);
#pragma unroll
      for (int u = 0; u < 4; ++u) l_mine[u] += sum[u];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = column + i * kRowsThreads;
      if (e < vdim) {
        const float* weights = &p_s[0][row_first];
        if (part_rows == 4) add_values<4>(acc, i, corr_s + row_first, weights, v_s + e, vdim, bad_s);
        else if (part_rows == 8) add_values<8>(acc, i, corr_s + row_first, weights, v_s + e, vdim, bad_s);
        else add_values<16>(acc, i, corr_s + row_first, weights, v_s + e, vdim, bad_s);
      }
    }
  }
  if (lane < 4) {
    m_s[warp * 4 + lane] = lane == 0 ? m_mine[0] : lane == 1 ? m_mine[1] : lane == 2 ? m_mine[2] : m_mine[3];
    l_s[warp * 4 + lane] = lane == 0 ? l_mine[0] : lane == 1 ? l_mine[1] : lane == 2 ? l_mine[2] : l_mine[3];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = column + i * kRowsThreads;
    if (e >= vdim) continue;
#pragma unroll
    for (int x = 0; x < kRowsTile; ++x) {
      const int r = row_first + x;
      if (x >= part_rows || r >= count) break;
      const int token = token_s[r], head = head_s[r];
      if (parts.splits == 1) {
        const float inv = rows.extras.sink ? sink_inverse_log2(m_s[r], l_s[r], rows.extras.sink[head]) : (l_s[r] == 0.f ? 0.f : 1.f / l_s[r]);
        out[(size_t)token * out_stride + (size_t)head * vdim + e] = from_float<T>(acc[x][i] * inv);
      } else {
        const size_t row = ((size_t)token * rows.num_heads + head) * parts.splits + split;
        parts.o[row * vdim + e] = acc[x][i];
        if (e == 0) {
          parts.ml[row * 2] = m_s[r];
          parts.ml[row * 2 + 1] = l_s[r];
        }
      }
    }
  }
}

// Joins the parts of (token, head) rows, SHARE warps a row.  Lane s looks at part s (and s + 32, ...): its maximum, its sum, and
// with the row's maximum what it counts, so that the loads of the parts wait for nothing but their addresses; a lane owns four
// columns (and, of more than 128, four more), and parts of up to 64 columns go to the halves (quarters, ...) of the warp in
// turn.  The order of the additions follows from the numbers of splits and rows alone.  SHARE 4 where a row has more than 16
// parts, or more than 4 and the rows are few: one warp would ask for them in several turns.  (A block a row, with barriers between its warps, cost two trees of 64
// tokens of 40 heads, 5,120 rows of 3 parts, 6 us more, and eight of 26 over an 8-bit cache 5.)
constexpr int kMergeThreads = 128;

template <typename T, int SHARE>
__global__ void __launch_bounds__(kMergeThreads)
attention_rows_merge_kernel(Partials parts, QueryRows rows, T* __restrict__ out, int out_stride, int num_rows, int value_dim) {
  constexpr int ROWS = kMergeThreads / 32 / SHARE, PASSES = kRowsMostDim / 128;
  __shared__ float sh_acc[SHARE][PASSES * 128 + 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % SHARE;
  const int row = blockIdx.x * ROWS + warp / SHARE;
  grid_dependency_release();
  if (SHARE == 1 && row >= num_rows) return;
  int across = 1;  // lanes that a part's row takes
  while (across < 32 && across * 4 < value_dim) across *= 2;
  const int groups = 32 / across, mine = lane / across, column = lane % across * 4;
  const bool whole = value_dim % 4 == 0;
  const size_t part0 = (size_t)row * parts.splits;
  const int token = row / rows.num_heads, head = row % rows.num_heads;
  const bool somebodys = token_is_somebodys(rows, token);
  grid_dependency_wait();
  if (!somebodys) return;  // (a block's warps that meet at a barrier share their row)
  // A part without a key has a sum of 0, one whose scores are all NaN a sum of NaN; both have no maximum.
  float m_mine = lane < parts.splits ? __ldcg(parts.ml + (part0 + lane) * 2) : -INFINITY, l_mine = lane < parts.splits ? __ldcg(parts.ml + (part0 + lane) * 2 + 1) : 0.f;
  float m_all = m_mine;
  for (int s = lane + 32; s < parts.splits; s += 32) m_all = fmaxf(m_all, __ldcg(parts.ml + (part0 + s) * 2));
  m_all = warp_max(m_all);
  float l_all = 0.f, acc[PASSES][4] = {};
  for (int base = 0; base < parts.splits; base += 32) {
    if (base > 0) {
      m_mine = lane < parts.splits - base ? __ldcg(parts.ml + (part0 + base + lane) * 2) : -INFINITY;
      l_mine = lane < parts.splits - base ? __ldcg(parts.ml + (part0 + base + lane) * 2 + 1) : 0.f;
    }
    const float weight = m_mine == -INFINITY ? l_mine : exp2f(m_mine - m_all);
    l_all += l_mine * weight;
    const int n = min(32, parts.splits - base);
    for (int first = share * groups; first < n; first += groups * SHARE * 4) {  // four turns' loads together
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        const int e = column + pass * 128;
        if (pass > 0 && pass * 128 >= value_dim) continue;
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = min(first + u * groups * SHARE + mine, n - 1);
          const float* from = parts.o + (part0 + base + i) * value_dim;
          if (whole) {
            v[u] = __ldcg(reinterpret_cast<const float4*>(from + min(e, value_dim - 4)));
          } else {
            v[u].x = __ldcg(from + min(e, value_dim - 1));
            v[u].y = __ldcg(from + min(e + 1, value_dim - 1));
            v[u].z = __ldcg(from + min(e + 2, value_dim - 1));
            v[u].w = __ldcg(from + min(e + 3, value_dim - 1));
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = first + u * groups * SHARE + mine;
          const float w = __shfl_sync(0xffffffffu, weight, min(i, 31));
          if (i < n) {
            acc[pass][0] += v[u].x * w; acc[pass][1] += v[u].y * w; acc[pass][2] += v[u].z * w; acc[pass][3] += v[u].w * w;
          }
        }
      }
    }
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    l_all += __shfl_xor_sync(0xffffffffu, l_all, d);
    if (d >= across)
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[pass][e] += __shfl_xor_sync(0xffffffffu, acc[pass][e], d);
  }
  if (SHARE > 1) {
    if (mine == 0)
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
        for (int e = 0; e < 4; ++e) sh_acc[share][pass * 128 + column + e] = acc[pass][e];
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        for (int w = 1; w < SHARE; ++w) acc[pass][e] += sh_acc[w][pass * 128 + column + e];
  }
  if (mine != 0) return;
  const float inv = rows.extras.sink ? sink_inverse_log2(m_all, l_all, rows.extras.sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
#pragma unroll
  for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = pass * 128 + column + e;
      if (at < value_dim) out[(size_t)token * out_stride + (size_t)head * value_dim + at] = from_float<T>(acc[pass][e] * inv);
    }
}

template <typename T>
static int rows_merge(const Partials& parts, const QueryRows& rows, void* out, int out_stride, int value_dim, cudaStream_t stream) {
  const int count = rows.tokens * rows.num_heads;
  if (parts.splits > 16 || (parts.splits > 4 && count <= 512))
    return (int)launch_dependent(attention_rows_merge_kernel<T, 4>, dim3(count), dim3(kMergeThreads), 0, stream, parts, rows, (T*)out, out_stride,
                                 count, value_dim);
  return (int)launch_dependent(attention_rows_merge_kernel<T, 1>, dim3((count + 3) / 4), dim3(kMergeThreads), 0, stream, parts, rows, (T*)out,
                               out_stride, count, value_dim);
}

int rows_merge_bf16(const Partials& parts, const QueryRows& rows, void* out, int out_stride, int value_dim, cudaStream_t stream) {
  return rows_merge<__nv_bfloat16>(parts, rows, out, out_stride, value_dim, stream);
}

}  // namespace distie

using namespace distie;

// q [tokens, >= heads * key_dim], out [tokens, heads * value_dim] of type `dtype`; seqs null: single tokens, `requests` of
// them, else [requests, 3] with at most most_nodes new tokens each.  scratch: tokens * heads * splits * (value size + 2) floats.
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
  if ((long long)num_pages * num_kv_heads * page_size > 0xffffffffLL) return DISTIE_ERR_UNSUPPORTED;
  const CachePages cache = make_pages(k_cache, v_cache, k_scale, v_scale, block_table, table_width, num_kv_heads, key_dim, value_dim,
                                      page_size, num_pages);
  const QueryRows rows{positions, token_seq, seq_seat, seqs, bits, words, tokens, requests, most_nodes, num_heads / num_kv_heads, num_heads, window, chunk, keep_first,
                       scale * 1.4426950408889634f, make_score_extras(scale, softcap, sink)};
  const Partials parts{scratch, scratch ? scratch + (size_t)tokens * num_heads * splits * value_dim : nullptr, splits};
  const int tiles = (most_nodes * rows.group + kRowsTile - 1) / kRowsTile;
  const dim3 grid(tiles * num_kv_heads, requests, splits);
  const size_t shared = ((size_t)kRowsTile * key_dim + (size_t)kRowsKeys * (rows_k_pitch(key_dim) + value_dim)) * sizeof(float);
  cudaError_t err;
#define DISTIE_ROWS(T, CACHE)                                                                                                       \
  {                                                                                                                                 \
    if (shared > 40 * 1024 && (err = cudaFuncSetAttribute(attention_rows_kernel<T, CACHE>, /* (48 KB hold the static arrays too) */  \
                                                          cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024)) != cudaSuccess)  \
      return (int)err;                                                                                        \
    err = launch_dependent(attention_rows_kernel<T, CACHE>, grid, dim3(kRowsThreads), shared, stream, (const T*)q, q_stride, (T*)out,         \
                           out_stride, rows, cache, parts, error);                                                                   \
    if (err != cudaSuccess) return (int)err;                                                                                        \
    if (splits > 1) return rows_merge<T>(parts, rows, out, out_stride, value_dim, stream);                                             \
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
