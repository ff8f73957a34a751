// Rows on their way into the cache and back: queries, keys and values of a step finished from the projection and stored,
// in the engine's type or as e4m3 numbers with a scale per row (cached_rows.cuh); pages of an 8-bit cache read back.
#include <cuda_fp16.h>

#include "cached_rows.cuh"
#include "packed.h"

namespace distie {

// ---- write --------------------------------------------------------------------------------------------------------
// From the projection [q | k | v] (float32, the slices of a split product, or 16-bit) plus bias: every head of q and k
// optionally divided by its root mean square before or after the rotation, rotated, q also times a temperature; q goes to
// q_out, k and v to their place in the pages.  A token's place in its request may differ from its position (drafted tokens:
// siblings share a position).  The value can be the key as projected.  All arithmetic is float32.
struct RowsInput {
  const void* q;
  const void* k;
  const void* v;      // null: the value is the key with its bias, before anything else is done to it
  int q_stride, k_stride, v_stride;  // elements between tokens
  int splits;
  long long split_stride;  // elements between slices (float32 only)
  const float* q_bias;
  const float* k_bias;
  const float* v_bias;
};
struct RowsNorm {
  int mode;  // 0 none, 1 before the rotation, 2 after it
  float eps;
  const float* q_weight;
  const float* k_weight;
};
struct RowsTurn {
  const float* inv_freq;  // null: nothing is rotated
  int rotary_dim, interleaved;
  int rounded;            // whether position * frequency is rounded to float32, as by the kernels for rows at their positions
  float factor;
  float temp_coef, temp_every;  // temp_every > 0: q at position p times 1 + coef ln(floor((p + 1) / every) + 1)
};
struct RowsPlace {
  const int* positions;
  const int* slots;  // places in the requests; null: the positions
  const int* token_seq;
  const int* seq_seat;
};

// cos and sin of position * frequency: of the float32 product (`rounded`), as the rotations of all other steps and of the
// checkpoints' own code take it, so that rows of drafted tokens fit the rows they stand beside; or of the exact product.  There
// the product's rounding error e, up to 2^-24 of an angle of many turns, comes back as a small rotation, without its terms from
// e^3 / 6 on: 8e-8 up to position 2^18.  (A float32 product alone is off by 4e-3 at position 65,536.)
__device__ __forceinline__ void turn_angle(int position, float frequency, int rounded, float& sn, float& cs) {
  const float p = (float)position, high = __fmul_rn(p, frequency), low = rounded ? 0.f : __fmaf_rn(p, frequency, -high);
  float s, c;
  sincosf(high, &s, &c);
  const float half = 0.5f * low * low;
  sn = s + (c * low - s * half);
  cs = c - (s * low + c * half);
}

template <typename IN>
__device__ __forceinline__ float input_at(const RowsInput& in, const void* rows, size_t at) {
  const IN* p = reinterpret_cast<const IN*>(rows) + at;
  float v = to_float(*p);
  for (int s = 1; s < in.splits; ++s) v += to_float(p[s * in.split_stride]);
  return v;
}

// Scale of a row of largest magnitude `most` (bad: some element is not finite).
__device__ __forceinline__ float row_scale(float most, bool bad) { return bad ? __int_as_float(0x7fc00000) : most / kE4m3Most; }

constexpr int kWriteWarps = 4;

// A warp per row, a row of any size through shared memory.
template <typename IN, typename T, int CACHE>
__global__ void __launch_bounds__(kWriteWarps * 32)
rows_write_kernel(RowsInput in, RowsNorm norm, RowsTurn turn, RowsPlace place, T* __restrict__ q_out, int q_out_stride,
                  CachePages cache, void* k_out, void* v_out, float* k_scale, float* v_scale, int num_heads, int num_kv_heads,
                  int write, int* __restrict__ error) {
  extern __shared__ __align__(16) float rows_s[];  // a piece per warp, then cos and sin of the token
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dim = cache.key_dim, vdim = cache.value_dim, piece = max(dim, vdim);
  float* row_s = rows_s + (size_t)warp * piece;
  float* cos_s = rows_s + (size_t)kWriteWarps * piece;
  const int half = turn.inv_freq ? turn.rotary_dim / 2 : 0;
  float* sin_s = cos_s + half;
  const int position = place.positions[t];
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    float sn, cs;
    turn_angle(position, turn.inv_freq[i], turn.rounded, sn, cs);
    cos_s[i] = cs * turn.factor;
    sin_s[i] = sn * turn.factor;
  }
  long long place_row = -1;  // of kv head 0
  if (write) {
    const int seat = place.seq_seat[place.token_seq[t]];
    const int slot = place.slots ? place.slots[t] : position;
    place_row = slot < 0 ? -1 : cache.row_of(cache.block_table + (size_t)seat * cache.table_width, slot, 0);
    if (place_row < 0 && threadIdx.x == 0 && error) atomicExch(error, 2);
  }
  const float temperature =
      turn.temp_every > 0.f ? 1.f + turn.temp_coef * logf(floorf((float)(position + 1) / turn.temp_every) + 1.f) : 1.f;
  __syncthreads();
  const int rows_here = num_heads + (write ? 2 * num_kv_heads : 0);
  for (int index = blockIdx.y * kWriteWarps + warp; index < rows_here; index += gridDim.y * kWriteWarps) {
    const bool is_query = index < num_heads, is_value = index >= num_heads + num_kv_heads;
    const int head = is_query ? index : (index - num_heads) % num_kv_heads;
    const bool from_key = is_value && in.v == nullptr;
    const int n = is_value ? vdim : dim;
    const void* rows = is_query ? in.q : (is_value && !from_key) ? in.v : in.k;
    const int stride = is_query ? in.q_stride : (is_value && !from_key) ? in.v_stride : in.k_stride;
    const float* bias = is_query ? in.q_bias : (is_value && !from_key) ? in.v_bias : in.k_bias;
    if (!is_query && place_row < 0) continue;
    const size_t at = (size_t)t * stride + (size_t)head * n;
    // A value goes straight to its page; a query or key stays in shared memory between the steps.
    float squares = 0.f;
    if (!is_value) {
      for (int e = lane; e < n; e += 32) {
        const float x = input_at<IN>(in, rows, at + e) + (bias ? bias[head * n + e] : 0.f);
        row_s[e] = x;
        squares += x * x;
      }
      const float* weight = is_query ? norm.q_weight : norm.k_weight;
      if (norm.mode == 1) {
        const float unit = rsqrtf(warp_sum(squares) / (float)n + norm.eps);
        for (int e = lane; e < n; e += 32) row_s[e] = row_s[e] * unit * (weight ? weight[e] : 1.f);
      }
      __syncwarp();
      for (int i = lane; i < half; i += 32) {
        const int a = turn.interleaved ? 2 * i : i, b = turn.interleaved ? 2 * i + 1 : i + half;
        const float sn = sin_s[i], cs = cos_s[i], u = row_s[a], v = row_s[b];
        row_s[a] = u * cs - v * sn;
        row_s[b] = v * cs + u * sn;
      }
      __syncwarp();
      if (norm.mode == 2) {
        squares = 0.f;
        for (int e = lane; e < n; e += 32) squares += row_s[e] * row_s[e];
        const float unit = rsqrtf(warp_sum(squares) / (float)n + norm.eps);
        for (int e = lane; e < n; e += 32) row_s[e] = row_s[e] * unit * (weight ? weight[e] : 1.f);
        __syncwarp();
      }
    } else {
      for (int e = lane; e < n; e += 32) row_s[e] = input_at<IN>(in, rows, at + e) + (bias ? bias[head * n + e] : 0.f);
      __syncwarp();
    }
    if (is_query) {
      for (int e = lane; e < n; e += 32) q_out[(size_t)t * q_out_stride + (size_t)head * n + e] = from_float<T>(row_s[e] * temperature);
    } else {
      const size_t to = (size_t)(place_row + (long long)head * cache.page_size) * n;
      void* out = is_value ? v_out : k_out;
      if (CACHE == DISTIE_E4M3) {
        float most = 0.f;
        bool bad = false;
        for (int e = lane; e < n; e += 32) {
          const float size = fabsf(row_s[e]);
          bad |= !(size <= 3.402823466e38f);
          most = fmaxf(most, size);
        }
        most = warp_max(most);
        bad = __any_sync(0xffffffffu, bad);
        const float scale = row_scale(most, bad);
        if (lane == 0) (is_value ? v_scale : k_scale)[place_row + (long long)head * cache.page_size] = scale;
        for (int e = lane; e < n; e += 32)
          reinterpret_cast<uint8_t*>(out)[to + e] =
              (bad || scale == 0.f) ? (uint8_t)0 : (uint8_t)__nv_cvt_float_to_fp8(row_s[e] / scale, __NV_SATFINITE, __NV_E4M3);
      } else {
        for (int e = lane; e < n; e += 32) {
          if (CACHE == DISTIE_BF16) reinterpret_cast<__nv_bfloat16*>(out)[to + e] = __float2bfloat16_rn(row_s[e]);
          else reinterpret_cast<float*>(out)[to + e] = row_s[e];
        }
      }
    }
    __syncwarp();  // before the next row overwrites the piece
  }
}

// The same for heads of 64 and 128 whose keys and values are of one size, turned whole (pairs half a head apart) or not at
// all, from float32: D / 16 lanes a row, a lane 8 elements and the 8 that are turned with them.  A block takes as many tokens
// as make one wave of blocks, up to 8, and walks their rows in one go, a lane's next row on its way: the tokens'
// places, three loads that hang on one another, and their angles, one a thread, are then paid for once a block.  Where tokens
// are few, a token's rows are spread over several blocks.  Behind the bytes (2,048 tokens of 40 and 8 heads of 128: 80 MB)
// the instructions set the pace: 18.4 us, 1.3 of them the divisions by the scales.
constexpr int kFastThreads = 256, kFastTokens = 8, kFastBlocksPerSm = 3;

template <typename T, int CACHE, int D>
__global__ void __launch_bounds__(kFastThreads, kFastBlocksPerSm)
rows_write_fast_kernel(RowsInput in, RowsNorm norm, RowsTurn turn, RowsPlace place, T* __restrict__ q_out, int q_out_stride,
                       CachePages cache, void* k_out, void* v_out, float* __restrict__ k_scale, float* __restrict__ v_scale, int tokens,
                       int per_block, int num_heads, int num_kv_heads, int write, int* __restrict__ error) {
  constexpr int LANES = D / 16, HALF = D / 2, PART = D / 4, ROWS = kFastThreads / LANES;
  constexpr unsigned ALL = 0xffffffffu;
  __shared__ __align__(16) float cos_s[kFastTokens][HALF], sin_s[kFastTokens][HALF];
  __shared__ long long place_s[kFastTokens];  // of kv head 0; -1: none
  __shared__ float temperature_s[kFastTokens];
  const int t0 = blockIdx.x * per_block, count = min(per_block, tokens - t0), e0 = (threadIdx.x % LANES) * 4;
  const int k_row = num_heads, v_row = num_heads + num_kv_heads, rows_here = num_heads + (write ? 2 * num_kv_heads : 0);
  const int step = gridDim.y * ROWS, total = count * rows_here;
  const int passes = (total - (int)blockIdx.y * ROWS + step - 1) / step;  // the same for every thread of the block
  grid_dependency_release();
  // Elements e0 .. + 3 and PART + e0 .. + 3 of the row, then their partners HALF further on.
  struct Row {
    float4 x[4];
    int token, row;  // of the block's tokens, of the token's rows
  };
  auto load = [&](Row& r) {  // a row as projected (behind the last one: a row of the last token, so that no load hangs on a branch)
    const bool is_query = r.row < k_row, is_value = r.row >= v_row;
    const bool own = is_value && in.v != nullptr;
    const float* rows = reinterpret_cast<const float*>(is_query ? in.q : own ? in.v : in.k);
    const int stride = is_query ? in.q_stride : own ? in.v_stride : in.k_stride;
    const int head = r.row - (is_query ? 0 : is_value ? v_row : k_row);
    const float* from = rows + (size_t)(t0 + min(r.token, count - 1)) * stride + head * D + e0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.x[i] = load4_cg(from + i * PART);
    for (int s = 1; s < in.splits; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 more = load4_cg(from + s * in.split_stride + i * PART);
        r.x[i].x += more.x; r.x[i].y += more.y; r.x[i].z += more.z; r.x[i].w += more.w;
      }
  };
  auto advance = [&](Row& r, int by) {
    r.row += by;
    while (r.row >= rows_here) {
      r.row -= rows_here;
      ++r.token;
    }
  };
  Row held[2];
  grid_dependency_wait();  // the projection comes from the kernel before this one
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    held[u].token = 0;
    held[u].row = blockIdx.y * ROWS + threadIdx.x / LANES;
    advance(held[u], u * step);
    load(held[u]);
  }
  // While they are on their way: the tokens' places and angles.
  if (threadIdx.x / 32 < count && threadIdx.x % 32 == 0) {
    const int mine = threadIdx.x / 32, t = t0 + mine, position = place.positions[t];
    long long row = -1;
    if (write) {
      const int seat = place.seq_seat[place.token_seq[t]], slot = place.slots ? place.slots[t] : position;
      row = slot < 0 ? -1 : cache.row_of(cache.block_table + (size_t)seat * cache.table_width, slot, 0);
      if (row < 0 && blockIdx.y == 0 && error) atomicExch(error, 2);
    }
    place_s[mine] = row;
    temperature_s[mine] =
        turn.temp_every > 0.f ? 1.f + turn.temp_coef * logf(floorf((float)(position + 1) / turn.temp_every) + 1.f) : 1.f;
  }
  if (turn.inv_freq) {
    for (int i = threadIdx.x; i < count * HALF; i += kFastThreads) {
      float sn, cs;
      turn_angle(place.positions[t0 + i / HALF], turn.inv_freq[i % HALF], turn.rounded, sn, cs);
      cos_s[i / HALF][i % HALF] = cs * turn.factor;
      sin_s[i / HALF][i % HALF] = sn * turn.factor;
    }
  }
  __syncthreads();
  auto finish = [&](Row& r) {
    const bool live = r.token < count, is_query = r.row < k_row, is_value = r.row >= v_row;
    const int token = min(r.token, count - 1), head = r.row - (is_query ? 0 : is_value ? v_row : k_row);
    const float* bias = is_query ? in.q_bias : is_value && in.v != nullptr ? in.v_bias : in.k_bias;
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[4 * i] = r.x[i].x; v[4 * i + 1] = r.x[i].y; v[4 * i + 2] = r.x[i].z; v[4 * i + 3] = r.x[i].w;
    }
    if (bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(bias + head * D + e0 + i * PART));
        v[4 * i] += b.x; v[4 * i + 1] += b.y; v[4 * i + 2] += b.z; v[4 * i + 3] += b.w;
      }
    }
    auto unit = [&]() {  // (all lanes: a warp's rows may be of several kinds)
      float squares = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) squares += v[e] * v[e];
#pragma unroll
      for (int d = LANES / 2; d >= 1; d >>= 1) squares += __shfl_xor_sync(ALL, squares, d);
      const float u = is_value ? 1.f : rsqrtf(squares / (float)D + norm.eps);
      const float* weight = is_query ? norm.q_weight : norm.k_weight;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4 w = make_float4(u, u, u, u);
        if (weight && !is_value) {
          const float4 given = __ldg(reinterpret_cast<const float4*>(weight + e0 + i * PART));
          w = make_float4(u * given.x, u * given.y, u * given.z, u * given.w);
        }
        v[4 * i] *= w.x; v[4 * i + 1] *= w.y; v[4 * i + 2] *= w.z; v[4 * i + 3] *= w.w;
      }
    };
    if (norm.mode == 1) unit();
    if (turn.inv_freq && !is_value) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 cs = load4(&cos_s[token][e0 + i * PART]), sn = load4(&sin_s[token][e0 + i * PART]);
        const float c[4] = {cs.x, cs.y, cs.z, cs.w}, s[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = v[4 * i + e], b = v[8 + 4 * i + e];
          v[4 * i + e] = a * c[e] - b * s[e];
          v[8 + 4 * i + e] = b * c[e] + a * s[e];
        }
      }
    }
    if (norm.mode == 2) unit();
    if (__any_sync(ALL, !is_query)) {
      const long long row = place_s[token] + (long long)head * cache.page_size;
      const bool there = live && !is_query && place_s[token] >= 0;
      void* out = is_value ? v_out : k_out;
      if (CACHE == DISTIE_E4M3) {
        float most = 0.f, nothing = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          most = fmaxf(most, fabsf(v[e]));
          nothing += v[e] * 0.f;  // NaN where an element is not finite
        }
#pragma unroll
        for (int d = LANES / 2; d >= 1; d >>= 1) {
          most = fmaxf(most, __shfl_xor_sync(ALL, most, d));
          nothing += __shfl_xor_sync(ALL, nothing, d);
        }
        if (there) {
          const bool bad = nothing != nothing;
          const float scale = row_scale(most, bad);
          if (e0 == 0) (is_value ? v_scale : k_scale)[row] = scale;
          const bool nothing_held = bad || scale == 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = nothing_held ? 0.f : v[e] / scale;  // (times 1 / scale, numbers next to a border fell on its other side)
          uint32_t* to = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(out) + (size_t)row * D + e0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            to[i * PART / 4] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
                               (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
        }
      } else if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 part = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          if (CACHE == DISTIE_BF16) store4(reinterpret_cast<__nv_bfloat16*>(out) + (size_t)row * D + e0 + i * PART, part);
          else store4(reinterpret_cast<float*>(out) + (size_t)row * D + e0 + i * PART, part);
        }
      }
    }
    if (live && is_query) {
      const float times = temperature_s[token];
      T* to = q_out + (size_t)(t0 + token) * q_out_stride + head * D + e0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(to + i * PART, make_float4(v[4 * i] * times, v[4 * i + 1] * times, v[4 * i + 2] * times, v[4 * i + 3] * times));
    }
  };
  for (int pass = 0; pass < passes; pass += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // (a row that moved from one place to the other would be waited for)
      if (pass + u < passes) {
        finish(held[u]);
        advance(held[u], 2 * step);
        load(held[u]);
      }
    }
  }
}

// ---- read back ----------------------------------------------------------------------------------------------------
// Pages of up to kReadRows requests, one page of the result per block: numbers times scales in the set's type, zeros behind
// a request's last row.  A page of the cache is one run of memory over all kv heads, and so is a page of the result.
constexpr int kReadRows = 256, kReadFewRows = 8;  // (a launch copies the whole plan: 6 KB or 200 bytes)
template <int ROWS>
struct ReadPlan {
  int count;
  int batch_row[ROWS];    // of the step: its seat is read
  int first_page[ROWS];   // pages of the result before this request's
  int first_column[ROWS]; // its first logical page that is read
  int hole[ROWS];         // logical pages hole .. hole_end - 1 are not read: a window has passed them
  int hole_end[ROWS];
  int length[ROWS];       // its keys
};

template <typename T>
__device__ __forceinline__ void store_row16(T* to, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float half[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) half[e] = v[8 * i + e];
    store8(to + 8 * i, half);
  }
}

// The rows of the result's table that belong to the requests' seats.  The attention that follows starts early and looks at its
// block table before it waits, as at an input of the step (common.cuh).  So this is a kernel of its own, launched the ordinary
// way before the pages are read and releasing nobody: rows_read_kernel does not start before it has ended, and releases the
// attention only once it has seen that.
template <int ROWS>
__global__ void __launch_bounds__(128)
rows_table_kernel(const __grid_constant__ ReadPlan<ROWS> plan, const int* __restrict__ seq_seat, int page_size, int* __restrict__ table_out,
                  int table_width) {
  const int i = blockIdx.x, columns = (plan.length[i] + page_size - 1) / page_size;
  int* row = table_out + (size_t)seq_seat[plan.batch_row[i]] * table_width;
  for (int c = threadIdx.x; c < table_width; c += blockDim.x)
    row[c] = c >= plan.first_column[i] && c < columns && (c < plan.hole[i] || c >= plan.hole_end[i])
                 ? plan.first_page[i] + c - plan.first_column[i] : -1;
}

constexpr int kReadThreads = 256;
constexpr int kReadPieces = 4;  // 16 numbers each, per thread: all requested before the first is stored

// A block takes kReadThreads * kReadPieces pieces of a page (blockIdx.y: which of them, K's first, then V's).
template <typename T, int ROWS>
__global__ void __launch_bounds__(kReadThreads)
rows_read_kernel(const __grid_constant__ ReadPlan<ROWS> plan, CachePages cache, const int* __restrict__ seq_seat, T* __restrict__ k_out,
                 T* __restrict__ v_out, int page0, int* __restrict__ error) {
  const int page_out = page0 + blockIdx.x;
  int i = 0;
  for (int step = ROWS / 2; step > 0; step >>= 1)
    if (i + step < plan.count && plan.first_page[i + step] <= page_out) i += step;
  const int column = plan.first_column[i] + page_out - plan.first_page[i];
  if (column >= plan.hole[i] && column < plan.hole_end[i]) return;  // (no table entry names this page of the result)
  const int seat = seq_seat[plan.batch_row[i]];
  const int page = column < cache.table_width ? cache.block_table[(size_t)seat * cache.table_width + column] : -1;
  const bool held = page >= 0 && page < cache.num_pages;
  const int live = held ? min(cache.page_size, plan.length[i] - column * cache.page_size) : 0;
  const int rows = cache.num_kv_heads * cache.page_size;
  const size_t from = (size_t)(held ? page : 0) * rows, to = (size_t)page_out * rows;
  grid_dependency_wait();  // the newest rows come from the kernels before this one
  grid_dependency_release();  // (not before the wait: see rows_table_kernel)
  if (!held && threadIdx.x == 0 && blockIdx.y == 0 && error) atomicExch(error, 5);
  auto live_row = [&](int row) { return (cache.page_shift >= 0 ? row & (cache.page_size - 1) : row % cache.page_size) < live; };
  if (((cache.key_dim | cache.value_dim) & 15) == 0) {
    const int k_pieces = rows * (cache.key_dim / 16), all = k_pieces + rows * (cache.value_dim / 16);
    const int first = blockIdx.y * kReadThreads * kReadPieces + threadIdx.x;
    uint4 raw[kReadPieces];
    float scale[kReadPieces];
    int row[kReadPieces];
#pragma unroll
    for (int u = 0; u < kReadPieces; ++u) {  // (every piece is loaded, those behind the last one as copies of it)
      const int p = min(first + u * kReadThreads, all - 1);
      const bool is_v = p >= k_pieces;
      const int piece = is_v ? p - k_pieces : p, dim = is_v ? cache.value_dim : cache.key_dim;
      row[u] = piece / (dim / 16);
      raw[u] = load16_cg(reinterpret_cast<const uint8_t*>(is_v ? cache.v : cache.k) + from * dim + (size_t)piece * 16);
      scale[u] = __ldcg((is_v ? cache.v_scale : cache.k_scale) + from + row[u]);
    }
#pragma unroll
    for (int u = 0; u < kReadPieces; ++u) {
      const int p = first + u * kReadThreads;
      if (p >= all) break;
      const bool is_v = p >= k_pieces, there = live_row(row[u]);
      const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      float v[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        e4m3x4_to_float(w[j], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = there ? f[e] * scale[u] : 0.f;
      }
      const int piece = is_v ? p - k_pieces : p;
      store_row16((is_v ? v_out + to * cache.value_dim : k_out + to * cache.key_dim) + (size_t)piece * 16, v);
    }
  } else if (blockIdx.y == 0) {
    for (int which = 0; which < 2; ++which) {
      const int dim = which ? cache.value_dim : cache.key_dim;
      const uint8_t* numbers = reinterpret_cast<const uint8_t*>(which ? cache.v : cache.k) + from * dim;
      const float* scales = (which ? cache.v_scale : cache.k_scale) + from;
      T* out = (which ? v_out : k_out) + to * dim;
      for (int e = threadIdx.x; e < rows * dim; e += blockDim.x) {
        const int row = e / dim;
        out[e] = from_float<T>(live_row(row) ? e4m3_to_float(numbers[e]) * scales[row] : 0.f);
      }
    }
  }
}

template <typename IN, typename T, int CACHE>
static int launch_write(const RowsInput& in, const RowsNorm& norm, const RowsTurn& turn, const RowsPlace& place, void* q_out,
                        int q_out_stride, const CachePages& cache, void* k_out, void* v_out, float* k_scale, float* v_scale,
                        int tokens, int num_heads, int num_kv_heads, int write, int* error, cudaStream_t stream) {
  const int rows = num_heads + (write ? 2 * num_kv_heads : 0);
  const int dim = cache.key_dim;
  auto aligned = [](const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; };
  if (sizeof(IN) == 4 && (dim == 64 || dim == 128) && cache.value_dim == dim &&
      (turn.rotary_dim == 0 || (turn.rotary_dim == dim && !turn.interleaved)) && !((in.q_stride | in.k_stride | in.v_stride) & 3) &&
      !(in.split_stride & 3) && !(q_out_stride & 3) && aligned(in.q, 16) && aligned(in.k, 16) && aligned(in.v, 16) && aligned(in.q_bias, 16) &&
      aligned(in.k_bias, 16) && aligned(in.v_bias, 16) && aligned(norm.q_weight, 16) && aligned(norm.k_weight, 16) && aligned(q_out, 16) &&
      aligned(k_out, 16) && aligned(v_out, 16)) {
    static int sms = 0;
    if (sms == 0) {
      int device = 0;
      if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms < 1)
        sms = 148;
    }
    const int wave = sms * kFastBlocksPerSm, blocks_a_token = (rows * dim / 16 + kFastThreads - 1) / kFastThreads;
    const int per_block = min(kFastTokens, (tokens + wave - 1) / wave);
    const dim3 fast((tokens + per_block - 1) / per_block, max(1, min(blocks_a_token, wave / tokens)));
#define DISTIE_ROWS_FAST(D)                                                                                                            \
  return (int)launch_dependent(rows_write_fast_kernel<T, CACHE, D>, fast, dim3(kFastThreads), 0, stream, in, norm, turn, place, (T*)q_out, \
                               q_out_stride, cache, k_out, v_out, k_scale, v_scale, tokens, per_block, num_heads, num_kv_heads, write, error)
    if (dim == 64) DISTIE_ROWS_FAST(64);
    DISTIE_ROWS_FAST(128);
#undef DISTIE_ROWS_FAST
  }
  const dim3 grid(tokens, tokens < 512 ? (rows + kWriteWarps - 1) / kWriteWarps : 1);
  const size_t shared = ((size_t)kWriteWarps * max(cache.key_dim, cache.value_dim) + turn.rotary_dim) * sizeof(float);
  rows_write_kernel<IN, T, CACHE><<<grid, kWriteWarps * 32, shared, stream>>>(in, norm, turn, place, (T*)q_out, q_out_stride, cache, k_out,
                                                                              v_out, k_scale, v_scale, num_heads, num_kv_heads, write, error);
  DISTIE_LAUNCH_CHECK();
  return 0;
}

}  // namespace distie

using namespace distie;

// in_type: DISTIE_F32 or DISTIE_BF16 (one slice).  out_type: of q_out.  cache_type: DISTIE_F32, DISTIE_BF16 or DISTIE_E4M3
// (with scales).  num_heads 0: there are no queries.  write 0: only the queries are made.
extern "C" int distie_rows_write(const void* q, int q_stride, const void* k, int k_stride, const void* v, int v_stride, int in_type,
                                 int splits, long long split_stride, const float* q_bias, const float* k_bias, const float* v_bias,
                                 int norm_mode, float norm_eps, const float* q_weight, const float* k_weight, const float* inv_freq,
                                 int rotary_dim, int interleaved, int rounded, float factor, float temp_coef, float temp_every,
                                 const int* positions, const int* slots, const int* token_seq, const int* seq_seat,
                                 const int* block_table, int table_width, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                 int tokens, int num_heads, int num_kv_heads, int key_dim, int value_dim, int page_size, int num_pages,
                                 int write, void* q_out, int q_out_stride, int out_type, int cache_type, int* error,
                                 cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (num_heads < 0 || num_kv_heads < 1 || key_dim < 1 || key_dim > 1024 || value_dim < 1 || value_dim > 1024 || rotary_dim < 0 ||
      rotary_dim > key_dim || (rotary_dim & 1) || splits < 1 || page_size < 1 || table_width < 1 || num_heads + 2 * num_kv_heads > 65535 ||
      (in_type == DISTIE_BF16 && splits != 1) || (num_heads > 0 && (q == nullptr || q_out == nullptr)) ||
      (write && (k == nullptr || k_cache == nullptr || v_cache == nullptr || block_table == nullptr)) ||
      (write && v == nullptr && value_dim != key_dim) || (write && cache_type == DISTIE_E4M3 && (k_scale == nullptr || v_scale == nullptr)) ||
      norm_mode < 0 || norm_mode > 2)
    return DISTIE_ERR_ARG;
  const RowsInput in{q, k, v, q_stride, k_stride, v_stride, splits, split_stride, q_bias, k_bias, v_bias};
  const RowsNorm norm{norm_mode, norm_eps, q_weight, k_weight};
  const RowsTurn turn{rotary_dim > 0 ? inv_freq : nullptr, rotary_dim, interleaved, rounded, factor, temp_coef, temp_every};
  const RowsPlace place{positions, slots, token_seq, seq_seat};
  const CachePages cache = make_pages(k_cache, v_cache, k_scale, v_scale, block_table, table_width, num_kv_heads, key_dim, value_dim,
                                      page_size, num_pages);
#define DISTIE_ROWS_WRITE(IN, T, CACHE)                                                                                     \
  return launch_write<IN, T, CACHE>(in, norm, turn, place, q_out, q_out_stride, cache, k_cache, v_cache, k_scale, v_scale,   \
                                    tokens, num_heads, num_kv_heads, write, error, stream)
  if (in_type == DISTIE_F32 && out_type == DISTIE_BF16) {
    if (cache_type == DISTIE_E4M3) DISTIE_ROWS_WRITE(float, __nv_bfloat16, DISTIE_E4M3);
    if (cache_type == DISTIE_BF16) DISTIE_ROWS_WRITE(float, __nv_bfloat16, DISTIE_BF16);
  } else if (in_type == DISTIE_BF16 && out_type == DISTIE_BF16) {
    if (cache_type == DISTIE_E4M3) DISTIE_ROWS_WRITE(__nv_bfloat16, __nv_bfloat16, DISTIE_E4M3);
    if (cache_type == DISTIE_BF16) DISTIE_ROWS_WRITE(__nv_bfloat16, __nv_bfloat16, DISTIE_BF16);
  } else if (in_type == DISTIE_F32 && out_type == DISTIE_F32) {
    if (cache_type == DISTIE_E4M3) DISTIE_ROWS_WRITE(float, float, DISTIE_E4M3);
    if (cache_type == DISTIE_F32) DISTIE_ROWS_WRITE(float, float, DISTIE_F32);
  }
#undef DISTIE_ROWS_WRITE
  return DISTIE_ERR_UNSUPPORTED;
}

template <int ROWS>
static ReadPlan<ROWS> read_plan(const int* plan, int count) {
  ReadPlan<ROWS> p;
  p.count = count;
  for (int i = 0; i < count; ++i) {
    p.batch_row[i] = plan[6 * i];
    p.first_page[i] = plan[6 * i + 1];
    p.first_column[i] = plan[6 * i + 2];
    p.hole[i] = plan[6 * i + 3];
    p.hole_end[i] = plan[6 * i + 4];
    p.length[i] = plan[6 * i + 5];
  }
  return p;
}

template <typename T>
static int launch_read(const int* plan, int count, const dim3& grid, const CachePages& cache, const int* seq_seat, void* k_out, void* v_out,
                       int page0, int* error, cudaStream_t stream) {
  if (count <= kReadFewRows)
    return (int)launch_dependent(rows_read_kernel<T, kReadFewRows>, grid, dim3(kReadThreads), 0, stream, read_plan<kReadFewRows>(plan, count),
                                 cache, seq_seat, (T*)k_out, (T*)v_out, page0, error);
  return (int)launch_dependent(rows_read_kernel<T, kReadRows>, grid, dim3(kReadThreads), 0, stream, read_plan<kReadRows>(plan, count), cache,
                               seq_seat, (T*)k_out, (T*)v_out, page0, error);
}

// plan: `count` rows (batch row, first page of the result, first logical page, hole, end of the hole, keys) on the host; their
// pages of the result are page0 .. page0 + pages - 1.
extern "C" int distie_rows_read(const int* plan, int count, const void* k_cache, const void* v_cache, const float* k_scale,
                                const float* v_scale, const int* block_table, int table_width, const int* seq_seat, int num_kv_heads,
                                int key_dim, int value_dim, int page_size, int num_pages, void* k_out, void* v_out, int page0, int pages,
                                int out_type, int* error, cudaStream_t stream) {
  if (count <= 0 || pages <= 0) return 0;
  if (count > kReadRows || num_kv_heads < 1 || key_dim < 1 || value_dim < 1 || page_size < 1 || table_width < 1 || k_scale == nullptr || v_scale == nullptr ||
      (long long)num_kv_heads * page_size * (key_dim + value_dim) > 1 << 30)
    return DISTIE_ERR_ARG;
  const CachePages cache = make_pages(k_cache, v_cache, k_scale, v_scale, block_table, table_width, num_kv_heads, key_dim, value_dim,
                                      page_size, num_pages);
  const long long pieces = (long long)num_kv_heads * page_size * (key_dim / 16 + value_dim / 16);
  const int per_block = kReadThreads * kReadPieces;
  const dim3 grid(pages, ((key_dim | value_dim) & 15) == 0 ? (unsigned)((pieces + per_block - 1) / per_block) : 1);
  if (out_type == DISTIE_BF16)
    return launch_read<__nv_bfloat16>(plan, count, grid, cache, seq_seat, k_out, v_out, page0, error, stream);
  if (out_type == DISTIE_F32) return launch_read<float>(plan, count, grid, cache, seq_seat, k_out, v_out, page0, error, stream);
  return DISTIE_ERR_UNSUPPORTED;
}

// Of the table [seats, table_width] of the pages read back, the rows of the plan's requests.
extern "C" int distie_rows_table(const int* plan, int count, const int* seq_seat, int page_size, int* table_out, int table_width,
                                 cudaStream_t stream) {
  if (count <= 0) return 0;
  if (count > kReadRows || page_size < 1 || table_width < 1) return DISTIE_ERR_ARG;
  if (count <= kReadFewRows)
    rows_table_kernel<kReadFewRows><<<count, 128, 0, stream>>>(read_plan<kReadFewRows>(plan, count), seq_seat, page_size, table_out, table_width);
  else
    rows_table_kernel<kReadRows><<<count, 128, 0, stream>>>(read_plan<kReadRows>(plan, count), seq_seat, page_size, table_out, table_width);
  DISTIE_LAUNCH_CHECK();
  return 0;
}

DISTIE_PACKED(distie_rows_write)
DISTIE_PACKED(distie_rows_read)
DISTIE_PACKED(distie_rows_table)
