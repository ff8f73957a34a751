// Split-KV attention of single tokens over an 8-bit cache on the tensor cores (heads of 64 and 128, 16-bit queries).
//
//   score_j = s^k_j (q . n^k_j) * scale,   out = sum_j p_j s^v_j n^v_j / sum_j p_j
//
// with n the e4m3 numbers of a row and s its scale.  Decoding reads every cached row once, here half the bytes of a 16-bit
// cache, so the instructions between the bytes and the products are what there is to save:
//
//   grid   (token, kv head * chunks of up to 16 query heads, split); how many splits: decode_splits in kernels/cached.py
//   block  4 warps; a warp takes groups of 32 keys of the split in turn, through a ring of its own in shared memory (cp.async)
//   S^T    16 keys are the rows of mma.m16n8k16, up to 8 (or 2 x 8) heads the columns, head_dim the reduction
//   O^T    16 dims are the rows, the heads the columns, 16 keys the reduction
//
// The numbers become float16 in registers, which holds every e4m3 number exactly (one conversion per two numbers).  The order
// of dims within a product's reduction, and of dims among its rows, is free: a lane takes the four neighbouring dims that
// ldmatrix hands it as they lie, and q is laid out to match; of V, transposed on the way in, it gets two keys of two dims,
// and one byte permutation makes them two pairs of keys.  q is multiplied by a power of two per head that brings its largest
// element to [1, 2), so that float16 holds it exactly down to 2^-24 of that.
//
// Scales: s^k multiplies the finished score.  s^v cannot ride on V without rounding it; p_j s^v_j goes into the second product
// in float16, in units of a running maximum m' of its own beside the softmax's m: (p_j s^v_j) 2^(m - m'), however the scales
// differ at most a few, and off by at most 2^-11 of itself (or of 2^-14); p_j below 2^-126 is 0 whatever its value's scale.  Both maxima are whole numbers, rounded down (what they
// scale, they scale exactly), and are not searched for in every group, only in a head's first and where weights outgrow the ones in
// use: no shuffles and no correction of O in most groups.  Sums and maxima are float32.  The warps, and with several splits the
// CTAs, are merged in the softmax's units: inside the cluster up to 8 splits, where every CTA sends its sums to the one that puts
// them together (no CTA reads another's memory, none waits to leave), by a second kernel beyond.
//
// What bounds it: with many long requests the bytes and the requests' uneven lengths (13 of 20,000 to 30,011 keys, 8 key heads of
// 128: 634 MB in 130 us, 4.9 TB/s); with heads of 64 the instructions (48 requests of up to 4,099 keys, 8 key heads: 162 MB in 45 us
// inside the kernel; 420 instructions a warp and group, 181 on the ALU pipe at half rate); with few keys a CTA's start
// (positions, seat, page ids, then q and the first rows: 5,000 cycles) and end (merge 1,200, cluster 3,500).  What was tried
// and took as long or longer: rings of 3, 4 and 6 groups and CTAs of 8 warps (fewer CTAs fit an SM), boxes of 16 rows by the copy
// engine in place of cp.async.
#include <cuda_fp16.h>

#include "cached_rows.cuh"
#include "packed.h"

namespace distie {

constexpr int kDecWarps = 4;
constexpr int kDecKeys = 32;      // keys of a group
constexpr int kDecStages = 2;     // groups of a warp's ring
constexpr int kDecPages = 992;    // page ids of a split that are kept in shared memory (so many, that three CTAs fit an SM)
constexpr int kDecClusterSplits = 8;
constexpr float kDecMostSum = 1073741824.f, kDecMostWeight = 16384.f;  // of a lane's four weights of a head

__device__ __forceinline__ void dec_copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void dec_copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dec_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void dec_ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t dec_movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// The two halves of four e4m3 numbers, as float16 pairs.
__device__ __forceinline__ uint32_t low_pair(uint32_t x) { return e4m3x2_to_half2((uint16_t)(x & 0xffffu)); }
__device__ __forceinline__ uint32_t high_pair(uint32_t x) { return e4m3x2_to_half2((uint16_t)(x >> 16)); }
__device__ __forceinline__ float dec_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float dec_log2(float x) {  // of a positive number or 0, subnormal ones included
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Into the shared memory of CTA `rank` of the cluster, where `local` lies in this one's.
__device__ __forceinline__ void cluster_store(float* local, uint32_t rank, float v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}
__device__ __forceinline__ void cluster_store(float* local, uint32_t rank, const float4& v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void store_row4(__nv_bfloat16* to, const float4& v) {  // (rows of the output may lie at any stride)
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
  to[0] = lo.x; to[1] = lo.y; to[2] = hi.x; to[3] = hi.y;
}

template <int D>
__device__ __forceinline__ uint32_t dec_offset(int row, int piece) {  // of a 16-byte piece of a row: free of bank conflicts by 8 rows
  return (uint32_t)(row * D + ((D == 128 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3)) << 4));
}

// PAGE16: the page size is a power of two from 16 on, so 16 keys from a multiple of 16 on lie in one page.
template <int D, int NH, bool PAGE16>
__global__ void __launch_bounds__(kDecWarps * 32, NH == 1 ? 3 : 2)
attention_decode_e4m3_kernel(const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride, QueryRows rows,
                             CachePages cache, Partials parts, int head_chunks, int cluster_merge, int* __restrict__ error) {
  constexpr int MT = D / 16;                  // dim tiles of O^T, reduction steps of S^T, 16-byte pieces of a row
  constexpr int TILE = kDecKeys * D;          // bytes of a K or V tile
  constexpr int STAGE = 2 * TILE + 2 * kDecKeys * 4;
  constexpr int RPI = 32 / MT;                // rows that one copy instruction of the warp covers
  extern __shared__ __align__(128) unsigned char dyn[];
  // The ring [warp][stage][K | V | scales of K | of V]; behind the main loop the warps' sums.
  constexpr int ROW = D + 8;  // (free of bank conflicts where the warps put theirs down)
  float(*sh_o)[NH * 8][ROW] = reinterpret_cast<float(*)[NH * 8][ROW]>(dyn);
  __shared__ float sh_m[kDecWarps][NH * 8], sh_l[kDecWarps][NH * 8], sh_f[kDecWarps][NH * 8];
  // What the CTAs of the cluster send here: their sums of this CTA's share of the output, their maxima and sums of weights.
  __shared__ alignas(16) float from_o[NH * 8 * D + kDecClusterSplits * 4];  // (the last share may be shorter than the others)
  __shared__ float from_m[kDecClusterSplits][NH * 8], from_l[kDecClusterSplits][NH * 8];
  __shared__ int sh_pages[kDecPages];

  grid_dependency_release();
  if (cluster_merge) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (waited for before anything is sent)
  const int t = blockIdx.x, split = blockIdx.z, num_splits = gridDim.z;
  const int kv_head = blockIdx.y / head_chunks, chunk = blockIdx.y % head_chunks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int head0 = kv_head * rows.group + chunk * 16, heads_here = min(NH * 8, rows.group - chunk * 16);

  const int pos = rows.positions[t], seat = rows.seq_seat[rows.token_seq[t]];
  const int* table = cache.block_table + (size_t)seat * cache.table_width;
  const int first = first_visible_key(pos, rows.window, rows.chunk);
  const int first_page = cache.column_of(first), pages = cache.column_of(pos) - first_page + 1;
  const int share = (pages + num_splits - 1) / num_splits, split_page = first_page + split * share;
  const int lo = max(first, split_page * cache.page_size), hi = min(pos, (split_page + share) * cache.page_size - 1);
  for (int i = threadIdx.x; i < min(share, kDecPages); i += kDecWarps * 32)
    sh_pages[i] = split_page + i < cache.table_width ? table[split_page + i] : -1;
  const int lo16 = lo & ~15;
  // Groups of the split's share of the window; behind them, in split 0, those of the first `kept` keys that it has passed.
  const int kept = split == 0 ? min(rows.keep_first, first) : 0;
  const int window_groups = hi >= lo ? (hi - lo16) / kDecKeys + 1 : 0;
  const int groups = window_groups + (kept + kDecKeys - 1) / kDecKeys;
  __syncthreads();
  grid_dependency_wait();  // q and the newest rows come from the kernels before this one

  auto page_of = [&](int key) {
    const int column = cache.column_of(key), i = column - split_page;
    if (i >= 0 && i < min(share, kDecPages)) return sh_pages[i];
    return column < cache.table_width ? table[column] : -1;
  };
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(dyn) + (uint32_t)warp * kDecStages * STAGE;
  const int row0 = lane / MT, piece = lane % MT;
  const uint8_t* k_numbers = reinterpret_cast<const uint8_t*>(cache.k);
  const uint8_t* v_numbers = reinterpret_cast<const uint8_t*>(cache.v);
  auto issue = [&](int grp, int stage) {
    if (grp < groups) {
      const bool in_window = grp < window_groups;
      const int base = in_window ? lo16 + grp * kDecKeys : (grp - window_groups) * kDecKeys;
      const int lo_key = in_window ? lo : 0, hi_key = in_window ? hi : kept - 1;
      const uint32_t k_dst = ring + (uint32_t)stage * STAGE, v_dst = k_dst + TILE, s_dst = v_dst + TILE;
#pragma unroll
      for (int sub = 0; sub < kDecKeys / 16; ++sub) {
        const int key0 = base + 16 * sub;
        if (PAGE16) {
          bool live = key0 <= hi_key && key0 + 15 >= lo_key;
          const int page = live ? page_of(key0) : 0;
          if (live && (page < 0 || page >= cache.num_pages)) {
            if (error) atomicExch(error, 4);
            live = false;
          }
          const size_t at = ((size_t)(live ? page : 0) * cache.num_kv_heads + kv_head) * cache.page_size + (key0 & (cache.page_size - 1));
#pragma unroll
          for (int i = 0; i < 16 / RPI; ++i) {
            const int row = i * RPI + row0;
            const bool ok = live && key0 + row >= lo_key && key0 + row <= hi_key;
            const uint32_t to = dec_offset<D>(16 * sub + row, piece);
            const size_t from = (at + row) * D + piece * 16;
            dec_copy16(k_dst + to, ok ? k_numbers + from : k_numbers, ok ? 16 : 0);
            dec_copy16(v_dst + to, ok ? v_numbers + from : v_numbers, ok ? 16 : 0);
          }
          if (lane < 8) {  // 16 + 16 scales (those of masked keys are read, from within the page, and not used)
            const float* from = (lane < 4 ? cache.k_scale : cache.v_scale) + at + 4 * (lane & 3);
            dec_copy16(s_dst + (lane >> 2) * (kDecKeys * 4) + sub * 64 + (lane & 3) * 16, from, live ? 16 : 0);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16 / RPI; ++i) {
            const int row = i * RPI + row0, key = key0 + row;
            bool ok = key >= lo_key && key <= hi_key;
            size_t at = 0;
            if (ok) {
              const int page = page_of(key);
              if (page < 0 || page >= cache.num_pages) {
                if (error) atomicExch(error, 4);
                ok = false;
              } else {
                at = ((size_t)page * cache.num_kv_heads + kv_head) * cache.page_size + cache.within(key);
              }
            }
            const uint32_t to = dec_offset<D>(16 * sub + row, piece);
            dec_copy16(k_dst + to, ok ? k_numbers + at * D + piece * 16 : k_numbers, ok ? 16 : 0);
            dec_copy16(v_dst + to, ok ? v_numbers + at * D + piece * 16 : v_numbers, ok ? 16 : 0);
            if (piece < 2)
              dec_copy4(s_dst + piece * (kDecKeys * 4) + (16 * sub + row) * 4, ok ? (piece ? cache.v_scale : cache.k_scale) + at : cache.k_scale,
                        ok ? 4 : 0);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // (q is asked for first: behind the copies its loads would queue, and nothing begins without it.  Columns behind the last
  // head are nobody's: copies of it, so that no load hangs on a branch.)
  uint2 q_raw[NH][MT];
#pragma unroll
  for (int nh = 0; nh < NH; ++nh)
#pragma unroll
    for (int ks = 0; ks < MT; ++ks)
      q_raw[nh][ks] = __ldcg(reinterpret_cast<const uint2*>(q + (size_t)t * q_stride + (size_t)(head0 + min(nh * 8 + g, heads_here - 1)) * D + 16 * ks + 4 * c));
#pragma unroll
  for (int s = 0; s < kDecStages - 1; ++s) issue(warp + s * kDecWarps, s);

  // B fragments of S^T: head g of a column tile, dims 16 ks + 4 c .. + 3, times the head's power of two.
  uint32_t qb[NH][MT][2];
  float times[NH][2];  // what turns the raw products of columns 2 c and 2 c + 1 into scores, before the keys' scales
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
    float x[MT][4], most = 0.f;
#pragma unroll
    for (int ks = 0; ks < MT; ++ks) {
      const uint2 raw = q_raw[nh][ks];
      x[ks][0] = __uint_as_float(raw.x << 16); x[ks][1] = __uint_as_float(raw.x & 0xffff0000u);
      x[ks][2] = __uint_as_float(raw.y << 16); x[ks][3] = __uint_as_float(raw.y & 0xffff0000u);
#pragma unroll
      for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[ks][e]));
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int exponent = most > 0.f ? min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126) : 0;
    const float down = __uint_as_float((uint32_t)(127 - exponent) << 23);
#pragma unroll
    for (int ks = 0; ks < MT; ++ks) {
      qb[nh][ks][0] = pack_half(x[ks][0] * down, x[ks][1] * down);
      qb[nh][ks][1] = pack_half(x[ks][2] * down, x[ks][3] * down);
    }
    const float up = __uint_as_float((uint32_t)(127 + exponent) << 23) * (rows.extras.cap > 0.f ? rows.extras.cap_pre : rows.scale_log2);
    times[nh][0] = __shfl_sync(0xffffffffu, up, 8 * c);
    times[nh][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
  }

  float o[NH][MT][4];  // O^T: dims 16 mt + 2 g (+ 1), heads 2 c (+ 1): [dim 2g: head, head + 1 | dim 2g + 1: head, head + 1]
  float col_max[NH][2], col_sum[NH][2], out_max[NH][2], units[NH][2];  // units: 2^(col_max - out_max)
  bool unset[NH];  // a maximum of the lane's two heads is still to be found
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[nh][i][r] = 0.f;
    unset[nh] = true;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      col_max[nh][e] = out_max[nh][e] = -INFINITY;
      col_sum[nh][e] = units[nh][e] = 0.f;
    }
  }
  const float cap = rows.extras.cap * 1.4426950408889634f;
  const int lm_mat = lane >> 3, lm_row = lane & 7;
  int stage = 0;
  for (int grp = warp; grp < groups; grp += kDecWarps) {
    const bool in_window = grp < window_groups;
    const int base = in_window ? lo16 + grp * kDecKeys : (grp - window_groups) * kDecKeys;
    const int lo_key = in_window ? lo : 0, hi_key = in_window ? hi : kept - 1;
    issue(grp + (kDecStages - 1) * kDecWarps, (stage + kDecStages - 1) % kDecStages);  // an empty group past the end
    asm volatile("cp.async.wait_group %0;" ::"n"(kDecStages - 1) : "memory");
    __syncwarp();
    const uint32_t k_tile = ring + (uint32_t)stage * STAGE, v_tile = k_tile + TILE;
    const float* scales = reinterpret_cast<const float*>(dyn + (size_t)warp * kDecStages * STAGE + (size_t)stage * STAGE + 2 * TILE);
    stage = (stage + 1) % kDecStages;

    // ---- S^T: rows = keys 16 sub + g (+ 8), columns = heads 2 c, 2 c + 1 -------------------------------------------
    float st[kDecKeys / 16][NH][4];
#pragma unroll
    for (int sub = 0; sub < kDecKeys / 16; ++sub)
#pragma unroll
      for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[sub][nh][r] = 0.f;
    {
      // Matrices: (keys 0-7, piece ks), (keys 8-15, ks), (keys 0-7, ks + 1), (keys 8-15, ks + 1).
      const int key = lm_row + 8 * (lm_mat & 1);
#pragma unroll
      for (int ks = 0; ks < MT; ks += 2) {
#pragma unroll
        for (int sub = 0; sub < kDecKeys / 16; ++sub) {
          uint32_t a[4];
          dec_ldmatrix(a, k_tile + dec_offset<D>(16 * sub + key, ks + (lm_mat >> 1)));
          const uint32_t a0 = low_pair(a[0]), a1 = low_pair(a[1]), a2 = high_pair(a[0]), a3 = high_pair(a[1]);
          const uint32_t b0 = low_pair(a[2]), b1 = low_pair(a[3]), b2 = high_pair(a[2]), b3 = high_pair(a[3]);
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) {
            mma_f16(st[sub][nh], a0, a1, a2, a3, qb[nh][ks][0], qb[nh][ks][1]);
            mma_f16(st[sub][nh], b0, b1, b2, b3, qb[nh][ks + 1][0], qb[nh][ks + 1][1]);
          }
        }
      }
    }
    // ---- scales, mask, maxima, exponentials ------------------------------------------------------------------------
    constexpr int RK = kDecKeys / 8;  // keys of a lane: g, g + 8, ...
    float ks_s[RK], vs_s[RK];
    bool keep[RK];
    const bool edge = base < lo_key || base + kDecKeys - 1 > hi_key;
#pragma unroll
    for (int i = 0; i < RK; ++i) {
      ks_s[i] = scales[8 * i + g];
      vs_s[i] = scales[kDecKeys + 8 * i + g];
      keep[i] = !edge || (base + 8 * i + g >= lo_key && base + 8 * i + g <= hi_key);
      if (edge && !keep[i]) vs_s[i] = 0.f;  // (a scale that is not finite would outlive its weight of 0)
    }
    uint32_t pb[kDecKeys / 16][NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      float x[RK][2], w[RK][2], sum[2];  // scores less the maximum in use
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float shift = col_max[nh][e] == -INFINITY ? 0.f : col_max[nh][e];
#pragma unroll
        for (int i = 0; i < RK; ++i) {
          const float raw = st[i >> 1][nh][(i & 1) * 2 + e], each = ks_s[i] * times[nh][e];
          // (cap * tanh, by its exponential: off by 2^-22 of the cap)
          const float s = rows.extras.cap > 0.f ? cap * (1.f - __fdividef(2.f, dec_exp2(raw * each * 2.8853900817779268f) + 1.f)) - shift
                                                : fmaf(raw, each, -shift);
          x[i][e] = s;
        }
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < RK; ++i)
          if (!keep[i]) x[i][0] = x[i][1] = -INFINITY;
      }
      bool search = false;
#pragma unroll 1
      while (true) {
        if (search) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = -INFINITY, mo = -INFINITY;
#pragma unroll
            for (int i = 0; i < RK; ++i) {
              m = fmaxf(m, x[i][e]);
              mo = fmaxf(mo, x[i][e] + dec_log2(vs_s[i]));
            }
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) {
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
              mo = fmaxf(mo, __shfl_xor_sync(0xffffffffu, mo, d));
            }
            const float shift = col_max[nh][e] == -INFINITY ? 0.f : col_max[nh][e];
            const float o_new = fmaxf(out_max[nh][e], shift + floorf(mo)), m_new = fmaxf(col_max[nh][e], shift + floorf(m));
            const float corr = o_new > out_max[nh][e] ? dec_exp2(out_max[nh][e] - o_new) : 1.f;  // (exp2(-inf) is 0)
            if (m_new > col_max[nh][e]) {
              col_sum[nh][e] *= dec_exp2(col_max[nh][e] - m_new);
#pragma unroll
              for (int i = 0; i < RK; ++i) x[i][e] -= m_new - shift;
            }
            col_max[nh][e] = m_new;
            out_max[nh][e] = o_new;
            // (2^(m - m') outgrows float32 only where every value so far is below 2^-126; those weights are 0.  Weight times scale
            // comes first in the products below: scale times 2^(m - m') can be infinite beside a weight of 0)
            units[nh][e] = o_new == -INFINITY ? 0.f : dec_exp2(fminf((m_new == -INFINITY ? 0.f : m_new) - o_new, 126.f));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              o[nh][mt][e] *= corr;
              o[nh][mt][e + 2] *= corr;
            }
          }
          unset[nh] = col_max[nh][0] == -INFINITY || col_max[nh][1] == -INFINITY || out_max[nh][0] == -INFINITY || out_max[nh][1] == -INFINITY;
          __syncwarp();
        }
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float weights = 0.f;
          sum[e] = 0.f;
#pragma unroll
          for (int i = 0; i < RK; ++i) {
            const float p = dec_exp2(x[i][e]);
            sum[e] += p;
            w[i][e] = (p * vs_s[i]) * units[nh][e];
            weights += w[i][e];
          }
          most = fmaxf(most, fmaxf(weights, sum[e] * (kDecMostWeight / kDecMostSum)));
        }
        if (search || !__any_sync(0xffffffffu, unset[nh] || most > kDecMostWeight)) break;
        search = true;
      }
      col_sum[nh][0] += sum[0];
      col_sum[nh][1] += sum[1];
#pragma unroll
      for (int sub = 0; sub < kDecKeys / 16; ++sub) {
        pb[sub][nh][0] = dec_movmatrix(pack_half(w[2 * sub][0], w[2 * sub][1]));
        pb[sub][nh][1] = dec_movmatrix(pack_half(w[2 * sub + 1][0], w[2 * sub + 1][1]));
      }
    }
    // ---- O^T += V^T P^T --------------------------------------------------------------------------------
    {
      const int key = lm_row + 8 * (lm_mat & 1);
#pragma unroll
      for (int mt = 0; mt < MT; mt += 2) {
#pragma unroll
        for (int sub = 0; sub < kDecKeys / 16; ++sub) {
          uint32_t a[4];
          dec_ldmatrix_trans(a, v_tile + dec_offset<D>(16 * sub + key, mt + (lm_mat >> 1)));
#pragma unroll
          for (int u = 0; u < 2; ++u) {  // a lane's four numbers: two keys of two dims; dims apart, keys together
            const uint32_t early = __byte_perm(a[2 * u], 0, 0x3120), late = __byte_perm(a[2 * u + 1], 0, 0x3120);
            const uint32_t a0 = low_pair(early), a1 = high_pair(early), a2 = low_pair(late), a3 = high_pair(late);
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) mma_f16(o[nh][mt + u], a0, a1, a2, a3, pb[sub][nh][0], pb[sub][nh][1]);
          }
        }
      }
    }
  }

  // ---- merge the warps, in units of the softmax's maximum ----------------------------------------------------------
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the ring is done with: its memory becomes the merge area
#pragma unroll
  for (int nh = 0; nh < NH; ++nh)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = col_sum[nh][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int hd = nh * 8 + 2 * c + e;
      if (g == 0) {
        sh_m[warp][hd] = col_max[nh][e];
        sh_l[warp][hd] = l;
        sh_f[warp][hd] = out_max[nh][e];
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<float2*>(&sh_o[warp][hd][16 * mt + 2 * g]) = make_float2(o[nh][mt][e], o[nh][mt][e + 2]);
    }
  __syncthreads();
  if (threadIdx.x < heads_here) {  // a head's maximum and sum, and what a warp's sum of values counts
    const int hd = threadIdx.x;
    float m_all = -INFINITY, l_all = 0.f, factor[kDecWarps];
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) m_all = fmaxf(m_all, sh_m[w][hd]);
    const float shift = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      // (a warp without a key has a sum of 0; one whose scores are all NaN a sum of NaN, and both have no maximum)
      const float l = sh_l[w][hd];
      l_all += l * (sh_m[w][hd] == -INFINITY ? l : dec_exp2(sh_m[w][hd] - shift));
      factor[w] = sh_f[w][hd] == -INFINITY ? l - l : dec_exp2(sh_f[w][hd] - shift);
    }
    const int head = head0 + hd;
    float inv = 1.f;
    if (num_splits == 1) inv = rows.extras.sink ? sink_inverse_log2(m_all, l_all, rows.extras.sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) sh_f[w][hd] = factor[w] * inv;
    if (cluster_merge) {
      sh_m[0][hd] = m_all;
      sh_l[0][hd] = l_all;
    } else if (num_splits > 1) {
      const size_t row = ((size_t)t * rows.num_heads + head) * num_splits + split;
      parts.ml[row * 2] = m_all;
      parts.ml[row * 2 + 1] = l_all;
    }
  }
  if (cluster_merge) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all CTAs of the cluster have begun
  __syncthreads();
  // Of the cluster, CTA s puts together the part4 pieces of 4 elements from s * part4 on.
  const int total4 = heads_here * (D / 4), part4 = (total4 + num_splits - 1) / num_splits;
  if (cluster_merge)
    for (int i = threadIdx.x; i < num_splits * heads_here; i += kDecWarps * 32) {
      const int hd = i % heads_here, to = i / heads_here;
      cluster_store(&from_m[split][hd], to, sh_m[0][hd]);
      cluster_store(&from_l[split][hd], to, sh_l[0][hd]);
    }
  for (int i = threadIdx.x; i < total4; i += kDecWarps * 32) {
    const int hd = i / (D / 4), e = i % (D / 4) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(&sh_o[w][hd][e]);
      const float f = sh_f[w][hd];
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    }
    if (num_splits == 1) {
      store_row4(out + (size_t)t * out_stride + (size_t)(head0 + hd) * D + e, acc);
    } else if (cluster_merge) {
      const int to = i / part4;
      cluster_store(&from_o[(split * part4 + i - to * part4) * 4], to, acc);
    } else {
      store4(parts.o + (((size_t)t * rows.num_heads + head0 + hd) * num_splits + split) * D + e, acc);
    }
  }
  if (cluster_merge) {
    cluster_barrier();  // everything has arrived
    for (int i = threadIdx.x; i < min(part4, total4 - split * part4); i += kDecWarps * 32) {
      const int hd = (split * part4 + i) / (D / 4), e = (split * part4 + i) % (D / 4) * 4, head = head0 + hd;
      float m_all = -INFINITY, l_all = 0.f;
      for (int s = 0; s < num_splits; ++s) m_all = fmaxf(m_all, from_m[s][hd]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < num_splits; ++s) {  // splits in order
        const float l = from_l[s][hd], weight = from_m[s][hd] == -INFINITY ? l : dec_exp2(from_m[s][hd] - m_all);
        const float4 v = *reinterpret_cast<const float4*>(&from_o[(s * part4 + i) * 4]);
        l_all += l * weight;
        acc.x += v.x * weight; acc.y += v.y * weight; acc.z += v.z * weight; acc.w += v.w * weight;
      }
      const float inv = rows.extras.sink ? sink_inverse_log2(m_all, l_all, rows.extras.sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
      store_row4(out + (size_t)t * out_stride + (size_t)head * D + e, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
  }
}

template <int D, int NH, bool PAGE16>
static cudaError_t launch_decode(const dim3& grid, const __nv_bfloat16* q, int q_stride, __nv_bfloat16* out, int out_stride, const QueryRows& rows,
                                 const CachePages& cache, const Partials& parts, int head_chunks, int cluster_merge, int* error, cudaStream_t stream) {
  constexpr size_t ring = (size_t)kDecWarps * kDecStages * (2 * kDecKeys * D + 2 * kDecKeys * 4);
  constexpr size_t merge = (size_t)kDecWarps * NH * 8 * (D + 8) * sizeof(float);
  constexpr size_t shared = ring > merge ? ring : merge;
  auto kernel = attention_decode_e4m3_kernel<D, NH, PAGE16>;
  if (shared > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
    if (err != cudaSuccess) return err;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(kDecWarps * 32);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  int count = 0;
  // Scales of pages that 16 keys do not fit are copied through L1, which a kernel that starts early could find stale.
  if (PAGE16) {
    attribute[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[count++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster_merge) {
    attribute[count].id = cudaLaunchAttributeClusterDimension;
    attribute[count].val.clusterDim.x = 1;
    attribute[count].val.clusterDim.y = 1;
    attribute[count++].val.clusterDim.z = grid.z;
  }
  config.attrs = attribute;
  config.numAttrs = count;
  return cudaLaunchKernelEx(&config, kernel, q, q_stride, out, out_stride, rows, cache, parts, head_chunks, cluster_merge, error);
}

}  // namespace distie

using namespace distie;

// Single tokens over an 8-bit cache: q [tokens, >= heads * head_dim] and out bfloat16; heads of 64 or 128, keys and values
// alike (else DISTIE_ERR_UNSUPPORTED, like rows that are not 8-byte aligned).  scratch: tokens * heads * splits * (value size + 2) floats, for more than 8 splits.
extern "C" int distie_attention_decode_e4m3(const void* q, int q_stride, void* out, int out_stride, float* scratch, const int* positions,
                                            const int* token_seq, const int* seq_seat, int tokens, const void* k_cache, const void* v_cache,
                                            const float* k_scale, const float* v_scale, const int* block_table, int table_width,
                                            int num_heads, int num_kv_heads, int head_dim, int page_size, int num_pages, int window,
                                            int chunk, int keep_first, float scale, float softcap, const float* sink, int splits,
                                            int* error, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads != 0 || page_size < 1 || table_width < 1 || keep_first < 0 || splits < 1 ||
      splits > 65535 || num_heads > 65535 || (splits > kDecClusterSplits && scratch == nullptr) || k_scale == nullptr || v_scale == nullptr)
    return DISTIE_ERR_ARG;
  if ((head_dim != 64 && head_dim != 128) || (q_stride & 3) || ((uintptr_t)q & 7) ||
      (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15))
    return DISTIE_ERR_UNSUPPORTED;
  const CachePages cache = make_pages(k_cache, v_cache, k_scale, v_scale, block_table, table_width, num_kv_heads, head_dim, head_dim,
                                      page_size, num_pages);
  const int group = num_heads / num_kv_heads, chunks = (group + 15) / 16;
  const QueryRows rows{positions, token_seq, seq_seat, nullptr, nullptr, 1, tokens, tokens, 1, group, num_heads, window, chunk, keep_first,
                       scale * 1.4426950408889634f, make_score_extras(scale, softcap, sink)};
  const Partials parts{scratch, scratch ? scratch + (size_t)tokens * num_heads * splits * head_dim : nullptr, splits};
  const int cluster_merge = splits > 1 && splits <= kDecClusterSplits;
  const dim3 grid(tokens, num_kv_heads * chunks, splits);
  const bool page16 = cache.page_shift >= 4;
  cudaError_t err;
#define DISTIE_DECODE_E4M3(D, NH)                                                                                                       \
  err = page16 ? launch_decode<D, NH, true>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts,   \
                                               chunks, cluster_merge, error, stream)                                                     \
               : launch_decode<D, NH, false>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts,  \
                                                chunks, cluster_merge, error, stream)
  if (head_dim == 64) {
    if (group <= 8) DISTIE_DECODE_E4M3(64, 1); else DISTIE_DECODE_E4M3(64, 2);
  } else {
    if (group <= 8) DISTIE_DECODE_E4M3(128, 1); else DISTIE_DECODE_E4M3(128, 2);
  }
#undef DISTIE_DECODE_E4M3
  if (err != cudaSuccess) return (int)err;
  if (splits > 1 && !cluster_merge) return rows_merge_bf16(parts, rows, out, out_stride, head_dim, stream);
  return 0;
}

DISTIE_PACKED(distie_attention_decode_e4m3)
