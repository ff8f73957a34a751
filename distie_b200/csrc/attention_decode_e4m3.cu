// Split-KV attention of single tokens over an 8-bit cache on the tensor cores (heads of 64 and 128, 16-bit queries).
//
//   score_j = s^k_j (q . n^k_j) * scale,   out = sum_j p_j s^v_j n^v_j / sum_j p_j
//
// with n the e4m3 numbers of a row and s its scale.  Decoding reads every cached row once, here half the bytes of a 16-bit
// cache, so the instructions between the bytes and the products are what there is to save:
//
//   grid   (token, kv head * chunks of up to 16 query heads, split)
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
// Scales: s^k multiplies the finished score.  s^v cannot ride on V without rounding it; p_j s^v_j is taken as one exponential,
// exp2(score_j + log2 s^v_j - m'), with a running maximum m' of its own beside the softmax's, so the weights that the second
// product gets in float16 have a largest element of 1 however the scales differ, and are off by at most 2^-11 of
// themselves (or of 2^-14).  Sums and maxima are float32.  The warps, and with several splits the CTAs, are merged in the
// softmax's units: inside the cluster up to 8 splits, by a second kernel beyond.
#include <cuda_fp16.h>

#include "cached_rows.cuh"
#include "packed.h"

namespace distie {

constexpr int kDecWarps = 4;
constexpr int kDecKeys = 32;      // keys of a group
constexpr int kDecPages = 1024;   // page ids of a split that are kept in shared memory
constexpr int kDecClusterSplits = 8;

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

template <int D>
__device__ __forceinline__ uint32_t dec_offset(int row, int piece) {  // of a 16-byte piece of a row: free of bank conflicts by 8 rows
  return (uint32_t)(row * D + ((D == 128 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3)) << 4));
}

// PAGE16: the page size is a power of two from 16 on, so 16 keys from a multiple of 16 on lie in one page.
template <int D, int STAGES, int NH, bool PAGE16>
__global__ void __launch_bounds__(kDecWarps * 32, NH == 1 ? 3 : 2)
attention_decode_e4m3_kernel(const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride, QueryRows rows,
                             CachePages cache, Partials parts, int head_chunks, int cluster_merge, int* __restrict__ error) {
  constexpr int MT = D / 16;                  // dim tiles of O^T, reduction steps of S^T, 16-byte pieces of a row
  constexpr int TILE = kDecKeys * D;          // bytes of a K or V tile
  constexpr int STAGE = 2 * TILE + 2 * kDecKeys * 4;
  constexpr int RPI = 32 / MT;                // rows that one copy instruction of the warp covers
  extern __shared__ __align__(128) unsigned char dyn[];
  // The ring [warp][stage][K | V | scales of K | of V]; behind the main loop the merge areas.
  float(*sh_o)[NH * 8][D + 1] = reinterpret_cast<float(*)[NH * 8][D + 1]>(dyn);
  float(*cl_o)[D] = reinterpret_cast<float(*)[D]>(dyn + kDecWarps * NH * 8 * (D + 1) * sizeof(float));
  __shared__ float sh_m[kDecWarps][NH * 8], sh_l[kDecWarps][NH * 8], sh_f[kDecWarps][NH * 8];
  __shared__ float cl_m[NH * 8], cl_l[NH * 8];
  __shared__ int sh_pages[kDecPages];

  grid_dependency_release();
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
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(dyn) + (uint32_t)warp * STAGES * STAGE;
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
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(warp + s * kDecWarps, s);

  // B fragments of S^T: head g of a column tile, dims 16 ks + 4 c .. + 3, times the head's power of two.
  uint32_t qb[NH][MT][2];
  float times[NH][2];  // what turns the raw products of columns 2 c and 2 c + 1 into scores, before the keys' scales
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
    const int hd = nh * 8 + g;
    float x[MT][4], most = 0.f;
#pragma unroll
    for (int ks = 0; ks < MT; ++ks) {
      // (columns behind the last head are nobody's: copies of it, so that no load hangs on a branch)
      const float4 v = load4_cg(q + (size_t)t * q_stride + (size_t)(head0 + min(hd, heads_here - 1)) * D + 16 * ks + 4 * c);
      x[ks][0] = v.x; x[ks][1] = v.y; x[ks][2] = v.z; x[ks][3] = v.w;
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
  float col_max[NH][2], col_sum[NH][2], out_max[NH][2];
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[nh][i][r] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      col_max[nh][e] = out_max[nh][e] = -INFINITY;
      col_sum[nh][e] = 0.f;
    }
  }
  const int lm_mat = lane >> 3, lm_row = lane & 7;
  int stage = 0;
  for (int grp = warp; grp < groups; grp += kDecWarps) {
    const bool in_window = grp < window_groups;
    const int base = in_window ? lo16 + grp * kDecKeys : (grp - window_groups) * kDecKeys;
    const int lo_key = in_window ? lo : 0, hi_key = in_window ? hi : kept - 1;
    issue(grp + (STAGES - 1) * kDecWarps, (stage + STAGES - 1) % STAGES);  // an empty group past the end
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    __syncwarp();
    const uint32_t k_tile = ring + (uint32_t)stage * STAGE, v_tile = k_tile + TILE;
    const float* scales = reinterpret_cast<const float*>(dyn + (size_t)warp * STAGES * STAGE + (size_t)stage * STAGE + 2 * TILE);
    stage = (stage + 1) % STAGES;

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
    float ks_s[RK], vs_log[RK];
    bool keep[RK];
    const bool edge = base < lo_key || base + kDecKeys - 1 > hi_key;
#pragma unroll
    for (int i = 0; i < RK; ++i) {
      ks_s[i] = scales[8 * i + g];
      vs_log[i] = dec_log2(scales[kDecKeys + 8 * i + g]);
      keep[i] = !edge || (base + 8 * i + g >= lo_key && base + 8 * i + g <= hi_key);
    }
    uint32_t pb[kDecKeys / 16][NH][2];
    float corr[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      float w[RK][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[RK], m = -INFINITY, mo = -INFINITY;
#pragma unroll
        for (int i = 0; i < RK; ++i) {
          float s = st[i >> 1][nh][(i & 1) * 2 + e] * (ks_s[i] * times[nh][e]);
          if (rows.extras.cap > 0.f)  // cap * tanh, by its exponential: off by 2^-22 of the cap
            s = rows.extras.cap * 1.4426950408889634f * (1.f - __fdividef(2.f, dec_exp2(s * 2.8853900817779268f) + 1.f));
          x[i] = keep[i] ? s : -INFINITY;
          w[i][e] = keep[i] ? s + vs_log[i] : -INFINITY;
          m = fmaxf(m, x[i]);
          mo = fmaxf(mo, w[i][e]);
        }
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          mo = fmaxf(mo, __shfl_xor_sync(0xffffffffu, mo, d));
        }
        m = fmaxf(col_max[nh][e], m);
        mo = fmaxf(out_max[nh][e], mo);
        const float shift = m == -INFINITY ? 0.f : m, out_shift = mo == -INFINITY ? 0.f : mo;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < RK; ++i) {
          sum += dec_exp2(x[i] - shift);
          w[i][e] = dec_exp2(w[i][e] - out_shift);
        }
        col_sum[nh][e] = col_sum[nh][e] * dec_exp2(col_max[nh][e] - shift) + sum;  // (exp2(-inf) is 0)
        corr[nh][e] = dec_exp2(out_max[nh][e] - out_shift);
        col_max[nh][e] = m;
        out_max[nh][e] = mo;
      }
#pragma unroll
      for (int sub = 0; sub < kDecKeys / 16; ++sub) {
        pb[sub][nh][0] = dec_movmatrix(pack_half(w[2 * sub][0], w[2 * sub][1]));
        pb[sub][nh][1] = dec_movmatrix(pack_half(w[2 * sub + 1][0], w[2 * sub + 1][1]));
      }
    }
    // ---- O^T = O^T * corr + V^T P^T --------------------------------------------------------------------------------
    {
      const int key = lm_row + 8 * (lm_mat & 1);
#pragma unroll
      for (int mt = 0; mt < MT; mt += 2) {
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            o[nh][mt + u][0] *= corr[nh][0]; o[nh][mt + u][1] *= corr[nh][1];
            o[nh][mt + u][2] *= corr[nh][0]; o[nh][mt + u][3] *= corr[nh][1];
          }
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
      for (int mt = 0; mt < MT; ++mt) {
        sh_o[warp][hd][16 * mt + 2 * g] = o[nh][mt][e];
        sh_o[warp][hd][16 * mt + 2 * g + 1] = o[nh][mt][e + 2];
      }
    }
  __syncthreads();
  for (int idx = threadIdx.x; idx < heads_here * D; idx += kDecWarps * 32) {
    const int hd = idx / D, e = idx % D;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) m_all = fmaxf(m_all, sh_m[w][hd]);
    const float shift = m_all == -INFINITY ? 0.f : m_all;
    float l_all = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      // (a warp without a key has a sum of 0; one whose scores are all NaN a sum of NaN, and both have no maximum)
      const float l = sh_l[w][hd], weight = sh_m[w][hd] == -INFINITY ? l : exp2f(sh_m[w][hd] - shift);
      l_all += l * weight;
      acc += sh_o[w][hd][e] * (sh_f[w][hd] == -INFINITY ? l - l : exp2f(sh_f[w][hd] - shift));
    }
    const int head = head0 + hd;
    if (num_splits == 1) {
      const float inv = rows.extras.sink ? sink_inverse_log2(m_all, l_all, rows.extras.sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
      out[(size_t)t * out_stride + (size_t)head * D + e] = __float2bfloat16_rn(acc * inv);
    } else if (cluster_merge) {
      cl_o[hd][e] = acc;
      if (e == 0) { cl_m[hd] = m_all; cl_l[hd] = l_all; }
    } else {
      const size_t row = ((size_t)t * rows.num_heads + head) * num_splits + split;
      parts.o[row * D + e] = acc;
      if (e == 0) {
        parts.ml[row * 2] = m_all;
        parts.ml[row * 2 + 1] = l_all;
      }
    }
  }
  if (num_splits > 1 && cluster_merge) {
    // The splits of a (token, head chunk) are the CTAs of one cluster: each combines its share of the output elements from
    // every CTA's shared memory, splits in order.
    cluster_barrier();
    const int total = heads_here * D, part = (total + num_splits - 1) / num_splits;
    const int end = min(total, (split + 1) * part);
    for (int idx = split * part + threadIdx.x; idx < end; idx += kDecWarps * 32) {
      const int hd = idx / D, e = idx % D;
      float ms[kDecClusterSplits], ls[kDecClusterSplits], os[kDecClusterSplits];
#pragma unroll
      for (int s = 0; s < kDecClusterSplits; ++s) {  // all loads from the other CTAs together
        const bool there = s < num_splits;
        ms[s] = there ? cluster_load(&cl_m[hd], s) : -INFINITY;
        ls[s] = there ? cluster_load(&cl_l[hd], s) : 0.f;
        os[s] = there ? cluster_load(&cl_o[hd][e], s) : 0.f;
      }
      float m_all = -INFINITY;
#pragma unroll
      for (int s = 0; s < kDecClusterSplits; ++s) m_all = fmaxf(m_all, ms[s]);
      float l_all = 0.f, acc = 0.f;
#pragma unroll
      for (int s = 0; s < kDecClusterSplits; ++s) {
        const float weight = ms[s] == -INFINITY ? ls[s] : exp2f(ms[s] - m_all);
        l_all += ls[s] * weight;
        acc += os[s] * weight;
      }
      const int head = head0 + hd;
      const float inv = rows.extras.sink ? sink_inverse_log2(m_all, l_all, rows.extras.sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
      out[(size_t)t * out_stride + (size_t)head * D + e] = __float2bfloat16_rn(acc * inv);
    }
    cluster_barrier_exit();  // no CTA leaves while another may still read its shared memory
  }
}

template <int D, int STAGES, int NH, bool PAGE16>
static cudaError_t launch_decode(const dim3& grid, const __nv_bfloat16* q, int q_stride, __nv_bfloat16* out, int out_stride, const QueryRows& rows,
                                 const CachePages& cache, const Partials& parts, int head_chunks, int cluster_merge, int* error, cudaStream_t stream) {
  constexpr size_t ring = (size_t)kDecWarps * STAGES * (2 * kDecKeys * D + 2 * kDecKeys * 4);
  constexpr size_t merge = (size_t)kDecWarps * NH * 8 * (D + 1) * sizeof(float) + (size_t)NH * 8 * D * sizeof(float);
  constexpr size_t shared = ring > merge ? ring : merge;
  auto kernel = attention_decode_e4m3_kernel<D, STAGES, NH, PAGE16>;
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
// alike (else DISTIE_ERR_UNSUPPORTED, like rows that are not 8-byte aligned).  scratch: distie_attention_rows_scratch_floats, for more than 8 splits.
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
  const QueryRows rows{positions, token_seq, seq_seat, nullptr, nullptr, 1, tokens, group, num_heads, window, chunk, keep_first,
                       scale * 1.4426950408889634f, make_score_extras(scale, softcap, sink)};
  const Partials parts{scratch, scratch ? scratch + (size_t)tokens * num_heads * splits * head_dim : nullptr, splits};
  const int cluster_merge = splits > 1 && splits <= kDecClusterSplits;
  const dim3 grid(tokens, num_kv_heads * chunks, splits);
  const bool page16 = cache.page_shift >= 4;
  cudaError_t err;
#define DISTIE_DECODE_E4M3(D, NH)                                                                                                       \
  err = page16 ? launch_decode<D, 2, NH, true>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts,   \
                                               chunks, cluster_merge, error, stream)                                                     \
               : launch_decode<D, 2, NH, false>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts,  \
                                                chunks, cluster_merge, error, stream)
  if (head_dim == 64) {
    if (group <= 8) DISTIE_DECODE_E4M3(64, 1); else DISTIE_DECODE_E4M3(64, 2);
  } else {
    if (group <= 8) DISTIE_DECODE_E4M3(128, 1); else DISTIE_DECODE_E4M3(128, 2);
  }
#undef DISTIE_DECODE_E4M3
  if (err != cudaSuccess) return (int)err;
  if (splits > 1 && !cluster_merge) return rows_merge_bf16(parts, out, out_stride, tokens, num_heads, head_dim, sink, stream);
  return 0;
}

DISTIE_PACKED(distie_attention_decode_e4m3)
