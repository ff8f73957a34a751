// Attention of drafted tokens over the paged cache on the 5th-generation tensor cores: 16-bit queries, a cache in 16 or 8
// bits, heads of 64 and 128.
//
// The new tokens of a request see the same cached keys, so their rows share one pass over them: row r of a request and kv
// head is head r % group of new token r / group, and a CTA takes up to 128 rows and a share of the keys in blocks of 128.
//
//   S = Q K^T        tcgen05.mma, M = 128 rows, N = 128 keys; S in tensor memory, two buffers of 128 columns
//   P = softmax      eight warps in two groups of four: group 0 owns keys 0..63 of every block, group 1 keys 64..127, a thread
//                    per row in each, two softmax streams that meet at the end.  P goes back over the group's columns of S
//                    as 16-bit numbers, two keys to a column.  Warps whose rows are all empty take no part.
//   O_g += P_g V_g   tcgen05.mma with P as the A operand straight from tensor memory
//
// K and V: a warp each asks the copy engine for the rows of a block, page by page, as soon as a stage is free: of a 16-bit cache
// with pages of 8, 16, ..., 128 rows they land swizzled, as the products read them; else they land packed (the rows of a page
// and kv head are one run of memory), and four warps, 32 keys each, read them into registers and write them back
// swizzled, of an 8-bit cache as float16, which holds every e4m3 number exactly.  (One set of warps for both took 6,600 cycles
// a block, each step waiting for the one before.)  So Q (times a power of two a row, float16), K, P and V are float16 there
// and bfloat16 of a 16-bit cache.  The
// scales of the rows go beside the tiles: s^k multiplies the finished score; the weights of the second product are p s^v over
// a running maximum m' of their own, (p s^v) 2^(m - m'), so that float16 holds the largest of a row near 1 whatever
// the scales.
//
// Masks: a block that lies before every row's new tokens and inside every row's window needs none; the others get 64 bits a
// row and group.  A masked weight is 0, and 0 * (what is not finite) is not 0: in blocks that need masks, values that are not
// finite (of an 8-bit cache: scales) are stored as zeros, and the rows that see them get them back at the end, element by
// element.  Rows of keys that belong to nobody are zeros.
//
// Running maxima are not searched for in every block, only in a row's first and where its weights outgrow the one in use;
// then O, and what P of the block is there already, are read, scaled and written back.  The maxima are whole numbers (rounded down), so
// that scaling is exact.
//
// What bounds it: the softmax warps.  Two trees of 64 new tokens over 16,001 keys (40 heads of 128, 8 key heads, bfloat16): 68 us
// with the joining kernel, 144 CTAs of 44 blocks at 2,200 cycles a block, of which the products take 1,050 and each
// scheduler's 128 exponentials 1,024; over an 8-bit cache 96 us, 3,400 cycles a block (scales read and multiplied, weights summed
// once more for their limit).  Registers decide: 15 warps have 128 each, and a version that keeps 64 scores a thread spills.
// With several shares of the keys, the parts go to scratch in float32 and attention_rows.cu joins them.
//
//   warps 0..7    softmax, end        warp 8   tensor memory, MMA issue        warps 9, 10   copies        warps 11..14   unpacking
//
// Every wait on an mbarrier is bounded; when one runs out the CTA sets the error word to 6 and every role stops at its
// next wait.
#include <cuda_fp16.h>

#include "cached_rows.cuh"
#include "packed.h"
#include "softmax_pairs.cuh"
#include "tcgen05.cuh"

namespace distie {

constexpr int kTreeRows = 128;
constexpr int kTreeKeys = 128;
constexpr int kTreeGroupKeys = 64;
constexpr int kTreeMmaWarp = 8;
constexpr int kTreeCopyWarp = 9;   // of K, and behind it of V
constexpr int kTreeLoadWarp = 11;  // the first of those that unpack
constexpr int kTreeLoaders = 4;
constexpr int kTreeThreads = 32 * 15;
constexpr int kTreeKStages = 2, kTreeVStages = 3, kTreeScaleSlots = 4;
constexpr int kTreeHalf = kTreeRows * 128;  // bytes of one [128 rows x 64 elements] swizzled half tile
constexpr int kTreeMostNodes = 256;
constexpr int kTreePages = 2048;   // page ids of a CTA's share that are kept in shared memory
constexpr float kTreeMostSum = 1073741824.f, kTreeMostWeight = 16384.f;  // of a row's weights of 32 keys

// The blocks of 128 keys that a tile of rows walks: those of the kept first keys, then those from the window's start on.
struct TreeSpan {
  int past, keys;       // cached keys, and all of them
  int oldest, newest;   // oldest key that any row's window holds; oldest one that every row's window holds
  int kept;             // first keys that stay visible before `oldest`
  int kept_blocks, start, blocks;

  __device__ __forceinline__ int key0(int j) const { return j < kept_blocks ? j * kTreeKeys : start + (j - kept_blocks) * kTreeKeys; }
  __device__ __forceinline__ int key_end(int j) const { return j < kept_blocks ? min(kept, start) : keys; }
  // Whether every row of the tile sees every key of the block.
  __device__ __forceinline__ bool whole(int j) const { return j >= whole_from() && j < whole_to(); }
  __device__ __forceinline__ int whole_from() const { return kept_blocks + (max(newest - start, 0) + kTreeKeys - 1) / kTreeKeys; }
  __device__ __forceinline__ int whole_to() const { return kept_blocks + max(past - start, 0) / kTreeKeys; }
};

template <int D>
struct TreeShared {
  alignas(1024) unsigned char q[kTreeRows * D * 2];
  alignas(1024) unsigned char k[kTreeKStages][kTreeKeys * D * 2];
  alignas(1024) unsigned char v[kTreeVStages][kTreeKeys * D * 2];
  float k_scale[kTreeScaleSlots][kTreeKeys];  // of the keys of a block
  float v_scale[kTreeScaleSlots][kTreeKeys];
  float v_log[kTreeScaleSlots][kTreeKeys];    // log2 of it
  float q_times[kTreeRows];                   // what turns a row's raw products into scores, before the keys' scales
  TreeSpan span;              // (here and not in registers: the softmax warps need theirs)
  int row_token[kTreeRows];   // token of a row, -1: no row
  int row_first[kTreeRows];   // its oldest visible key
  int node_position[kTreeMostNodes];
  int pages[kTreePages];
  uint64_t q_full;
  uint64_t k_full[kTreeKStages], k_empty[kTreeKStages];
  uint64_t v_full[kTreeVStages], v_empty[kTreeVStages];
  uint64_t k_landed[kTreeKStages], v_landed[kTreeVStages];  // the copies of a tile
  uint64_t scale_full[kTreeScaleSlots];
  uint64_t s_full[2];
  uint64_t p_full[2][2];  // [group][S buffer]
  uint64_t pv_done[2];    // [group]
  uint64_t merge_ready;
  float row_max[2][kTreeRows], row_sum[2][kTreeRows], row_out[2][kTreeRows];
  uint32_t tmem_base;
  uint32_t failed;
  uint32_t bad;  // a masked block holds a value that is not finite
};

__device__ __forceinline__ uint32_t tree_offset(int row, int piece) {  // of 8 elements of a row in a tile of swizzled halves
  return (uint32_t)((piece >> 3) * kTreeHalf + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {  // whether that phase is over, without waiting
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ float tree_log2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two 16-bit bfloat16 numbers of which some are not finite: those become zeros.
__device__ __forceinline__ uint32_t finite_pair(uint32_t x, bool& bad) {
  uint32_t keep = 0xffffffffu;
  if ((x & 0x7f80u) == 0x7f80u) keep &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) keep &= 0x0000ffffu;
  bad |= keep != 0xffffffffu;
  return x & keep;
}

// Whether the row sees a key.
template <int D>
__device__ __forceinline__ bool tree_seen(const TreeShared<D>& sm, int r, int key, int key_end, const int* bits, int words, int keep_first) {
  const int token = sm.row_token[r];
  if (token < 0 || key >= key_end) return false;
  int place = key;
  if (key >= sm.span.past) {
    const int n = key - sm.span.past;
    if (!((__ldg(bits + (size_t)token * words + (n >> 5)) >> (n & 31)) & 1)) return false;
    place = sm.node_position[n];
  }
  return place >= sm.row_first[r] || place < keep_first;
}
// The keys of [key0, key0 + 64) that the row sees, a bit each.
template <int D>
__device__ __forceinline__ uint64_t tree_seen64(const TreeShared<D>& sm, int r, int key0, int key_end, const int* bits, int words, int keep_first) {
  uint64_t mask = 0;
  const int token = sm.row_token[r], past = sm.span.past;
  if (token < 0) return mask;
  const int first = sm.row_first[r];
  if (first <= past) {  // the window holds all new tokens: two ranges of cached keys, then the row's mask
    // Bits low .. high - 1 of the 64.
    auto range = [](int low, int high) {
      low = min(max(low, 0), 64);
      high = min(max(high, 0), 64);
      if (low >= high) return 0ull;
      return (high == 64 ? ~0ull : (1ull << high) - 1) & ~((1ull << low) - 1);
    };
    const int end = min(past, key_end);
    mask = range(first - key0, end - key0) | range(-key0, min(min(keep_first, first), end) - key0);
    const int cached = min(max(past - key0, 0), 64), there = min(64 - cached, key_end - max(key0, past));
    if (there > 0) {
      const int skip = max(key0 - past, 0), word = skip >> 5, shift = skip & 31;  // new tokens before key0
      auto load = [&](int w) { return w < words ? (uint32_t)__ldg(bits + (size_t)token * words + w) : 0u; };
      const uint32_t w0 = load(word), w1 = load(word + 1), w2 = load(word + 2);
      uint64_t draft = (uint64_t)__funnelshift_r(w0, w1, shift) | ((uint64_t)__funnelshift_r(w1, w2, shift) << 32);
      if (there < 64) draft &= (1ull << there) - 1;
      mask |= draft << cached;  // (cached < 64 here)
    }
  } else {
    for (int i = 0; i < 64; ++i)
      if (tree_seen(sm, r, key0 + i, key_end, bits, words, keep_first)) mask |= 1ull << i;
  }
  return mask;
}
// What the values that are not finite, in blocks block0 .. block1 - 1 that need masks, add to element e of the row's sum.
template <int D, bool E4M3>
__device__ __forceinline__ float tree_not_finite(const TreeShared<D>& sm, int r, int e, int block0, int block1, const CachePages& cache,
                                                 const int* table, int kv_head, const int* bits, int words, int keep_first) {
  float sum = 0.f;
  for (int j = block0; j < block1; ++j) {
    if (sm.span.whole(j)) continue;
    for (int key = sm.span.key0(j); key < sm.span.key0(j) + kTreeKeys; ++key) {
      if (!tree_seen(sm, r, key, sm.span.key_end(j), bits, words, keep_first)) continue;
      const long long at = cache.row_of(table, key, kv_head);
      if (at < 0) continue;
      float v;
      if (E4M3) v = e4m3_to_float(reinterpret_cast<const uint8_t*>(cache.v)[(size_t)at * D + e]) * cache.v_scale[at];
      else v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(cache.v)[(size_t)at * D + e]);
      if (!(fabsf(v) <= 3.402823466e38f)) sum += v;
    }
  }
  return sum;
}

// Four floats of shared memory.  (Volatile: the compiler otherwise keeps a block's scales in registers from one look to the next.)
__device__ __forceinline__ float4 tree_shared4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}

__device__ __forceinline__ void tree_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kTreeThreads, 1)
attention_tree_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, int direct,
                              const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride, QueryRows rows,
                              CachePages cache, Partials parts, int* __restrict__ error) {
  extern __shared__ unsigned char raw_shared[];
  auto& sm = *reinterpret_cast<TreeShared<D>*>((reinterpret_cast<uintptr_t>(raw_shared) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t TMEM_COLS = 512, O_COL = 256;  // S0 | S1 | O of group 0 | O of group 1
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* failed = &sm.failed;

  const int split = blockIdx.z;
  const int tiles = gridDim.x / cache.num_kv_heads, kv_head = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  if (warp == kTreeLoadWarp) {  // (a thousand cycles, while the others wait for the request)
    if (lane == 0) {
      mbar_init(&sm.q_full, kTreeMmaWarp);
      sm.failed = 0;
      sm.bad = 0;
    }
    if (lane < kTreeKStages) {
      mbar_init(&sm.k_full[lane], kTreeLoaders);
      mbar_init(&sm.k_empty[lane], 1);
      mbar_init(&sm.k_landed[lane], 1);
    }
    if (lane < kTreeVStages) {
      mbar_init(&sm.v_full[lane], kTreeLoaders);
      mbar_init(&sm.v_empty[lane], 1);
      mbar_init(&sm.v_landed[lane], 1);
    }
    if (lane < kTreeScaleSlots) mbar_init(&sm.scale_full[lane], kTreeLoaders);
    if (lane < 2) {
      mbar_init(&sm.s_full[lane], 1);
      mbar_init(&sm.pv_done[lane], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const Request request = request_of(rows, blockIdx.y);
  const int row0 = tile * kTreeRows, count = min(kTreeRows, request.nodes * rows.group - row0);
  if (count <= 0) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && split == 0) grid_dependency_wait();  // (some CTA of the grid always waits: kernels end in order)
    return;
  }
  const int active = (count + 31) / 32;  // warps of a softmax group that have rows
  const int* table = cache.block_table + (size_t)request.seat * cache.table_width;

  grid_dependency_release();
  int block0, blocks, column0, columns;
  const bool everything = rows.window == 0 && rows.chunk == 0;  // (no need to look at positions)
  {
    TreeSpan span;
    int low = everything ? 0 : 0x7fffffff, high = 0;
    const int node0 = row0 / rows.group, node1 = (row0 + count - 1) / rows.group;
    for (int n = node0 + lane; n <= node1 && !everything; n += 32) {
      const int first = first_visible_key(rows.positions[request.first + n], rows.window, rows.chunk);
      low = min(low, first);
      high = max(high, first);
    }
#pragma unroll
    for (int d = 16; d >= 1 && !everything; d >>= 1) {
      low = min(low, __shfl_xor_sync(0xffffffffu, low, d));
      high = max(high, __shfl_xor_sync(0xffffffffu, high, d));
    }
    span.past = request.past;
    span.keys = request.past + request.nodes;
    span.oldest = min(low, request.past);  // (all new tokens' keys are walked)
    span.newest = high;
    span.kept = min(rows.keep_first, span.oldest);
    span.kept_blocks = (span.kept + kTreeKeys - 1) / kTreeKeys;
    span.start = span.oldest / kTreeKeys * kTreeKeys;
    span.blocks = span.kept_blocks + (span.keys - span.start + kTreeKeys - 1) / kTreeKeys;
    const int share = (span.blocks + parts.splits - 1) / parts.splits;
    block0 = min(span.blocks, split * share);
    blocks = min(span.blocks, block0 + share) - block0;
    // The page ids of the share's keys from its window's first block on.
    column0 = cache.column_of(span.key0(max(block0, span.kept_blocks)));
    columns = block0 + blocks > span.kept_blocks
                  ? min(kTreePages, cache.column_of(min(span.keys - 1, span.key0(block0 + blocks - 1) + kTreeKeys - 1)) - column0 + 1) : 0;
    if (threadIdx.x == 0) sm.span = span;
  }
  if (blocks == 0) {  // a share without keys: its parts count nothing
    grid_dependency_wait();
    for (int r = warp; r < count; r += kTreeThreads / 32) {
      const int token = request.first + (row0 + r) / rows.group, head = kv_head * rows.group + (row0 + r) % rows.group;
      const size_t at = ((size_t)token * rows.num_heads + head) * parts.splits + split;
      for (int e = lane; e < D; e += 32) parts.o[at * D + e] = 0.f;
      if (lane == 0) {
        parts.ml[2 * at] = -INFINITY;
        parts.ml[2 * at + 1] = 0.f;
      }
    }
    return;
  }

  // Three jobs at once: tensor memory, what is known of the rows, page ids (they wait for one load each).
  if (warp == 0 && lane < 4) mbar_init(&sm.p_full[lane >> 1][lane & 1], active);
  if (warp == 0 && lane == 0) mbar_init(&sm.merge_ready, 2 * active);
  if (warp == kTreeMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (warp >= kTreeCopyWarp)  // (the warps below alone look at them)
    for (int i = threadIdx.x - kTreeCopyWarp * 32; i < columns; i += (kTreeLoaders + 2) * 32)
      sm.pages[i] = column0 + i < cache.table_width ? table[column0 + i] : -1;
  if (warp < kTreeMmaWarp)
    for (int n = threadIdx.x; n < max(kTreeRows, min(request.nodes, kTreeMostNodes)); n += kTreeMmaWarp * 32) {
      if (n < request.nodes) sm.node_position[n] = everything ? 0 : rows.positions[request.first + n];
      if (n < kTreeRows) {
        const int token = n < count ? request.first + (row0 + n) / rows.group : -1;
        sm.row_token[n] = token;
        sm.row_first[n] = token < 0 || everything ? 0 : first_visible_key(rows.positions[token], rows.window, rows.chunk);
      }
    }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const TreeSpan& span = sm.span;
  const int block1 = block0 + blocks;
  const uint32_t tmem = sm.tmem_base;
  grid_dependency_wait();  // q and the newest rows come from the kernels before this one

  if (warp >= kTreeCopyWarp) {
    constexpr int BYTES = E4M3 ? D : 2 * D;  // of a row in the cache
    // Packed rows: those of 32 keys land in the first 32 lines of 128 bytes that these keys will take, rows of 256 bytes in two
    // halves of 16 keys.
    constexpr int FIT = BYTES > 128 ? 16 : 32;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_unless(bar, parity, failed)) != 0; };
    auto page_at = [&](int column) {
      const int index = column - column0;
      return index >= 0 && index < columns ? sm.pages[index] : column < cache.table_width ? __ldg(table + column) : -1;
    };
    auto wanted = [&](int key, int key_end) { return key < key_end && (key >= span.oldest || key < span.kept); };
    bool ok = true;
    if (warp < kTreeLoadWarp) {
      // ---- copies of K or V: a lane a page, in rounds of 32 pages -------------------------------------------------------------
      const bool is_k = warp == kTreeCopyWarp;
      const int stages = is_k ? kTreeKStages : kTreeVStages;
      uint64_t* empty = is_k ? sm.k_empty : sm.v_empty;
      uint64_t* landed = is_k ? sm.k_landed : sm.v_landed;
      const CUtensorMap* map = is_k ? &map_k : &map_v;
      const unsigned char* rows_at = reinterpret_cast<const unsigned char*>(is_k ? cache.k : cache.v);
      int requested = 0, stage = 0, turn = 0;
      for (; requested < blocks; ++requested) {
        const int j = block0 + requested;
        const int key0 = span.key0(j), end = min(key0 + kTreeKeys, span.key_end(j));
        const int first_column = cache.column_of(key0), last_column = end > key0 ? cache.column_of(end - 1) : first_column - 1;
        unsigned char* tile_at = (is_k ? sm.k[0] : sm.v[0]) + (size_t)stage * kTreeKeys * D * 2;
        bool waited = false;
        for (int round = first_column; !waited || round <= last_column; round += 32) {
          // The lane's run of a round: keys from .. to - 1 of its page, wanted ones and what lies between them.
          const int column = round + lane;
          int from = 0, to = 0, page = 0;
          if (column <= last_column) {
            const int page0 = column * cache.page_size;
            from = max(key0, page0);
            to = min(end, page0 + cache.page_size);
            if (from < span.oldest && from >= span.kept) from = span.oldest;  // between the kept keys and the window
            if (from < span.kept && to > span.kept && to <= span.oldest) to = span.kept;
            to = max(to, from);
            if (to > from) page = page_at(column);
            if (page < 0 || page >= cache.num_pages) {
              to = from;
              if (error) atomicExch(error, 8);
            }
          }
          const int bytes = __reduce_add_sync(0xffffffffu, direct ? (to > from ? cache.page_size : 0) : to - from) * BYTES;
          if (!waited && !wait(&empty[stage], turn ^ 1)) { ok = false; break; }
          waited = true;
          if (lane == 0) {
            if (round + 32 > last_column) mbar_expect_tx(&landed[stage], bytes);
            else asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&landed[stage])), "r"(bytes) : "memory");
          }
          __syncwarp();
          if (to > from) {
            const long long row = ((long long)page * cache.num_kv_heads + kv_head) * cache.page_size;
            if (!E4M3 && direct) {  // the whole page
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                tma_load_2d(tile_at + h * kTreeHalf + (column * cache.page_size - key0) * 128, map, &landed[stage], h * 64, (int)row);
            } else {
              for (int at = from; at < to;) {
                const int local = at - key0, stop = min(to, key0 + (local / FIT + 1) * FIT);
                const unsigned char* source = rows_at + (size_t)(row + cache.within(at)) * BYTES;
                const uint32_t target = smem_u32(tile_at) + (local % 32 / FIT) * kTreeHalf + local / 32 * 4096 + local % FIT * BYTES;
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(target), "l"(source),
                             "r"((stop - at) * BYTES), "r"(smem_u32(&landed[stage])) : "memory");
                at = stop;
              }
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        if (++stage == stages) {
          stage = 0;
          turn ^= 1;
        }
      }
      // Copies still on their way must land before the CTA may leave.
      for (int i = max(0, requested - stages); !ok && i < requested; ++i) mbar_wait(&landed[i % stages], (i / stages) & 1);
    } else {
      // ---- unpacking: 32 keys a warp --------------------------------------------------------------------------------------
      constexpr int PPR = BYTES / 16;   // 16-byte pieces of a row
      constexpr int RPI = 32 / PPR;     // rows that the warp reads at a time
      constexpr int PIECES = 32 / RPI;  // of a tile, per lane
      const int row0_mine = (warp - kTreeLoadWarp) * 32, sub_row = lane / PPR, piece = lane % PPR;
      // A tile whose rows have landed (`there`: which of the warp's 32, a bit each): made what the product reads.  `check`: values
      // that are not finite become zeros, and are remembered.
      auto finish = [&](unsigned char* stage, uint32_t there, bool check) {
        if (!E4M3 && direct && !check) return;
        uint4 raw[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int row = i * RPI + sub_row;
          raw[i] = *reinterpret_cast<const uint4*>(stage + (!E4M3 && direct ? tree_offset(row0_mine + row, piece)
                                                                           : row / FIT * kTreeHalf + row0_mine * 128 + row % FIT * BYTES + piece * 16));
        }
        __syncwarp();
        const uint32_t base = smem_u32(stage);
        bool bad = false;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int row = i * RPI + sub_row;
          uint4 x = (there >> row) & 1 ? raw[i] : make_uint4(0u, 0u, 0u, 0u);
          if (E4M3) {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h[2 * e] = e4m3x2_to_half2((uint16_t)(w[e] & 0xffffu));
              h[2 * e + 1] = e4m3x2_to_half2((uint16_t)(w[e] >> 16));
            }
            store_shared16(base + tree_offset(row0_mine + row, 2 * piece), h[0], h[1], h[2], h[3]);
            store_shared16(base + tree_offset(row0_mine + row, 2 * piece + 1), h[4], h[5], h[6], h[7]);
          } else {
            if (check) {
              x.x = finite_pair(x.x, bad);
              x.y = finite_pair(x.y, bad);
              x.z = finite_pair(x.z, bad);
              x.w = finite_pair(x.w, bad);
            }
            store_shared16(base + tree_offset(row0_mine + row, piece), x.x, x.y, x.z, x.w);
          }
        }
        if (bad) atomicExch(&sm.bad, 1u);
      };
      auto ready = [&](uint64_t* bar) {  // this warp's stores are in shared memory, for the tensor cores and for other warps
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };
      // The row of this lane's key of block j among the slot's rows, -1: none.
      auto find = [&](int j) -> long long {
        if (j >= block1) return -1;
        const int key = span.key0(j) + row0_mine + lane;
        if (!wanted(key, span.key_end(j))) return -1;
        const int page = page_at(cache.column_of(key));
        if (page < 0 || page >= cache.num_pages) return -1;
        return ((long long)page * cache.num_kv_heads + kv_head) * cache.page_size + cache.within(key);
      };
      // Scales, a lane per key, one block ahead in registers (of no key: the slot's first row's, never read behind the mask).
      long long at = find(block0);
      float ks = 0.f, vs = 0.f;
      if (E4M3) {
        ks = __ldcg(cache.k_scale + max(at, 0ll));
        vs = __ldcg(cache.v_scale + max(at, 0ll));
      }
      for (int n = 0; n < blocks; ++n) {
        const int k_stage = n % kTreeKStages, v_stage = n % kTreeVStages;
        const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
        if (!wait(&sm.k_landed[k_stage], (n / kTreeKStages) & 1)) { ok = false; break; }
        if (E4M3) {
          // The slot's last scales have been read: the S of two blocks ago, whose stage K has taken, was issued behind the P of
          // two blocks before that.
          const int slot = n % kTreeScaleSlots, key = row0_mine + lane;
          if (!((there >> lane) & 1)) ks = vs = 0.f;
          if (!span.whole(block0 + n) && !(fabsf(vs) <= 3.402823466e38f)) {  // (the weight of who does not see it would not be 0)
            vs = 0.f;
            atomicExch(&sm.bad, 1u);
          }
          sm.k_scale[slot][key] = ks;
          sm.v_scale[slot][key] = vs;
          sm.v_log[slot][key] = tree_log2(vs);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.scale_full[slot]);
        }
        finish(sm.k[k_stage], there, false);
        ready(&sm.k_full[k_stage]);
        at = find(block0 + n + 1);
        if (E4M3) {
          ks = __ldcg(cache.k_scale + max(at, 0ll));
          vs = __ldcg(cache.v_scale + max(at, 0ll));
        }
        if (!wait(&sm.v_landed[v_stage], (n / kTreeVStages) & 1)) { ok = false; break; }
        finish(sm.v[v_stage], there, !span.whole(block0 + n));
        ready(&sm.v_full[v_stage]);
      }
    }
    if (!ok) atomicExch(&sm.failed, 1u);
  } else if (warp == kTreeMmaWarp) {
    // ---- MMA issuer ----------------------------------------------------------------------------------------------------
    if (elect_one()) {
      constexpr uint32_t type = E4M3 ? 0u : (1u << 7) | (1u << 10);  // float16 or bfloat16 operands
      constexpr uint32_t idesc_s = (1u << 4) | type | ((uint32_t)(kTreeKeys >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      const uint64_t q_desc = smem_desc(sm.q);
      bool ok = mbar_wait_unless(&sm.q_full, 0, failed);
      auto issue_s = [&](int n) {
        const int s = n & 1, ks = n % kTreeKStages;
        if (!mbar_wait_unless(&sm.k_full[ks], (n / kTreeKStages) & 1, failed)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t k_desc = smem_desc(sm.k[ks]);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t step = (uint64_t)(((kk >> 2) * kTreeHalf + (kk & 3) * 32) >> 4);
          umma_bf16(tmem + s * kTreeKeys, q_desc + step, k_desc + step, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&sm.k_empty[ks]);
        umma_commit(&sm.s_full[s]);
        return true;
      };
      ok = ok && issue_s(0);
      if (ok && blocks > 1) ok = issue_s(1);
      for (int n = 0; n < blocks && ok; ++n) {
        const int s = n & 1, vs = n % kTreeVStages;
        if (!mbar_wait_unless(&sm.v_full[vs], (n / kTreeVStages) & 1, failed)) { ok = false; break; }
        const uint64_t v_desc = smem_desc_mn(sm.v[vs], kTreeHalf, 1024);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (!mbar_wait_unless(&sm.p_full[g][s], (n >> 1) & 1, failed)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int kk = 0; kk < kTreeGroupKeys / 16; ++kk) {
            const uint64_t v_step = (uint64_t)(((g * kTreeGroupKeys + kk * 16) * 128) >> 4);
            umma_bf16_ts(tmem + O_COL + g * D, tmem + s * kTreeKeys + g * kTreeGroupKeys + kk * 8, v_desc + v_step, idesc_o,
                         (n > 0 || kk > 0) ? 1u : 0u);
          }
          umma_commit(&sm.pv_done[g]);
        }
        if (!ok) break;
        umma_commit(&sm.v_empty[vs]);
        if (n + 2 < blocks) ok = issue_s(n + 2);
      }
      if (!ok) atomicExch(&sm.failed, 1u);
    }
  } else {
    // ---- queries into shared memory: a warp takes 16 rows ---------------------------------------------------------------
    {
      constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;  // lanes of 8 elements to a row; rows that the warp takes at a time
      const float unit_times = rows.extras.cap > 0.f ? rows.extras.cap_pre : rows.scale_log2;
      uint2 x[16 / AT_ONCE][2];
#pragma unroll
      for (int i = 0; i < 16 / AT_ONCE; ++i) {
        const int r = min(warp * 16 + i * AT_ONCE + lane / LANES, count - 1);  // (rows behind the last one are nobody's: copies of it)
        const int token = sm.row_token[r], head = kv_head * rows.group + row0 + r - (token - request.first) * rows.group;
        const __nv_bfloat16* from = q + (size_t)token * q_stride + (size_t)head * D + lane % LANES * 8;
        x[i][0] = __ldcg(reinterpret_cast<const uint2*>(from));
        x[i][1] = __ldcg(reinterpret_cast<const uint2*>(from + 4));
      }
#pragma unroll
      for (int i = 0; i < 16 / AT_ONCE; ++i) {
        const int r = warp * 16 + i * AT_ONCE + lane / LANES;
        uint32_t w[4] = {x[i][0].x, x[i][0].y, x[i][1].x, x[i][1].y};
        if (E4M3) {  // times a power of two that brings the row's largest element to [1, 2): float16 then holds it
          float most = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
#pragma unroll
          for (int d = LANES / 2; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
          const int exponent = most > 0.f ? min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126) : 0;
          const float down = __uint_as_float((uint32_t)(127 - exponent) << 23);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 pair = __floats2half2_rn(__uint_as_float(w[e] << 16) * down, __uint_as_float(w[e] & 0xffff0000u) * down);
            w[e] = *reinterpret_cast<const uint32_t*>(&pair);
          }
          if (lane % LANES == 0) sm.q_times[r] = __uint_as_float((uint32_t)(127 + exponent) << 23) * unit_times;
        }
        store_shared16(smem_u32(sm.q) + tree_offset(r, lane % LANES), w[0], w[1], w[2], w[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full);
    }
    // ---- softmax, correction of O, end: group g owns 64 keys of every block, thread = row ---------------------------------
    const int quadrant = warp & 3, g = warp >> 2, r = quadrant * 32 + lane;
    if (quadrant < active) {
      const uint32_t lane_base = tmem + ((uint32_t)(quadrant * 32) << 16);
      const uint32_t o_addr = lane_base + O_COL + g * D;
      bool ok = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_unless(bar, parity, failed)) != 0; };
      ok = wait_all(&sm.q_full, 0);
      const float times = E4M3 ? sm.q_times[r] : (rows.extras.cap > 0.f ? rows.extras.cap_pre : rows.scale_log2);
      const uint64_t times2 = pair_of(times, times);
      const bool capped = rows.extras.cap > 0.f;
      const float cap = rows.extras.cap * 1.4426950408889634f;
      const int whole0 = span.whole_from(), whole1 = span.whole_to();
      float m_used = -INFINITY, o_used = -INFINITY, l = 0.f;  // o_used: the maximum that P is taken with, of scores with the values' scales
      for (int n = 0; n < blocks && ok; ++n) {
        const int j = block0 + n, s = n & 1, slot = n % kTreeScaleSlots;
        const uint32_t s_addr = lane_base + s * kTreeKeys + g * kTreeGroupKeys;
        const bool whole = j >= whole0 && j < whole1;
        const uint64_t mask = whole ? ~0ull : tree_seen64(sm, r, span.key0(j) + g * kTreeGroupKeys, span.key_end(j), rows.bits, rows.words, rows.keep_first);
        if (E4M3 && !wait_all(&sm.scale_full[slot], (n / kTreeScaleSlots) & 1)) { ok = false; break; }
        if (!wait_all(&sm.s_full[s], (n >> 1) & 1)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t scales = smem_u32(&sm.k_scale[slot][g * kTreeGroupKeys]);
        // 32 keys at a time: 64 scores do not fit a thread's registers beside the rest, and what spills goes to L2 (shared memory
        // leaves L1 next to nothing).  P, two keys a column, takes the columns of scores that have been read.
        uint32_t next[32];
#pragma unroll
        for (int piece = 0; piece < 2; ++piece) {
          uint32_t sv[32];  // scores in base-2 units, less the maximum in use
          if (E4M3 || piece == 0) tmem_load_32(s_addr + piece * 32, next);
          tree_loaded(next);
#pragma unroll
          for (int i = 0; i < 32; ++i) sv[i] = next[i];
          if (!E4M3 && piece == 0) tmem_load_32(s_addr + 32, next);
          const uint32_t bits = (uint32_t)(mask >> (piece * 32));
          const uint32_t k_scale = scales + piece * 128, v_scale = k_scale + (uint32_t)sizeof(sm.k_scale), v_log = v_scale + (uint32_t)sizeof(sm.v_scale);
          float shift = m_used == -INFINITY ? 0.f : m_used;
          const uint64_t less2 = capped ? pair_of(0.f, 0.f) : pair_of(-shift, -shift);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            uint64_t x = pair_of(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), y = pair_of(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
            if (E4M3) {
              const float4 ks = tree_shared4(k_scale + i * 4);
              x = mul_pairs(x, pair_of(ks.x, ks.y));
              y = mul_pairs(y, pair_of(ks.z, ks.w));
            }
            float v[4];
            halves_of(fma_pairs(x, times2, less2), v[0], v[1]);
            halves_of(fma_pairs(y, times2, less2), v[2], v[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sv[i + e] = __float_as_uint(v[e]);
          }
          if (capped) {  // cap * tanh, by its exponential: off by 2^-22 of the cap
#pragma unroll
            for (int i = 0; i < 32; ++i)
              sv[i] = __float_as_uint(cap * (1.f - __fdividef(2.f, exp2_approx(__uint_as_float(sv[i]) * 2.8853900817779268f) + 1.f)) - shift);
          }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((bits >> i) & 1)) sv[i] = 0xff800000u;  // -inf
          }
          // The maxima in use (whole numbers: what they scale, they scale exactly) are raised where a row has none yet, and where
          // its weights outgrow them: the sum of 32 bfloat16 weights may reach 2^30, of float16 ones 2^14.
          bool search = __any_sync(0xffffffffu, (m_used == -INFINITY || (E4M3 && o_used == -INFINITY)) && bits != 0);
          uint32_t packed[16];
          float sum;
#pragma unroll 1
          while (true) {
            if (search) {
              float mx = -INFINITY, ox = -INFINITY;
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                mx = fmaxf(max3(mx, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), fmaxf(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])));
                if (E4M3) {
                  const float4 vl = tree_shared4(v_log + i * 4);
                  ox = fmaxf(max3(ox, __uint_as_float(sv[i]) + vl.x, __uint_as_float(sv[i + 1]) + vl.y),
                             fmaxf(__uint_as_float(sv[i + 2]) + vl.z, __uint_as_float(sv[i + 3]) + vl.w));
                }
              }
              // The maximum for the sum, and the one for O (of a 16-bit cache they are one).
              const float m_new = fmaxf(m_used, shift + floorf(mx));
              float corr = 1.f;
              if (E4M3) {
                const float o_new = fmaxf(o_used, shift + floorf(ox));
                if (o_new > o_used) {
                  corr = exp2_approx(o_used - o_new);
                  o_used = o_new;
                }
              }
              if (m_new > m_used) {
                const float down = exp2_approx(m_used - m_new), less = m_new - shift;
                if (!E4M3) corr = down;
                l *= down;
                m_used = shift = m_new;
#pragma unroll
                for (int i = 0; i < 32; ++i) sv[i] = __float_as_uint(__uint_as_float(sv[i]) - less);
              }
              if ((n > 0 || piece > 0) && __any_sync(0xffffffffu, corr != 1.f)) {
                if (n > 0) {  // the group's O is in use by its product of the block before this one until that has completed
                  if (!wait_all(&sm.pv_done[g], (n - 1) & 1)) { ok = false; break; }
                  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                  for (int c0 = 0; c0 < D; c0 += 16) {
                    tmem_load_16(o_addr + c0, packed);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 16; ++i) packed[i] = __float_as_uint(__uint_as_float(packed[i]) * corr);
                    tmem_store_16(o_addr + c0, packed);
                  }
                }
                if (piece > 0) {  // and the weights of the block's first 32 keys
                  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                  tmem_load_16(s_addr, packed);
                  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                  for (int i = 0; i < 16; ++i) {
                    if (E4M3) {
                      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed[i]));
                      const __half2 pair = __floats2half2_rn(f.x * corr, f.y * corr);
                      packed[i] = *reinterpret_cast<const uint32_t*>(&pair);
                    } else {
                      const __nv_bfloat162 pair = __floats2bfloat162_rn(__uint_as_float(packed[i] << 16) * corr, __uint_as_float(packed[i] & 0xffff0000u) * corr);
                      packed[i] = *reinterpret_cast<const uint32_t*>(&pair);
                    }
                  }
                  tmem_store_16(s_addr, packed);
                }
              }
              __syncwarp();
            }
            // (2^(m - m') outgrows float32 only where every value so far is below 2^-126; those weights are 0)
            const float units = E4M3 && o_used != -INFINITY ? exp2_approx(fminf(shift - o_used, 126.f)) : 0.f;
            const uint64_t units2 = pair_of(units, units);
            uint64_t sum4[4] = {0ull, 0ull, 0ull, 0ull}, weight4[2] = {0ull, 0ull};
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 vs = make_float4(0.f, 0.f, 0.f, 0.f);
              if (E4M3) vs = tree_shared4(v_scale + i * 4);
              const uint64_t scale2[2] = {pair_of(vs.x, vs.y), pair_of(vs.z, vs.w)};
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const uint64_t p = pair_of(exp2_approx(__uint_as_float(sv[i + e])), exp2_approx(__uint_as_float(sv[i + e + 1])));
                uint64_t& total = sum4[((i + e) >> 1) & 3];
                float w0, w1;
                if (E4M3) {
                  total = add_pairs(total, p);
                  const uint64_t w = mul_pairs(mul_pairs(p, scale2[e >> 1]), units2);  // (scale times units can be infinite beside a weight of 0)
                  weight4[e >> 1] = add_pairs(weight4[e >> 1], w);
                  halves_of(w, w0, w1);
                  const __half2 pair = __floats2half2_rn(w0, w1);
                  packed[(i + e) >> 1] = *reinterpret_cast<const uint32_t*>(&pair);
                } else {  // the sum is that of the weights as the product takes them
                  halves_of(p, w0, w1);
                  const __nv_bfloat162 pair = __floats2bfloat162_rn(w0, w1);
                  const uint32_t both = *reinterpret_cast<const uint32_t*>(&pair);
                  packed[(i + e) >> 1] = both;
                  total = add_pairs(total, pair_of(__uint_as_float(both << 16), __uint_as_float(both & 0xffff0000u)));
                }
              }
            }
            float even, odd;
            halves_of(add_pairs(add_pairs(sum4[0], sum4[1]), add_pairs(sum4[2], sum4[3])), even, odd);
            sum = even + odd;
            bool outgrown = sum > kTreeMostSum;
            if (E4M3) {
              halves_of(add_pairs(weight4[0], weight4[1]), even, odd);
              outgrown = outgrown || even + odd > kTreeMostWeight;
            }
            if (search || !__any_sync(0xffffffffu, outgrown)) break;
            search = true;
          }
          if (!ok) break;
          tmem_store_16(s_addr + piece * 16, packed);
          l += sum;
        }
        if (!ok) break;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[g][s]);
      }
      if (!ok) atomicExch(&sm.failed, 1u);
      // ---- end: the two groups' parts of a row at a common maximum -------------------------------------------------------
      sm.row_max[g][r] = m_used;
      sm.row_sum[g][r] = l;
      sm.row_out[g][r] = E4M3 ? o_used : m_used;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.merge_ready);
      if (ok && wait_all(&sm.merge_ready, 0) && wait_all(&sm.pv_done[0], (blocks - 1) & 1) && wait_all(&sm.pv_done[1], (blocks - 1) & 1)) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float m_all = fmaxf(sm.row_max[0][r], sm.row_max[1][r]), at_most = m_all == -INFINITY ? 0.f : m_all;
        float l_all = 0.f, f[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // (no maximum: a sum of 0 without a key, of NaN where every score is NaN)
          const float sum = sm.row_sum[u][r], weight = sm.row_max[u][r] == -INFINITY ? sum : exp2_approx(sm.row_max[u][r] - at_most);
          l_all += sum * weight;
          f[u] = sm.row_out[u][r] == -INFINITY ? sum - sum : exp2_approx(sm.row_out[u][r] - at_most);
        }
        const bool alone = parts.splits == 1, live = r < count;
        // (rows behind the last one: nobody's, and not written)
        const int token = live ? sm.row_token[r] : request.first, head = live ? kv_head * rows.group + row0 + r - (token - request.first) * rows.group : 0;
        float inv = 1.f;
        if (alone && live) inv = rows.extras.sink ? sink_inverse_log2(m_all, l_all, rows.extras.sink[head]) : (l_all == 0.f ? 0.f : 1.f / l_all);
        const float f0 = f[0] * inv, f1 = f[1] * inv;
        constexpr int SIDE = D / 2;  // group g writes columns g * D / 2 ... of the row, from both accumulators
        const size_t part_row = ((size_t)token * rows.num_heads + head) * parts.splits + split;
        // Parts go to scratch by the copy engine, half a row at a time, from rows of shared memory that K and V have left.
        constexpr int PITCH = SIDE * 4 + 16;
        unsigned char* mine = &sm.k[0][0] + ((g * 4 + quadrant) * 32 + lane) * PITCH;
        static_assert(2 * kTreeRows * PITCH <= kTreeKStages * kTreeKeys * D * 2 + kTreeVStages * kTreeKeys * D * 2);
#pragma unroll 1
        for (int c0 = 0; c0 < SIDE; c0 += 16) {
          uint32_t a[16], b[16];
          tmem_load_16(lane_base + O_COL + g * SIDE + c0, a);
          tmem_load_16(lane_base + O_COL + D + g * SIDE + c0, b);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          float y[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(a[i]) * f0 + __uint_as_float(b[i]) * f1;
          if (live && alone) {
            __nv_bfloat16* to = out + (size_t)token * out_stride + (size_t)head * D + g * SIDE + c0;
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              const float part[8] = {y[i], y[i + 1], y[i + 2], y[i + 3], y[i + 4], y[i + 5], y[i + 6], y[i + 7]};
              store8(to + i, part);
            }
          } else if (live) {
            float* to = reinterpret_cast<float*>(mine) + c0;
#pragma unroll
            for (int i = 0; i < 16; i += 4) store4(to + i, make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]));
          }
        }
        if (live && !alone) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(parts.o + part_row * D + g * SIDE), "r"(smem_u32(mine)),
                       "r"(SIDE * 4) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          // (read from here before the CTA leaves; written before anything else looks at them below)
          if (sm.bad) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        if (sm.bad && live) {  // values that are not finite join the sums of the rows that see them
#pragma unroll 1
          for (int e = g * SIDE; e < (g + 1) * SIDE; ++e) {
            const float more = tree_not_finite<D, E4M3>(sm, r, e, block0, block1, cache, table, kv_head, rows.bits, rows.words, rows.keep_first);
            if (more == 0.f) continue;
            if (alone) {
              __nv_bfloat16* to = out + (size_t)token * out_stride + (size_t)head * D + e;
              *to = __float2bfloat16_rn(__bfloat162float(*to) + more);
            } else {
              parts.o[part_row * D + e] += more;
            }
          }
        }
        if (live && !alone && g == 0) {
          parts.ml[2 * part_row] = m_all;
          parts.ml[2 * part_row + 1] = l_all;
        }
      } else {
        atomicExch(&sm.failed, 1u);
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == kTreeMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
  if (threadIdx.x == 0 && sm.failed && error) atomicCAS(error, 0, 6);
}

template <int D, bool E4M3>
static int launch_tree(const dim3& grid, const __nv_bfloat16* q, int q_stride, __nv_bfloat16* out, int out_stride, const QueryRows& rows,
                       const CachePages& cache, const Partials& parts, int* error, cudaStream_t stream) {
  const size_t shared = sizeof(TreeShared<D>) + 1024;
  // Pages that the copy engine puts down swizzled: a box of [page_size x 64].
  const int direct = !E4M3 && cache.page_size >= 8 && cache.page_size <= 128 && cache.page_shift >= 0;
  CUtensorMap map_k = {}, map_v = {};
  if (direct) {
    const int all_rows = (int)((long long)cache.num_pages * cache.num_kv_heads * cache.page_size);
    int status;
    if ((status = make_map(&map_k, cache.k, all_rows, D, D, cache.page_size)) != 0) return status;
    if ((status = make_map(&map_v, cache.v, all_rows, D, D, cache.page_size)) != 0) return status;
  }
  auto kernel = attention_tree_tcgen05_kernel<D, E4M3>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
  if (err != cudaSuccess) return (int)err;
  return (int)launch_dependent(kernel, grid, dim3(kTreeThreads), shared, stream, map_k, map_v, direct, q, q_stride, out, out_stride, rows, cache, parts,
                               error);
}

}  // namespace distie

using namespace distie;

// Drafted tokens: q [tokens, >= heads * head_dim] and out [tokens, heads * head_dim] bfloat16, a cache of bfloat16 or (with
// scales) e4m3, heads of 64 or 128 (else DISTIE_ERR_UNSUPPORTED, like rows that are not aligned to what a thread moves), at most
// 256 new tokens a request.  seqs [requests, 3], bits [tokens, words].  scratch: tokens * heads * splits * (value size + 2) floats.
extern "C" int distie_attention_tree_tcgen05(const void* q, int q_stride, void* out, int out_stride, float* scratch, const int* positions,
                                             const int* token_seq, const int* seq_seat, const int* seqs, const int* bits, int words, int requests, int tokens,
                                             int most_nodes, const void* k_cache, const void* v_cache, const float* k_scale,
                                             const float* v_scale, const int* block_table, int table_width, int num_heads, int num_kv_heads,
                                             int head_dim, int page_size, int num_pages, int window, int chunk, int keep_first, float scale,
                                             float softcap, const float* sink, int splits, int* error, cudaStream_t stream) {
  if (tokens <= 0 || requests <= 0) return 0;
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads != 0 || page_size < 1 || table_width < 1 || keep_first < 0 || splits < 1 ||
      splits > 65535 || requests > 65535 || most_nodes < 1 || most_nodes > kTreeMostNodes || words > kTreeMostNodes / 32 || words * 32 < most_nodes || seqs == nullptr ||
      bits == nullptr || (splits > 1 && scratch == nullptr) || (k_scale == nullptr) != (v_scale == nullptr))
    return DISTIE_ERR_ARG;
  if ((head_dim != 64 && head_dim != 128) || (q_stride & 3) || ((uintptr_t)q & 7) || (out_stride & 7) || ((uintptr_t)out & 15) ||
      (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)scratch) & 15) || (long long)num_pages * num_kv_heads * page_size > 0x7fffffffLL)
    return DISTIE_ERR_UNSUPPORTED;
  const CachePages cache = make_pages(k_cache, v_cache, k_scale, v_scale, block_table, table_width, num_kv_heads, head_dim, head_dim,
                                      page_size, num_pages);
  const int group = num_heads / num_kv_heads;
  const QueryRows rows{positions, token_seq, seq_seat, seqs, bits, words, tokens, requests, most_nodes, group, num_heads, window, chunk, keep_first,
                       scale * 1.4426950408889634f, make_score_extras(scale, softcap, sink)};
  const Partials parts{scratch, scratch ? scratch + (size_t)tokens * num_heads * splits * head_dim : nullptr, splits};
  const dim3 grid((unsigned)(((long long)most_nodes * group + kTreeRows - 1) / kTreeRows * num_kv_heads), requests, splits);
  int status;
  if (head_dim == 64)
    status = k_scale ? launch_tree<64, true>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts, error, stream)
                     : launch_tree<64, false>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts, error, stream);
  else
    status = k_scale ? launch_tree<128, true>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts, error, stream)
                     : launch_tree<128, false>(grid, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, rows, cache, parts, error, stream);
  if (status != 0 || splits == 1) return status;
  return rows_merge_bf16(parts, rows, out, out_stride, head_dim, stream);
}

DISTIE_PACKED(distie_attention_tree_tcgen05)
