// Backward of differential attention for sm_100a: dQ, dK, dV and dlam of O = (A_1 - lam A_2) V.
//
// With dP = dO V^T and delta_m = rowsum(A_m o dP) = dO . (A_m V):
//   dV = (A_1 - lam A_2)^T dO      dS_1 = A_1 o (dP - delta_1)      dS_2 = -lam A_2 o (dP - delta_2)      dlam = -sum delta_2
// and dQ_m = scale dS_m K_m, dK_m = scale dS_m^T Q_m, each over its half of the head dimension.  dP and dV are one product for both
// maps and the others have half the depth or width, so that a pair of tiles takes the products of ONE attention head of that size;
// as two query heads with half of d set to zero it took those of two.  What stays double is the exponentials.
//
//   1. preprocess   -delta_1, -delta_2 and -LSE_m * log2(e) per row, from dO, O, A_2 V; interleaved by 64 rows (one copy per tile)
//   2. dK/dV kernel items of 128 keys of a KV head, over the 64-row Q tiles of the heads of its group; beside it dlam
//   3. dQ kernel    items of 128 query rows, over blocks of 128 keys
// Both are persistent, with the warp roles, rings and work counters of the plain backward (bwd_sm100.cu): sixteen elementwise warps (four
// threads per TMEM lane), a TMA producer, one thread that issues the products, a scheduler.  Every result is bitwise reproducible.
#include "bwd_common.cuh"

#include <algorithm>

#include "diff.cuh"
#include "packed_rows.cuh"
#include "work_order.cuh"

namespace fa {
namespace {

// Statistics of 64 rows lie together, 64 floats each: -LSE_1, -LSE_2 (base 2), -delta_1, -delta_2 (dQ kernel), delta_1 - delta_2 (dK/dV
// kernel).  The dK/dV kernel, whose threads hold keys, would have to read the statistics of every query from shared memory, a wavefront for
// each four bytes and warp: with the operands of the products that was 91 % of what the memory can deliver, 2470 clocks a tile.  There
// the products add them: a 64-column row per query holds -LSE_1 / c, -LSE_2 / c and -delta_1 (c = scale * log2(e)), each cut into three fp16
// numbers for three columns of a K = 16 slice of its own, whose other operand is the constants kSplit in every row.  So S_m comes
// as S_m - LSE_m / c and dP as dP - delta_1.
constexpr int kStatRows = 64;
constexpr int kStatFloats = 5 * kStatRows;
constexpr int kExtColumns = 64;  // slices at columns 0 (S_1), 16 (S_2), 32 (dP); 48-63 are not used
// The tile of 64 rows that the statistics of a (batch, head) begin with; `tiles`: of a (batch, head), or of a head in packed batches.  There
// a sequence that begins at token q_off has the tiles from q_off / 64 + batch on, as many as it needs and none twice, so that the scratch
// memory follows the tokens and not the longest sequence times the batch: 1000 texts, one of 8192 tokens and the others of 24, 16 heads:
// 0.2 GB instead of 19.
__device__ __forceinline__ int64_t first_stat_tile(bool packed, int q_off, int batch, int head, int h, int tiles) {
  return packed ? static_cast<int64_t>(head) * tiles + (q_off >> 6) + batch : (static_cast<int64_t>(batch) * h + head) * tiles;
}
static_assert(kStatRows == 64, "q_off >> 6");
// 2^15, 2^4, 2^-8: each number holds what the one before leaves over, 2^9 to 2^11 times smaller.  Up to 2 * 10^9 in all, the rest below
// 2^-33 of the value (or 2^-32).
__device__ __forceinline__ void split3(float x, __half (&h)[3]) {
  h[0] = __float2half_rn(x * 0x1p-15f);
  if (x == -INFINITY) {  // rows that do not exist
    h[1] = h[2] = __float2half_rn(0.f);
    return;
  }
  x -= __half2float(h[0]) * 0x1p15f;
  h[1] = __float2half_rn(x * 0x1p-4f);
  x -= __half2float(h[1]) * 0x1p4f;
  h[2] = __float2half_rn(x * 0x1p8f);
}

struct DiffKernelParams {
  CUtensorMap tm_q, tm_k, tm_v, tm_do;  // boxes of 128 rows; dK/dV kernel: q and do of 64
  CUtensorMap tm_ext;  // dK/dV kernel: (tiles of all heads * 64, 64) fp16, boxes of 64 rows
  __half *dq, *dk, *dv;
  int64_t dq_batch_stride, dq_row_stride, dq_head_stride;
  int64_t dk_batch_stride, dk_row_stride, dk_head_stride;
  int64_t dv_batch_stride, dv_row_stride, dv_head_stride;
  const float* stats;  // (b, h, stat_tiles, 5, 64); packed: (h, stat_tiles, 5, 64)
  int stat_tiles;
  int seqlen_q, seqlen_k, h, h_k, group, b;
  float scale, scale_log2;
  int is_causal, causal_shift;
  const int* cu_seqlens_q;
  const int* cu_seqlens_k;
  FaDiffWeights weights;
  float* head_dlam;  // (h) dlam of each head, or null: to dlam
  void* dlam;
  int* status;
  int* sched;
  int items_x, total_items, section_rows;
};

// =============================================================================================
// preprocess
// =============================================================================================
struct DiffPreParams {
  const __half *o, *o2, *dout;
  const float* lse;
  float* stats;
  __half* ext;
  float inv_scale_log2;  // 1 / c
  int64_t o_batch_stride, o_row_stride, o_head_stride;
  int64_t o2_batch_stride, o2_row_stride, o2_head_stride;
  int64_t do_batch_stride, do_row_stride, do_head_stride;
  int64_t lse_row_stride;
  int h, seqlen_q, sq_pad, stat_tiles, d;
  FaDiffWeights weights;
  const int* cu_seqlens_q;
  PackedRows clear[3];  // dq, dk, dv; base null: nothing to clear
  const int* status;
  int keys_written;     // keys per sequence that the dK/dV kernel writes
};

// As in the plain backward: an item is kPreRows rows of a head, heads fastest, d / 8 threads per item with 16-byte loads.  Bound by memory:
// B2 S4096 H16 D128 23 us for 102 MB read and 19 written, which stay in L2 mostly.
constexpr int kPreRows = 4;
static_assert(kClearThreads == 256, "the clearing threads are those of the preprocess kernel");
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b) {
  const __half2 *x = reinterpret_cast<const __half2*>(&a), *y = reinterpret_cast<const __half2*>(&b);
  float acc = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 u = __half22float2(x[k]), v = __half22float2(y[k]);
    acc = fmaf(u.x, v.x, acc);
    acc = fmaf(u.y, v.y, acc);
  }
  return acc;
}
template <bool kClear>
__global__ void __launch_bounds__(256, 3) diff_preprocess_kernel(const __grid_constant__ DiffPreParams p) {
  grid_launch_dependents();
  const bool stopped = kClear && wait_timed_out(p.status);
  const int tpr = p.d / 8;  // threads per item: 8 or 16
  const int item = blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
  const int sub = threadIdx.x % tpr;
  const int head = item % p.h, row0 = (item / p.h) * kPreRows, batch = blockIdx.z;
  const int q_off = p.cu_seqlens_q ? p.cu_seqlens_q[batch] : 0;
  const int sq = p.cu_seqlens_q ? min(p.cu_seqlens_q[batch + 1] - q_off, p.seqlen_q) : p.seqlen_q;  // rows past max_seqlen_q have no LSE
  auto base = [&](int64_t batch_stride, int64_t row_stride, int64_t head_stride) {
    return (p.cu_seqlens_q ? q_off * row_stride : batch * batch_stride) + head * head_stride + sub * 8;
  };
  const __half* o = p.o + base(p.o_batch_stride, p.o_row_stride, p.o_head_stride);
  const __half* o2 = p.o2 + base(p.o2_batch_stride, p.o2_row_stride, p.o2_head_stride);
  const __half* dout = p.dout + base(p.do_batch_stride, p.do_row_stride, p.do_head_stride);
  // Behind the last row the dK/dV kernel needs -inf up to the end of its 64-row tile, but not in packed batches, where it masks those rows; the
  // dQ kernel does not store them.  (Up to the end of the 128-row tile: 1000 texts of 24 tokens, 16 heads D128 213 us, 111 so.)
  const int rows = p.cu_seqlens_q ? sq : min((sq + kStatRows - 1) / kStatRows * kStatRows, p.sq_pad);
  if (__any_sync(0xffffffffu, row0 < rows)) {
    uint4 a[kPreRows], b[kPreRows], c[kPreRows];
#pragma unroll
    for (int i = 0; i < kPreRows; ++i) {
      a[i] = b[i] = c[i] = make_uint4(0, 0, 0, 0);
      if (row0 + i < sq) {
        a[i] = *reinterpret_cast<const uint4*>(o + static_cast<int64_t>(row0 + i) * p.o_row_stride);
        b[i] = *reinterpret_cast<const uint4*>(o2 + static_cast<int64_t>(row0 + i) * p.o2_row_stride);
        c[i] = *reinterpret_cast<const uint4*>(dout + static_cast<int64_t>(row0 + i) * p.do_row_stride);
      }
    }
    // lane `sub` of the item writes the statistics of row sub % kPreRows: map 1 the first kPreRows lanes, map 2 the next
    const int mine = sub % kPreRows, map = sub / kPreRows;
    const int64_t bh = static_cast<int64_t>(batch) * p.h + head;
    float lse = 0.f;
    if (map < 2 && row0 + mine < sq) lse = p.lse[(2 * bh + map) * p.lse_row_stride + row0 + mine];
    const float lam = weight_of(p.weights, head);
    float delta = 0.f, other = 0.f;  // of this lane's map, of the other one
#pragma unroll
    for (int i = 0; i < kPreRows; ++i) {
      float x = dot8(a[i], c[i]), y = dot8(b[i], c[i]);
      for (int off = tpr / 2; off > 0; off >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, off);
        y += __shfl_xor_sync(0xffffffffu, y, off);
      }
      if (i == mine) {  // dO . A_1 V = dO . O + lam dO . A_2 V
        const float first = fmaf(lam, y, x);
        delta = map == 0 ? first : y, other = map == 0 ? y : first;
      }
    }
    if (map < 2 && row0 < rows) {  // kPreRows rows of one tile; in packed batches the next tile may be another sequence's
      const int row = row0 + mine;
      const int64_t tile = first_stat_tile(p.cu_seqlens_q != nullptr, q_off, batch, head, p.h, p.stat_tiles) + row / kStatRows;
      float* to = p.stats + tile * kStatFloats + row % kStatRows;
      const bool valid = row < sq;
      const float nl = valid ? -lse * kLog2e : -INFINITY;
      to[map * kStatRows] = nl;
      to[(2 + map) * kStatRows] = valid ? -delta : 0.f;
      if (map == 0) to[4 * kStatRows] = valid ? delta - other : 0.f;
      // 16 columns of S_m, by the lane of map 1 those of dP too
      uint4* ext = reinterpret_cast<uint4*>(p.ext + (tile * kStatRows + row % kStatRows) * kExtColumns);
      auto put = [&](int slice, float x) {
        __half h[4];
        split3(x, reinterpret_cast<__half(&)[3]>(h));
        h[3] = __float2half_rn(0.f);
        const uint32_t* w = reinterpret_cast<const uint32_t*>(h);
        ext[2 * slice] = make_uint4(w[0], w[1], 0u, 0u);
        ext[2 * slice + 1] = make_uint4(0u, 0u, 0u, 0u);
      };
      put(map, nl * p.inv_scale_log2);
      if (map == 0) put(2, valid ? -delta : 0.f);
    }
  }
  if constexpr (kClear) {  // the other kernels write all other rows of dq, dk, dv
    const int64_t block = static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x;
    const int64_t blocks = min(static_cast<int64_t>(gridDim.x) * gridDim.z, static_cast<int64_t>(kMaxClearBlocks));
    if (block < blocks) {
      const uint32_t worker = static_cast<uint32_t>(block) * kClearThreads + threadIdx.x;
#pragma unroll 1
      for (int i = 0; i < 3; ++i) clear_unused_rows(p.clear[i], stopped, worker, static_cast<uint32_t>(blocks) * kClearThreads);
    }
    // rows past max_seqlen_q and keys past max_seqlen_k: the first blocks of the sequence
    const uint32_t workers = min(gridDim.x, static_cast<unsigned>(kMaxClearBlocks)) * kClearThreads;
    if (blockIdx.x < kMaxClearBlocks) {
#pragma unroll 1
      for (int i = 0; i < 3; ++i) {
        const int* cu = p.clear[i].cu_seqlens;
        const int64_t first = static_cast<int64_t>(cu[batch]) + (i == 0 ? p.seqlen_q : p.keys_written);
        const int64_t last = min(static_cast<int64_t>(cu[batch + 1]), p.clear[i].total);
        clear_rows(p.clear[i], first, last, blockIdx.x * kClearThreads + threadIdx.x, workers);
      }
    }
  }
}

// dlam of a head by one warp, in a fixed order: the rows' -delta_2, eight loads in flight.  Of one sequence where there are few, else of eight
// sequences: many short ones would be a memory latency each (1000 texts of 24 tokens, 4 heads, D64: a training step
// 656 -> 486 us, the dK/dV kernel 437 -> 208).
__device__ __forceinline__ void sum_dlam(const DiffKernelParams& p, int head, int lane) {
  constexpr int kLoads = 8;
  auto rows_of = [&](int batch) {
    return p.cu_seqlens_q ? min(p.cu_seqlens_q[batch + 1] - p.cu_seqlens_q[batch], p.seqlen_q) : p.seqlen_q;
  };
  auto tile_of = [&](int batch) {
    const int q_off = p.cu_seqlens_q ? p.cu_seqlens_q[batch] : 0;
    return static_cast<int>(first_stat_tile(p.cu_seqlens_q != nullptr, q_off, batch, head, p.h, p.stat_tiles));
  };
  auto stats_at = [&](int tile) { return p.stats + static_cast<int64_t>(tile) * kStatFloats + 3 * kStatRows; };
  float part[kLoads] = {};
  if (p.b < kLoads) {
    for (int batch = 0; batch < p.b; ++batch) {
      const int rows = rows_of(batch);
      const float* s = stats_at(tile_of(batch));
      for (int r0 = 0; r0 < rows; r0 += kLoads * 32) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int r = r0 + i * 32 + lane;
          if (r < rows) part[i] += s[r / kStatRows * kStatFloats + r % kStatRows];
        }
      }
    }
  } else {
    for (int first = 0; first < p.b; first += kLoads) {
      const bool has = lane < kLoads && first + lane < p.b;
      const int mine = has ? rows_of(first + lane) : 0, tile = has ? tile_of(first + lane) : 0;
      const int most = __reduce_max_sync(0xffffffffu, mine);
      int rows[kLoads], tiles[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) rows[i] = __shfl_sync(0xffffffffu, mine, i), tiles[i] = __shfl_sync(0xffffffffu, tile, i);
      for (int r = lane; r - lane < most; r += 32) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          if (r < rows[i]) part[i] += stats_at(tiles[i])[r / kStatRows * kStatFloats + r % kStatRows];
      }
    }
  }
  float sum = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane != 0) return;
  if (p.head_dlam != nullptr) p.head_dlam[head] = sum;
  else if (p.weights.is_half) static_cast<__half*>(p.dlam)[head] = __float2half_rn(sum);
  else static_cast<float*>(p.dlam)[head] = sum;
}

// One weight for all heads: the sum of their gradients
__global__ void join_dlam_kernel(const float* head_dlam, int h, void* dlam, int is_half) {
  float sum = 0.f;
  for (int i = threadIdx.x; i < h; i += 32) sum += head_dlam[i];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (threadIdx.x != 0) return;
  if (is_half) *static_cast<__half*>(dlam) = __float2half_rn(sum);
  else *static_cast<float*>(dlam) = sum;
}

// =============================================================================================
// products
// =============================================================================================
// Pair i of exponentials: every kEvery-th is a polynomial on the FMA pipes (see the forward kernel).  These kernels are short of issue slots as
// well, and a polynomial takes 13 for two: eight are best in the dQ kernel, four in the dK/dV kernel at D = 64 and eight at D = 128 (B2 S4096 H16
// D64 causal, both at four 437 us, dQ at three, eight, none 434, 429, 436, dK/dV at eight, none 439, 444; B2 S2048 Hq16 Hkv4 D128 causal dK/dV at
// four, eight, none 181, 176, 178).
template <int kEvery>
__device__ __forceinline__ float2 exp2_of_pair(int i, float2 x) {
  return i % kEvery == kEvery - 1 ? exp2_polynomial<true>(x) : exp2_pair(x);
}

// C = A[:, half m of d] B[:, half m of d]^T: slices of 16 columns, of tiles of kRowsA and kRowsB rows (a swizzle chunk of 64 columns is
// 128 bytes a row)
template <int D, int kRowsA, int kRowsB>
__device__ __forceinline__ void product_slices(uint32_t d_tmem, uint32_t a_tile, uint32_t b_tile, uint32_t idesc, int first, int count) {
  const uint64_t ad = make_smem_desc(a_tile, 16, 1024), bd = make_smem_desc(b_tile, 16, 1024);
#pragma unroll
  for (int k = 0; k < count; ++k) {
    const int s = first + k;
    mma_ss(d_tmem, desc_advance(ad, (s >> 2) * kRowsA * 128 + (s & 3) * 32), desc_advance(bd, (s >> 2) * kRowsB * 128 + (s & 3) * 32), idesc,
           k > 0);
  }
}
// C[:, half m of d] (+)= A[tmem, kK packed contraction elements] B[kK rows of the tile, half m of d].  The slices of 16 elements (8
// columns) of A lie kPitch columns apart, in pairs or singly.
template <int D, int kK, class Column>
__device__ __forceinline__ void product_half(uint32_t d_tmem, uint32_t a_tmem, Column column, uint32_t b_tile, int m, uint32_t idesc,
                                             bool zero_init) {
  // half of d: a chunk of 64 columns at D = 128, half of the 128-byte rows of the only chunk at D = 64
  const uint64_t bd = make_smem_desc(b_tile + (D == 128 ? m * kK * 128 : m * 64), kK * 128, 1024);
#pragma unroll
  for (int k = 0; k < kK / 16; ++k) mma_ts(d_tmem, a_tmem + column(k), desc_advance(bd, k * 2048), idesc, (zero_init && k == 0) ? 0u : 1u);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}

// =============================================================================================
// dQ kernel
// =============================================================================================
// TMEM: S_1 [0, 128), S_2 [128, 256), dP [256, 384), dQ [384, 384 + D), all of it at D = 128.  A thread packs dS_m into the first 16 of
// its own 32 columns of S_m, so that no other thread's scores are in the way; the dQ products take their slices from there.
// The elementwise warps go through a block map by map, dP in registers: while they are at map 2, dQ_1 of the block and S_1, dP of the
// next one run, while they are at map 1 of the next, dQ_2 and S_2.  Nothing is double-buffered and nothing stands still.
// B2 S4096 H16 D128 without mask 400-440 us by itself: 3147 clocks a block of both maps, of which the products take 1536 and the
// special-function unit, with every eighth pair a polynomial, 1792; the one is busy half of the time, the other 58 %, instructions are issued in
// 0.51 of the slots.  Bound by the chain barrier, TMEM load, exponentials, store of each warp; causal S8192 by the power cap (1.65 GHz).
constexpr int kDiffThreads = 608;
constexpr int kDiffSched = 18;
constexpr int kDiffReaders = kComputeWarps + 2;  // elementwise warps, producer warp, issuing thread
constexpr int kDqSlots = 3;     // the item to be stored, the current one, the next (see the plain dQ kernel)
constexpr int kDqKStages = 3;   // a K tile lives from S_1 of its block to dQ_2, which is issued a block later
constexpr int kDqVStages = 2;
constexpr int kDqStatFloats = 4 * kStatRows;  // without the last ones

struct __align__(16) DiffDqItem {
  int nb;  // key blocks to visit; < 0: no more work
  int sk, shift, row0;
  int q_off, k_off, sq, bq;
  int batch, head, head_k, fix_k_tail;
  float lam;
  int pad[3];
};
struct DiffDqBarriers {
  uint64_t q_full, q_free;
  uint64_t k_full[kDqKStages], k_empty[kDqKStages];
  uint64_t v_full[kDqVStages], v_empty[kDqVStages];
  uint64_t s1_full;     // S_1 and dP of a block
  uint64_t s2_full;
  uint64_t ds1_full, ds2_full;  // dS_m written; dP (S_2) sits in registers
  uint64_t acc_full, acc_free;
  uint64_t tail_fixed[kDqSlots];
  uint64_t sched_full[kDqSlots], sched_empty[kDqSlots], sched_go;
  DiffDqItem items[kDqSlots];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(DiffDqBarriers) <= 1024, "barrier block");

template <int D>
struct DqCfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kChunkBytes = 128 * 128;
  static constexpr int kTileBytes = kChunks * kChunkBytes;
  static constexpr int kAlignPad = D == 128 ? 0 : 1024;  // no room: the kernel checks that its memory starts on 1024 bytes
  static constexpr int kSmemBytes = (2 + kDqKStages + kDqVStages) * kTileBytes + 2 * kDqStatFloats * 4 + 1024 + kAlignPad;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

__device__ __forceinline__ void make_dq_item(const DiffKernelParams& p, int batch, int head, int mblk, DiffDqItem& w) {
  const bool varlen = p.cu_seqlens_q != nullptr;
  w.batch = batch, w.head = head;
  w.q_off = varlen ? p.cu_seqlens_q[batch] : 0;
  w.sq = varlen ? p.cu_seqlens_q[batch + 1] - w.q_off : p.seqlen_q;
  w.k_off = varlen ? p.cu_seqlens_k[batch] : 0;
  w.sk = varlen ? p.cu_seqlens_k[batch + 1] - w.k_off : p.seqlen_k;
  w.row0 = mblk * kBlock;
  w.bq = varlen ? 0 : batch;
  w.head_k = head / p.group;
  const int nkb = (w.sk + kBlock - 1) / kBlock;
  w.shift = (p.is_causal == 2) ? p.causal_shift : w.sk - w.sq;
  w.sq = min(w.sq, p.seqlen_q);  // rows past max_seqlen_q have no statistics
  w.nb = nkb;
  if (p.is_causal) {
    const int x = w.row0 + kBlock + w.shift;
    w.nb = x <= 0 ? 0 : min(nkb, (x + kBlock - 1) / kBlock);
  }
  w.fix_k_tail = varlen && (w.sk % kBlock) != 0 && w.nb == nkb && w.nb > 0;
  w.lam = weight_of(p.weights, head);
}

template <int D>
__global__ void __launch_bounds__(kDiffThreads, 1) diff_dq_kernel(const __grid_constant__ DiffKernelParams p) {
  using C = DqCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int stop_probe = stop_probe_begin(p.status);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  if (smem - smem_raw > C::kAlignPad) {  // uniform over the CTA: nothing has been set up yet
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, kStatusSmemLayout);
    grid_dependency_wait();
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* sdO = sQ + C::kTileBytes;
  uint8_t* sK = sdO + C::kTileBytes;
  uint8_t* sV = sK + kDqKStages * C::kTileBytes;
  float* sStats = reinterpret_cast<float*>(sV + kDqVStages * C::kTileBytes);  // [row / 64][4][64]
  DiffDqBarriers* bars = reinterpret_cast<DiffDqBarriers*>(sStats + 2 * kDqStatFloats);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kS1 = 0, kS2 = 128, kDP = 256, kAcc = 384;

  if (warp == kProducerWarp && lane == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_free, 1 + kComputeWarps);
    for (int i = 0; i < kDqKStages; ++i) mbar_init(&bars->k_full[i], 1), mbar_init(&bars->k_empty[i], 1);
    for (int i = 0; i < kDqVStages; ++i) mbar_init(&bars->v_full[i], 1), mbar_init(&bars->v_empty[i], 1);
    mbar_init(&bars->s1_full, 1);
    mbar_init(&bars->s2_full, 1);
    mbar_init(&bars->ds1_full, kComputeWarps);
    mbar_init(&bars->ds2_full, kComputeWarps);
    mbar_init(&bars->acc_full, 1);
    mbar_init(&bars->acc_free, kComputeWarps);
    for (int i = 0; i < kDqSlots; ++i) {
      mbar_init(&bars->tail_fixed[i], 1);
      mbar_init(&bars->sched_full[i], 1);
      mbar_init(&bars->sched_empty[i], kDiffReaders);
    }
    mbar_init(&bars->sched_go, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  const bool stop = __syncthreads_or(stop_probe) != 0;
  tc_fence_after_sync();
  const uint32_t tmem_base = bars->tmem_base;
  WaitCtx ctx{&bars->abort_flag, p.status};
  auto wait_item = [&](int n) -> bool { return mbar_wait(&bars->sched_full[n % kDqSlots], (n / kDqSlots) & 1, ctx); };
  auto release_item = [&](int n) { mbar_arrive(&bars->sched_empty[n % kDqSlots]); };

  if (stop) {
  } else if (warp == kDiffSched) {
    if (lane == 0) {
      bool finished = false;
      int seq = 0;
      for (int n = 0;; ++n) {
        int next = blockIdx.x;
        if (n > 0) {
          if (!mbar_wait(&bars->sched_go, (n - 1) & 1, ctx)) break;
          next = gridDim.x + atomicAdd(p.sched, 1);
        }
        DiffDqItem it;
        it.nb = -1;
        while (next < p.total_items) {
          int batch, head, mblk, sq;
          if (p.cu_seqlens_q == nullptr) {
            const HeadPlace at = section_item(next, p.h * p.b, p.items_x, p.group, p.seqlen_k, p.section_rows);
            batch = at.head / p.h, head = at.head - batch * p.h, mblk = p.items_x - 1 - at.place, sq = p.seqlen_q;
          } else {  // slots per sequence from cu_seqlens_q / 128 (at most one spare slot per sequence and head)
            while (seq + 1 < p.b && p.h * ((p.cu_seqlens_q[seq + 1] >> 7) + seq + 1) <= next) ++seq;
            const int v0 = (p.cu_seqlens_q[seq] >> 7) + seq, v1 = (p.cu_seqlens_q[seq + 1] >> 7) + seq + 1;
            const int rel = next - p.h * v0, cnt = v1 - v0;
            sq = p.cu_seqlens_q[seq + 1] - p.cu_seqlens_q[seq];
            batch = seq, head = 0, mblk = -1;
            if (rel >= 0 && rel < p.h * cnt) {  // else before the first sequence (cu_seqlens_q[0] >= 128) or past the last one
              const HeadPlace at = section_item(rel, p.h, cnt, p.group, p.cu_seqlens_k[seq + 1] - p.cu_seqlens_k[seq], p.section_rows);
              head = at.head, mblk = (sq + kBlock - 1) / kBlock - 1 - at.place;
            }
          }
          if (mblk >= 0 && mblk * kBlock < min(sq, p.seqlen_q)) {
            make_dq_item(p, batch, head, mblk, it);
            break;
          }
          next = gridDim.x + atomicAdd(p.sched, 1);
        }
        if (!mbar_wait(&bars->sched_empty[n % kDqSlots], ((n / kDqSlots) & 1) ^ 1, ctx)) break;
        bars->items[n % kDqSlots] = it;
        mbar_arrive(&bars->sched_full[n % kDqSlots]);
        if (it.nb < 0) {
          finished = true;
          break;
        }
      }
      if (finished) {
        __threadfence();
        if (atomicAdd(p.sched + 1, 1) == static_cast<int>(gridDim.x) - 1) {
          atomicExch(p.sched, 0);
          atomicExch(p.sched + 1, 0);
        }
      }
    }
  } else if (warp == kProducerWarp) {
    int G = 0, ni = 0, nf = 0;
    for (int n = 0;; ++n) {
      bool ok = wait_item(n);
      if (!__all_sync(0xffffffffu, ok)) break;
      const DiffDqItem w = bars->items[n % kDqSlots];
      __syncwarp();
      if (lane == 0) release_item(n);
      if (w.nb < 0) break;
      if (w.nb == 0) continue;
      if (lane == 0) {
        ok = mbar_wait(&bars->q_free, (ni & 1) ^ 1, ctx);
        if (ok) {
          mbar_arrive_expect_tx(&bars->q_full, 2 * C::kTileBytes + 2 * kDqStatFloats * 4);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c) {
            tma_load_4d(sQ + c * C::kChunkBytes, &p.tm_q, &bars->q_full, c * 64, w.head, w.q_off + w.row0, w.bq);
            tma_load_4d(sdO + c * C::kChunkBytes, &p.tm_do, &bars->q_full, c * 64, w.head, w.q_off + w.row0, w.bq);
          }
          const int64_t tile = first_stat_tile(p.cu_seqlens_q != nullptr, w.q_off, w.batch, w.head, p.h, p.stat_tiles) + w.row0 / kStatRows;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            bulk_load_1d(sStats + i * kDqStatFloats, p.stats + (tile + i) * kStatFloats, kDqStatFloats * 4, &bars->q_full);
        }
        for (int j = 0; ok && j < w.nb; ++j) {
          const int g = G + j, s = g % kDqKStages, sv = g % kDqVStages;
          const int krow = w.k_off + j * kBlock;
          if (!(ok = mbar_wait(&bars->k_empty[s], ((g / kDqKStages) & 1) ^ 1, ctx))) break;
          mbar_arrive_expect_tx(&bars->k_full[s], C::kTileBytes);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
            tma_load_4d(sK + s * C::kTileBytes + c * C::kChunkBytes, &p.tm_k, &bars->k_full[s], c * 64, w.head_k, krow, w.bq);
          if (!(ok = mbar_wait(&bars->v_empty[sv], ((g / kDqVStages) & 1) ^ 1, ctx))) break;
          mbar_arrive_expect_tx(&bars->v_full[sv], C::kTileBytes);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
            tma_load_4d(sV + sv * C::kTileBytes + c * C::kChunkBytes, &p.tm_v, &bars->v_full[sv], c * 64, w.head_k, krow, w.bq);
        }
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      if (w.fix_k_tail) {  // rows of the next sequence: 0 times what they hold may be NaN
        const int g = G + w.nb - 1, s = g % kDqKStages;
        if (!mbar_wait_warp(&bars->k_full[s], (g / kDqKStages) & 1, ctx)) break;
        zero_tile_rows_from<D>(sK + s * C::kTileBytes, w.sk - (w.nb - 1) * kBlock, lane);
        if (lane == 0) mbar_arrive(&bars->tail_fixed[nf % kDqSlots]);  // in turn: see the plain dQ kernel
        ++nf;
      }
      G += w.nb;
      ++ni;
    }
  } else if (warp == kMmaWarp) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_f16(128, kBlock, false, false);
      constexpr uint32_t idesc_acc = make_idesc_f16(128, D / 2, false, true);
      const uint32_t q_addr = smem_u32(sQ), do_addr = smem_u32(sdO);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, ctx); };
      auto k_tile = [&](int g) { return smem_u32(sK + (g % kDqKStages) * C::kTileBytes); };
      // dQ of block `held` is issued a block later (see above)
      int G = 0, ni = 0, nf = 0, held = -1, items_begun = 0;
      bool held_first = false, held_last = false, held_fix = false, ok = true;
      auto packed_column = [](int k) { return (k >> 1) * 32 + (k & 1) * 8; };
      auto dq_1 = [&]() -> bool {
        if (!wait(&bars->ds1_full, held & 1)) return false;
        if (held_fix && !wait(&bars->tail_fixed[nf % kDqSlots], (nf / kDqSlots) & 1)) return false;
        if (held_first && items_begun++ > 0 && !wait(&bars->acc_free, items_begun & 1)) return false;  // phase items_begun - 2
        tc_fence_after_sync();
        product_half<D, kBlock>(tmem_base + kAcc, tmem_base + kS1, packed_column, k_tile(held), 0, idesc_acc, held_first);
        return true;
      };
      auto dq_2 = [&]() -> bool {
        if (!wait(&bars->ds2_full, held & 1)) return false;
        tc_fence_after_sync();
        product_half<D, kBlock>(tmem_base + kAcc + D / 2, tmem_base + kS2, packed_column, k_tile(held), 1, idesc_acc, held_first);
        tc_commit(&bars->k_empty[held % kDqKStages]);
        if (held_last) tc_commit(&bars->acc_full);
        nf += held_fix;
        held = -1;
        return true;
      };
      for (int n = 0; ok; ++n) {
        if (!(ok = wait_item(n))) break;
        const int nb = bars->items[n % kDqSlots].nb, fix = bars->items[n % kDqSlots].fix_k_tail;
        release_item(n);
        if (nb <= 2 && nb >= 0) mbar_arrive(&bars->sched_go);  // short item: claim the next one right away
        if (nb <= 0) {
          // the item before ends here: its last dQ is waited for by the warps that store it
          if (held >= 0) ok = dq_1() && dq_2();
          if (nb < 0) break;
          continue;
        }
        if (!(ok = wait(&bars->q_full, ni & 1))) break;
        for (int j = 0; ok && j < nb; ++j) {
          const int g = G + j, s = g % kDqKStages, sv = g % kDqVStages;
          if (!(ok = wait(&bars->k_full[s], (g / kDqKStages) & 1))) break;
          if (!(ok = wait(&bars->v_full[sv], (g / kDqVStages) & 1))) break;
          const bool had = held >= 0;
          if (had && !(ok = dq_1())) break;  // dS_1(g-1) written: S_1 may be overwritten behind dQ_1, and dP has been read
          product_slices<D, 128, 128>(tmem_base + kS1, q_addr, k_tile(g), idesc_s, 0, D / 32);
          product_slices<D, 128, 128>(tmem_base + kDP, do_addr, smem_u32(sV + sv * C::kTileBytes), idesc_s, 0, D / 16);
          tc_commit(&bars->s1_full);
          tc_commit(&bars->v_empty[sv]);
          if (had && !(ok = dq_2())) break;
          product_slices<D, 128, 128>(tmem_base + kS2, q_addr, k_tile(g), idesc_s, D / 32, D / 32);
          tc_commit(&bars->s2_full);
          if (j + 1 == nb) tc_commit(&bars->q_free);  // Q and dO may be replaced
          if (nb > 2 && j + 3 == nb) mbar_arrive(&bars->sched_go);
          held = g, held_first = j == 0, held_last = j + 1 == nb, held_fix = fix && held_last;
        }
        G += nb;
        ++ni;
      }
    }
  } else if (warp < kComputeWarps) {
    // ---- elementwise warps: thread = (row, 32-column quarter) ----
    const int cq = warp >> 2, quarter = warp & 3;
    const int row_in_tile = quarter * 32 + lane;
    const uint32_t t_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + cq * 32;
    const float* stats = sStats + row_in_tile / kStatRows * kDqStatFloats + row_in_tile % kStatRows;
    const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
    int G = 0, ni = 0, pending = -1;  // pending: the item whose dQ is still to be stored
    bool ok = true;
    float nl1 = 0.f, nl2 = 0.f, nd1 = 0.f, nd2 = 0.f;
    // dS = P o (dP - delta), in place of the scores
    auto elementwise = [&](uint32_t t_s, const uint32_t (&dp)[32], uint32_t (&s)[32], float nl, float nd, int limit) {
      const float2 l = make_float2(nl, nl), d = make_float2(nd, nd);
      float2 x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = ffma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, l);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = exp2_of_pair<8>(i, x[i]);
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 v = fmul2(x[i], fadd2(make_float2(__uint_as_float(dp[2 * i]), __uint_as_float(dp[2 * i + 1])), d));
        pk[i] = pack_half2(v.x, v.y);
      }
      if (limit < 31) {  // by selection: the scores and dP of a masked column may be NaN (rows of the next sequence)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (2 * i > limit) pk[i] &= 0xffff0000u;
          if (2 * i + 1 > limit) pk[i] &= 0x0000ffffu;
        }
      }
      tmem_st16(t_s, pk);
    };
    for (int n = 0; ok; ++n) {
      ok = wait_item(n);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      const DiffDqItem* it = &bars->items[n % kDqSlots];  // stays in its slot until this warp has stored its dQ
      const int nb = it->nb, sk = it->sk, shift = it->shift, row = it->row0 + row_in_tile;
      int j = 0;
      do {
        uint32_t dp[32];
        int limit = 0;
        const int g = G + j;
        if (j < nb) {
          if (!(ok = mbar_wait_warp(&bars->s1_full, g & 1, ctx))) break;
          tc_fence_after_sync();
          uint32_t s[32];
          tmem_ld32(t_base + kS1, s);
          tmem_ld32(t_base + kDP, dp);
          if (j == 0) {  // S_1 of the item was issued after its statistics had landed
            nl1 = stats[0], nl2 = stats[kStatRows], nd1 = stats[2 * kStatRows], nd2 = stats[3 * kStatRows];
          }
          tmem_wait_ld();
          if (j == 0) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->q_free);  // the statistics are in registers
          }
          const int col0 = j * kBlock + cq * 32;
          limit = sk - 1 - col0;
          if (p.is_causal) limit = min(limit, row + shift - col0);
          elementwise(t_base + kS1, dp, s, nl1, nd1, limit);
          warp_arrive(&bars->ds1_full, lane);
        }
        // ---- epilogue of the item before: dQ_m = scale * acc, with the weight of map 2 ----
        if (j == 0 && pending >= 0) {
          if (!(ok = mbar_wait_warp(&bars->acc_full, ni & 1, ctx))) break;
          ++ni;
          tc_fence_after_sync();
          if (cq < D / 32) {
            const DiffDqItem* done = &bars->items[pending % kDqSlots];
            const int first = done->row0 + quarter * 32;
            uint32_t r[32];
            tmem_ld32(t_base + kAcc, r);
            tmem_wait_ld();
            const float mul = 2 * cq < D / 32 ? p.scale : -done->lam * p.scale;
            store_scaled_rows(p.dq + done->bq * p.dq_batch_stride + static_cast<int64_t>(done->q_off + first) * p.dq_row_stride +
                                  done->head * p.dq_head_stride + cq * 32,
                              p.dq_row_stride, done->sq - first, r, mul, lane);
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->acc_free);
          if (lane == 0) release_item(pending);
          pending = -1;
        }
        if (j < nb) {
          if (!(ok = mbar_wait_warp(&bars->s2_full, g & 1, ctx))) break;
          tc_fence_after_sync();
          uint32_t s[32];
          tmem_ld32(t_base + kS2, s);
          tmem_wait_ld();
          elementwise(t_base + kS2, dp, s, nl2, nd2, limit);
          warp_arrive(&bars->ds2_full, lane);
        }
      } while (++j < nb);
      if (!ok || nb < 0) break;
      if (nb > 0) {
        pending = n;
        G += nb;
      } else {  // no key is visible to any row
        if (cq < D / 32 && row < it->sq) {
          __half* to = p.dq + it->bq * p.dq_batch_stride + static_cast<int64_t>(it->q_off + row) * p.dq_row_stride +
                       it->head * p.dq_head_stride + cq * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(to + i * 8) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
        if (lane == 0) release_item(n);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (bars->abort_flag) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
    __syncthreads();
  }
  // the dK/dV kernel may still be running: this launch must not complete before it
  if (blockIdx.x == 0 && threadIdx.x == 0) grid_dependency_wait();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// =============================================================================================
// dK/dV kernel
// =============================================================================================
// TMEM: S_1^T [0, 64), S_2^T [64, 128), dP^T [128, 192), packed P^T [192, 224) and dS_1^T [224, 256), dV [256, 256 + D), dK behind it; the
// packed dS_2^T lies in the threads' own columns of dP^T.  Q tiles of 64 rows, because three score tiles of 128 columns do not fit beside the
// accumulators of D = 128; a thread then holds 16 columns of each and both P in 32 bits.
// Per tile: scores into registers (handed back, S of the next tile is issued), exponentials, dP^T waited for (which says that the products
// of the tile before are over, and with them their packed operands), P^T and dS_m^T written and handed over together; then dV, dK_1, dK_2
// and dP^T of the next tile run under its exponentials.
// B2 S4096 H16 D128 without mask 550-590 us by itself: 2150 clocks a tile of both maps, of which 1139 are products and 896 exponentials (tensor
// pipe 53 % busy, shared memory 69 %, of it 53 the products' operands, issue slots 0.50).  Bound by the chain of a warp (barriers, TMEM loads, exponentials,
// stores): with room for two of dP and the packed operands (D = 64, where the columns are 128, 256 and 320 on) the products of a tile are not waited for by
// the next, which gained 2 %; dK_2 and dP of the next tile ahead of dV and dK_1 at D = 128 lost 3 %.
constexpr int kQRows = 64;
constexpr int kDkvThreads = 640;
constexpr int kLamWarp = 19;  // sums dlam of a head while the others work: at the end of a launch it would be waited for
static_assert((kDkvThreads / 32 + 3) / 4 * 32 * 96 <= 16384, "register file of one SM sub-partition");

struct __align__(16) DiffDkvItem {
  int batch, head_k, nblk, q_off;  // nblk < 0: no more work
  int k_off, sq, sk, pad;
};
constexpr int kMaxQStages = 8;
struct DiffDkvBarriers {
  uint64_t kv_full, kv_free;
  uint64_t q_full[kMaxQStages], q_empty[kMaxQStages];  // Q, dO and statistics of a tile
  uint64_t s_full, s_loaded, dp_full[2], ds_full[2], acc_full;  // [2]: in turn, where a role may be a tile ahead
  uint64_t tail_fixed[kMaxQStages];
  uint64_t sched_full[2], sched_empty[2], sched_go;
  DiffDkvItem items[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(DiffDkvBarriers) <= 512, "barrier block");

template <int D>
struct DkvCfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kKvChunkBytes = 128 * 128, kKvTileBytes = kChunks * kKvChunkBytes;
  static constexpr int kQChunkBytes = kQRows * 128, kQTileBytes = kChunks * kQChunkBytes;
  static constexpr int kExtBytes = kQRows * 128, kOnesBytes = 1024, kStatBytes = kStatRows * 4;
  static constexpr int kStages = D == 128 ? 4 : 7;
  static constexpr int kAlignPad = D == 128 ? 0 : 1024;  // no room: the kernel checks that its memory starts on 1024 bytes
  static constexpr int kSmemBytes = 2 * kKvTileBytes + kOnesBytes + kStages * (2 * kQTileBytes + kExtBytes + kStatBytes) + 512 + kAlignPad;
  static_assert(kSmemBytes <= 227 * 1024 && kStages <= kMaxQStages, "shared memory budget");
};

struct DiffDkvWork {
  int batch, head_k, q_off, k_off, sq, sk, key0, nq, i_min, shift, per_head, n_it;
};
__device__ __forceinline__ DiffDkvWork decode_dkv(const DiffKernelParams& p, const DiffDkvItem& it) {
  DiffDkvWork w;
  w.batch = it.batch, w.head_k = it.head_k, w.q_off = it.q_off, w.k_off = it.k_off, w.sq = it.sq, w.sk = it.sk;
  w.key0 = it.nblk * kBlock;
  w.shift = (p.is_causal == 2) ? p.causal_shift : w.sk - w.sq;  // key j visible to query i iff j <= i + shift
  w.sq = min(w.sq, p.seqlen_q);  // rows past max_seqlen_q have no statistics
  w.nq = (w.sq + kQRows - 1) / kQRows;
  w.i_min = 0;
  if (p.is_causal) {
    const int first_row = w.key0 - w.shift;  // first query row that can see key0
    w.i_min = first_row <= 0 ? 0 : first_row / kQRows;
  }
  w.per_head = max(0, w.nq - w.i_min);
  w.n_it = w.per_head * p.group;
  return w;
}

// Rows of a 64-row tile from first_row on, as zero_tile_rows_from()
template <int D>
__device__ __forceinline__ void zero_q_rows_from(uint8_t* tile, int first_row, int lane) {
  using C = DkvCfg<D>;
  for (int idx = lane; idx < (kQRows - first_row) * C::kChunks * 8; idx += 32) {
    const int r = first_row + idx / (C::kChunks * 8), u = idx % (C::kChunks * 8);
    *reinterpret_cast<uint4*>(tile + (u >> 3) * C::kQChunkBytes + r * 128 + (u & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

template <int D, bool kVarlen>
__global__ void __launch_bounds__(kDkvThreads, 1) diff_dkdv_kernel(const __grid_constant__ DiffKernelParams p) {
  using C = DkvCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int stop_probe = stop_probe_begin(p.status);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  if (smem - smem_raw > C::kAlignPad) {  // uniform over the CTA: nothing has been set up yet
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, kStatusSmemLayout);
    grid_dependency_wait();
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::kKvTileBytes;
  uint8_t* sQ = sV + C::kKvTileBytes;
  uint8_t* sdO = sQ + C::kStages * C::kQTileBytes;
  uint8_t* sExt = sdO + C::kStages * C::kQTileBytes;
  uint8_t* sOnes = sExt + C::kStages * C::kExtBytes;  // eight rows of the constants of split3(), for all groups of eight keys
  float* sStats = reinterpret_cast<float*>(sOnes + C::kOnesBytes);
  DiffDkvBarriers* bars = reinterpret_cast<DiffDkvBarriers*>(sStats + C::kStages * kStatRows);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kAhead = D == 64 ? 2 : 1;  // buffers of dP^T and the packed operands
  constexpr int kS1 = 0, kS2 = 64, kDP = 128, kP = kDP + kAhead * 64, kDS1 = kP + kAhead * 32, kAccV = kDS1 + kAhead * 32, kAccK = kAccV + D;
  static_assert(kAccK + D <= kTmemCols, "TMEM");

  if (warp == kProducerWarp && lane == 0) {
    mbar_init(&bars->kv_full, 1);
    mbar_init(&bars->kv_free, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 1);
      mbar_init(&bars->tail_fixed[i], 1);
    }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->s_loaded, kComputeWarps);
    for (int i = 0; i < 2; ++i) mbar_init(&bars->dp_full[i], 1), mbar_init(&bars->ds_full[i], kComputeWarps);
    mbar_init(&bars->acc_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->sched_full[i], 1);
      mbar_init(&bars->sched_empty[i], kDiffReaders);
    }
    mbar_init(&bars->sched_go, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    grid_dependency_wait();  // the row statistics; everything behind the synchronisation below may read them
    fence_acq_rel_gpu();     // ... and so may the dQ kernel, which starts behind the next line without a wait of its own
    grid_launch_dependents();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 0) {
    for (int u = lane; u < 64; u += 32) {  // 16-byte units of the eight rows; slices 0 to 2 begin at units 0, 2, 4
      const int row = u >> 3, unit = u & 7;
      const bool constants = (unit & 1) == 0 && unit < 6;
      *reinterpret_cast<uint4*>(sOnes + row * 128 + ((unit ^ row) << 4)) =
          constants ? make_uint4(pack_half2(0x1p15f, 0x1p4f), pack_half2(0x1p-8f, 0.f), 0u, 0u) : make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before_sync();
  const bool stop = __syncthreads_or(stop_probe) != 0;
  tc_fence_after_sync();
  const uint32_t tmem_base = bars->tmem_base;
  WaitCtx ctx{&bars->abort_flag, p.status};
  auto read_item = [&](int n, DiffDkvItem& it) -> bool {
    if (!mbar_wait(&bars->sched_full[n & 1], (n >> 1) & 1, ctx)) return false;
    it = bars->items[n & 1];
    return true;
  };
  auto release_item = [&](int n) { mbar_arrive(&bars->sched_empty[n & 1]); };

  if (stop) {
  } else if (warp == kLamWarp) {
    for (int head = blockIdx.x; head < p.h; head += gridDim.x) sum_dlam(p, head, lane);
  } else if (warp == kDiffSched) {
    if (lane == 0) {
      bool finished = false;
      int seq = 0;
      for (int n = 0;; ++n) {
        int next = blockIdx.x;
        if (n > 0) {
          if (!mbar_wait(&bars->sched_go, (n - 1) & 1, ctx)) break;
          next = gridDim.x + atomicAdd(p.sched, 1);
        }
        DiffDkvItem it;
        it.batch = 0, it.head_k = 0, it.nblk = -1, it.pad = 0, it.q_off = 0, it.k_off = 0;
        it.sq = p.seqlen_q, it.sk = p.seqlen_k;
        if constexpr (!kVarlen) {
          if (next < p.total_items) {  // every index is a live item: key tile 0 of a head is the heaviest
            const HeadPlace at = section_item(next, p.h_k * p.b, p.items_x, 1, p.seqlen_q, p.section_rows);
            it.batch = at.head / p.h_k, it.head_k = at.head - it.batch * p.h_k, it.nblk = at.place;
          }
        } else {
          while (next < p.total_items) {  // slots per sequence from cu_seqlens_k / 128
            while (seq + 1 < p.b && p.h_k * ((p.cu_seqlens_k[seq + 1] >> 7) + seq + 1) <= next) ++seq;
            const int k0 = p.cu_seqlens_k[seq], k1 = p.cu_seqlens_k[seq + 1];
            const int v0 = (k0 >> 7) + seq, v1 = (k1 >> 7) + seq + 1;
            const int rel = next - p.h_k * v0, cnt = v1 - v0;
            if (rel >= 0 && rel < p.h_k * cnt) {
              it.q_off = p.cu_seqlens_q[seq], it.sq = p.cu_seqlens_q[seq + 1] - it.q_off;
              const HeadPlace at = section_item(rel, p.h_k, cnt, 1, it.sq, p.section_rows);
              if (at.place < p.items_x && at.place * kBlock < k1 - k0) {  // items_x: key tiles up to max_seqlen_k
                it.batch = seq, it.head_k = at.head, it.nblk = at.place;
                it.k_off = k0, it.sk = k1 - k0;
                break;
              }
            }
            next = gridDim.x + atomicAdd(p.sched, 1);
          }
        }
        if (!mbar_wait(&bars->sched_empty[n & 1], ((n >> 1) & 1) ^ 1, ctx)) break;
        bars->items[n & 1] = it;
        mbar_arrive(&bars->sched_full[n & 1]);
        if (it.nblk < 0) {
          finished = true;
          break;
        }
      }
      if (finished) {
        __threadfence();
        if (atomicAdd(p.sched + 1, 1) == static_cast<int>(gridDim.x) - 1) {
          atomicExch(p.sched, 0);
          atomicExch(p.sched + 1, 0);
        }
      }
    }
  } else if (warp == kProducerWarp) {
    int T0 = 0, ni = 0;
    for (int n = 0;; ++n) {
      DiffDkvItem item;
      bool ok = read_item(n, item);
      if (!__all_sync(0xffffffffu, ok)) break;
      __syncwarp();
      if (lane == 0) release_item(n);
      if (item.nblk < 0) break;
      const DiffDkvWork w = decode_dkv(p, item);
      if (w.n_it == 0) continue;
      const int bq = kVarlen ? 0 : w.batch;
      auto load_q_do = [&](int it) -> bool {
        const int T = T0 + it, s = T % C::kStages;
        const int head = w.head_k * p.group + it / w.per_head, i = w.i_min + it % w.per_head;
        const int64_t tile = first_stat_tile(kVarlen, w.q_off, w.batch, head, p.h, p.stat_tiles) + i;
        if (!mbar_wait(&bars->q_empty[s], ((T / C::kStages) & 1) ^ 1, ctx)) return false;
        mbar_arrive_expect_tx(&bars->q_full[s], 2 * C::kQTileBytes + C::kExtBytes + C::kStatBytes);
        bulk_load_1d(sStats + s * kStatRows, p.stats + tile * kStatFloats + 4 * kStatRows, C::kStatBytes, &bars->q_full[s]);
        tma_load_4d(sExt + s * C::kExtBytes, &p.tm_ext, &bars->q_full[s], 0, 0, static_cast<int>(tile) * kStatRows, 0);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
          tma_load_4d(sQ + s * C::kQTileBytes + c * C::kQChunkBytes, &p.tm_q, &bars->q_full[s], c * 64, head, w.q_off + i * kQRows, bq);
          tma_load_4d(sdO + s * C::kQTileBytes + c * C::kQChunkBytes, &p.tm_do, &bars->q_full[s], c * 64, head, w.q_off + i * kQRows, bq);
        }
        return true;
      };
      if (lane == 0) {
        ok = mbar_wait(&bars->kv_free, (ni & 1) ^ 1, ctx);
        if (ok) {
          mbar_arrive_expect_tx(&bars->kv_full, 2 * C::kKvTileBytes);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c) {
            tma_load_4d(sK + c * C::kKvChunkBytes, &p.tm_k, &bars->kv_full, c * 64, w.head_k, w.k_off + w.key0, bq);
            tma_load_4d(sV + c * C::kKvChunkBytes, &p.tm_v, &bars->kv_full, c * 64, w.head_k, w.k_off + w.key0, bq);
          }
        }
      }
      if (!kVarlen || (w.sq % kQRows) == 0) {
        if (lane == 0) {
          for (int it = 0; ok && it < w.n_it; ++it) ok = load_q_do(it);
        }
      } else {
        // the whole warp walks the tiles: lane 0 issues the loads, all lanes zero the rows of the next sequence
        ok = __all_sync(0xffffffffu, ok);
        for (int it = 0; ok && it < w.n_it; ++it) {
          if (lane == 0) ok = load_q_do(it);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          if (it % w.per_head == w.per_head - 1) {  // the last Q tile of this head
            const int T = T0 + it, s = T % C::kStages;
            if (!(ok = mbar_wait_warp(&bars->q_full[s], (T / C::kStages) & 1, ctx))) break;
            const int tail = w.sq - (w.nq - 1) * kQRows;
            zero_q_rows_from<D>(sQ + s * C::kQTileBytes, tail, lane);
            zero_q_rows_from<D>(sdO + s * C::kQTileBytes, tail, lane);
            if (lane == 0) mbar_arrive(&bars->tail_fixed[s]);
          }
        }
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      T0 += w.n_it;
      ++ni;
    }
  } else if (warp == kMmaWarp) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_f16(128, kQRows, false, false);
      constexpr uint32_t idesc_dv = make_idesc_f16(128, D, false, true), idesc_dk = make_idesc_f16(128, D / 2, false, true);
      const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, ctx); };
      auto q_tile = [&](int T) { return smem_u32(sQ + (T % C::kStages) * C::kQTileBytes); };
      auto do_tile = [&](int T) { return smem_u32(sdO + (T % C::kStages) * C::kQTileBytes); };
      auto q_full = [&](int T) { return wait(&bars->q_full[T % C::kStages], (T / C::kStages) & 1); };
      const uint64_t ones = make_smem_desc(smem_u32(sOnes), 16, 0);  // the same eight rows for every group of eight
      auto statistics = [&](uint32_t d_tmem, int T, int slice) {  // their slice
        const uint64_t ext = make_smem_desc(smem_u32(sExt + (T % C::kStages) * C::kExtBytes), 16, 1024);
        mma_ss(d_tmem, desc_advance(ones, slice * 32), desc_advance(ext, slice * 32), idesc_s, 1u);
      };
      auto scores = [&](int T) {  // S_m^T = K_m Q_m^T - LSE_m / c
        product_slices<D, 128, kQRows>(tmem_base + kS1, k_addr, q_tile(T), idesc_s, 0, D / 32);
        statistics(tmem_base + kS1, T, 0);
        product_slices<D, 128, kQRows>(tmem_base + kS2, k_addr, q_tile(T), idesc_s, D / 32, D / 32);
        statistics(tmem_base + kS2, T, 1);
        tc_commit(&bars->s_full);
      };
      auto dp = [&](int T) {  // dP^T = V dO^T - delta_1
        const uint32_t to = tmem_base + kDP + T % kAhead * 64;
        product_slices<D, 128, kQRows>(to, v_addr, do_tile(T), idesc_s, 0, D / 16);
        statistics(to, T, 2);
        tc_commit(&bars->dp_full[T % kAhead]);
      };
      int T0 = 0, ni = 0;
      uint32_t tail_phase = 0;  // bit s: parity of the next tail_fixed[s] phase to wait for
      bool ok = true;
      for (int n = 0; ok; ++n) {
        DiffDkvItem item;
        if (!(ok = read_item(n, item))) break;
        release_item(n);
        if (item.nblk < 0) break;
        const DiffDkvWork w = decode_dkv(p, item);
        constexpr int kGoAhead = 4;  // the next item is claimed so many tiles before this one ends
        if (w.n_it <= kGoAhead) mbar_arrive(&bars->sched_go);
        if (w.n_it == 0) continue;
        if (!(ok = wait(&bars->kv_full, ni & 1) && q_full(T0))) break;
        if (T0 > 0 && !(ok = wait(&bars->s_loaded, (T0 - 1) & 1))) break;
        tc_fence_after_sync();
        scores(T0);
        dp(T0);
        if (w.n_it == 1) tc_commit(&bars->kv_free);
        if (kAhead == 2 && w.n_it > 1) {
          if (!(ok = q_full(T0 + 1))) break;
          dp(T0 + 1);
        }
        for (int it = 0; ok && it < w.n_it; ++it) {
          const int T = T0 + it, s = T % C::kStages;
          if (it + 1 < w.n_it) {
            if (!(ok = q_full(T + 1) && wait(&bars->s_loaded, T & 1))) break;
            tc_fence_after_sync();
            scores(T + 1);
            if (kAhead == 2 && it + 2 == w.n_it) tc_commit(&bars->kv_free);  // K and V may be replaced
          }
          if (!(ok = wait(&bars->ds_full[T % kAhead], (T / kAhead) & 1))) break;
          if (kVarlen && (w.sq % kQRows) != 0 && it % w.per_head == w.per_head - 1) {
            if (!(ok = wait(&bars->tail_fixed[s], (tail_phase >> s) & 1))) break;
            tail_phase ^= 1u << s;
          }
          tc_fence_after_sync();
          {  // dV += P^T dO
            const uint64_t bd = make_smem_desc(do_tile(T), C::kQChunkBytes, 1024);
#pragma unroll
            for (int k = 0; k < kQRows / 16; ++k)
              mma_ts(tmem_base + kAccV, tmem_base + kP + T % kAhead * 32 + k * 8, desc_advance(bd, k * 2048), idesc_dv, (it == 0 && k == 0) ? 0u : 1u);
          }
          product_half<D, kQRows>(tmem_base + kAccK, tmem_base + kDS1 + T % kAhead * 32, [](int k) { return k * 8; }, q_tile(T), 0, idesc_dk, it == 0);
          product_half<D, kQRows>(tmem_base + kAccK + D / 2, tmem_base + kDP + T % kAhead * 64, [](int k) { return k * 16; }, q_tile(T), 1, idesc_dk, it == 0);
          tc_commit(&bars->q_empty[s]);
          if (it + kAhead < w.n_it) {
            if (kAhead == 2 && !(ok = q_full(T + 2))) break;
            dp(T + kAhead);
            if (kAhead == 1 && it + 2 == w.n_it) tc_commit(&bars->kv_free);  // K and V may be replaced
          }
          if (w.n_it > kGoAhead && it + kGoAhead + 1 == w.n_it) mbar_arrive(&bars->sched_go);
        }
        if (ok) tc_commit(&bars->acc_full);
        T0 += w.n_it;
        ++ni;
      }
    }
  } else if (warp < kComputeWarps) {
    // ---- elementwise warps: thread = (key row, 16 query columns) ----
    const int cq = warp >> 2, quarter = warp & 3;
    const int row_in_tile = quarter * 32 + lane;
    const uint32_t t_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
    constexpr int kEvery = D == 64 ? 4 : 8;
    int T0 = 0, ni = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      int n_it, per_head, cmin0, cmax_last, head;
      {
        DiffDkvItem item;
        ok = read_item(n, item);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (item.nblk < 0) break;
        const DiffDkvWork w = decode_dkv(p, item);
        n_it = w.n_it, per_head = w.per_head, head = w.head_k * p.group;
        // valid columns in the last Q tile
        cmax_last = kVarlen ? max(0, min(16, w.sq - (w.nq - 1) * kQRows - cq * 16)) : 16;
        // causal: the columns of this thread below  key - shift - (i * 64 + cq * 16)  are masked
        cmin0 = p.is_causal ? (w.key0 + row_in_tile) - w.shift - (w.i_min * kQRows + cq * 16) : 0;
      }
      int i_rel = 0;  // Q tile within the current head
      float lam = 0.f;
      for (int it = 0; it < n_it; ++it) {
        const int T = T0 + it;
        if (i_rel == 0) lam = weight_of(p.weights, head);
        if (!(ok = mbar_wait_warp(&bars->s_full, T & 1, ctx))) break;
        tc_fence_after_sync();
        uint32_t s1[16], s2[16];
        tmem_ld16(t_base + kS1 + cq * 16, s1);
        tmem_ld16(t_base + kS2 + cq * 16, s2);
        tmem_wait_ld();
        warp_arrive_loaded(&bars->s_loaded, lane);  // the scores of the next tile may come
        float2 p1[8], p2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p1[e] = exp2_of_pair<kEvery>(e, fmul2(make_float2(__uint_as_float(s1[2 * e]), __uint_as_float(s1[2 * e + 1])), c2));
          p2[e] = exp2_of_pair<kEvery>(e, fmul2(make_float2(__uint_as_float(s2[2 * e]), __uint_as_float(s2[2 * e + 1])), c2));
        }
        const int cmin = max(0, min(16, cmin0 - i_rel * kQRows)), cmax = kVarlen && i_rel == per_head - 1 ? cmax_last : 16;
        const bool masked = cmin > 0 || cmax < 16;
        if (++i_rel == per_head) i_rel = 0, ++head;
        const float2 minus = make_float2(-lam, -lam);
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p2[e] = fmul2(p2[e], minus);  // -lam A_2: what both dV and dS_2 take
          const float2 v = fadd2(p1[e], p2[e]);
          pk[e] = pack_half2(v.x, v.y);
        }
        // by selection: the scores and dP of a masked column may be NaN (rows of the next sequence)
        auto select = [&](uint32_t (&x)[8]) {
          if (!masked) return;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (2 * e < cmin || 2 * e >= cmax) x[e] &= 0xffff0000u;
            if (2 * e + 1 < cmin || 2 * e + 1 >= cmax) x[e] &= 0x0000ffffu;
          }
        };
        select(pk);
        // dP^T(T) complete: so are dV, dK of the tile before, which read the packed operands
        if (!(ok = mbar_wait_warp(&bars->dp_full[T % kAhead], (T / kAhead) & 1, ctx))) break;
        tc_fence_after_sync();
        uint32_t dp[16];
        const uint32_t t_dp = t_base + kDP + T % kAhead * 64 + cq * 16, t_packed = t_base + T % kAhead * 32 + cq * 8;
        tmem_ld16(t_dp, dp);
        tmem_st8(t_packed + kP, pk);
        const float4* differences = reinterpret_cast<const float4*>(sStats + (T % C::kStages) * kStatRows + cq * 16);
        tmem_wait_ld();
        uint32_t pk2[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 a = differences[e];
          const float2 x = make_float2(__uint_as_float(dp[4 * e]), __uint_as_float(dp[4 * e + 1]));
          const float2 y = make_float2(__uint_as_float(dp[4 * e + 2]), __uint_as_float(dp[4 * e + 3]));
          const float2 u0 = fmul2(p1[2 * e], x), u1 = fmul2(p1[2 * e + 1], y);
          const float2 v0 = fmul2(p2[2 * e], fadd2(x, make_float2(a.x, a.y))), v1 = fmul2(p2[2 * e + 1], fadd2(y, make_float2(a.z, a.w)));
          pk[2 * e] = pack_half2(u0.x, u0.y), pk[2 * e + 1] = pack_half2(u1.x, u1.y);
          pk2[2 * e] = pack_half2(v0.x, v0.y), pk2[2 * e + 1] = pack_half2(v1.x, v1.y);
        }
        select(pk);
        select(pk2);
        tmem_st8(t_packed + kDS1, pk);
        tmem_st8(t_dp, pk2);
        warp_arrive(&bars->ds_full[T % kAhead], lane);
      }
      if (!ok) break;
      // ---- epilogue: column quarters 0,1 store the halves of dV, quarters 2,3 the halves of dK * scale ----
      DiffDkvItem item;
      {
        const volatile int* src = reinterpret_cast<const volatile int*>(&bars->items[n & 1]);
        item.batch = src[0], item.head_k = src[1], item.nblk = src[2], item.q_off = src[3];
        item.k_off = src[4], item.sq = src[5], item.sk = src[6], item.pad = 0;
      }
      const DiffDkvWork w = decode_dkv(p, item);
      const int key = w.key0 + row_in_tile, which = cq >> 1, col_half = cq & 1;
      __half* dst_base = which == 0 ? p.dv : p.dk;
      const int64_t bs = which == 0 ? p.dv_batch_stride : p.dk_batch_stride;
      const int64_t rs = which == 0 ? p.dv_row_stride : p.dk_row_stride;
      const int64_t hs = which == 0 ? p.dv_head_stride : p.dk_head_stride;
      __half* dst = dst_base + (kVarlen ? 0 : w.batch * bs) + static_cast<int64_t>(w.k_off + key) * rs + w.head_k * hs + col_half * (D / 2);
      if (n_it > 0) {
        if (!(ok = mbar_wait_warp(&bars->acc_full, ni & 1, ctx))) break;
        ++ni;
        tc_fence_after_sync();
#pragma unroll
        for (int q = 0; q < D / 64; ++q) {
          uint32_t r[32];
          tmem_ld32(t_base + (which == 0 ? kAccV : kAccK) + col_half * (D / 2) + q * 32, r);
          tmem_wait_ld();
          store_scaled_rows(dst - lane * rs + q * 32, rs, w.sk - (key - lane), r, which == 0 ? 1.f : p.scale, lane);
        }
        tc_fence_before_sync();
      } else if (key < w.sk) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *reinterpret_cast<uint4*>(dst + i * 8) = make_uint4(0, 0, 0, 0);
      }
      T0 += n_it;
      __syncwarp();
      if (lane == 0) release_item(n);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (bars->abort_flag) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

int round_up(int x, int m) { return (x + m - 1) / m * m; }
size_t align256(size_t x) { return (x + 255) / 256 * 256; }
// Tiles of statistics of a (batch, head); packed: of a head, with one more behind the last, which the dQ kernel reads with its pair
int64_t stat_tiles(const FaBwdParams& p) {
  return p.cu_seqlens_q ? p.total_q / kStatRows + p.b + 1 : round_up(p.seqlen_q, kBlock) / kStatRows;
}
int64_t all_stat_tiles(const FaBwdParams& p) { return stat_tiles(p) * p.h * (p.cu_seqlens_q ? 1 : p.b); }
size_t stats_bytes(const FaBwdParams& p) { return align256(all_stat_tiles(p) * kStatFloats * sizeof(float)); }
size_t ext_bytes(const FaBwdParams& p) { return all_stat_tiles(p) * kStatRows * kExtColumns * sizeof(__half); }

template <class Kernel>
int configure(Kernel kernel, int smem, bool (&done)[64]) {
  int dev = 0;
  FA_CHECK_CUDA(cudaGetDevice(&dev));
  if (!done[dev & 63]) {
    FA_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done[dev & 63] = true;
  }
  return FA_OK;
}

// One launch of a persistent kernel
template <class Kernel>
int launch_persistent(Kernel kernel, DiffKernelParams kp, int64_t total, int threads, int smem, cudaStream_t stream) {
  const int sms = device_sm_count();
  kp.sched = next_sched_slot(stream);
  if (sms <= 0 || kp.sched == nullptr) return set_error(FA_ERR_CUDA, "fa_diff_bwd: device attributes not available");
  FA_CHECK_ARG(total < (1ll << 30), "fa_diff_bwd: too many work items");
  kp.total_items = static_cast<int>(total);
  FA_CHECK_CUDA(launch_overlapped(kernel, dim3(std::min(kp.total_items, sms)), threads, smem, stream, kp));
  return FA_OK;
}

// The kernels overlap as those of the plain backward do, the other way round: the dK/dV kernel waits for the statistics and then lets the
// dQ kernel start, which reads nothing that it writes, on the SMs that it leaves.  Its items are long ones (a key tile of a KV head times all
// queries of the group), those of the dQ kernel short, and what is left at the end of the launch is a short one then.
template <int D>
int launch(const FaBwdParams& b, DiffKernelParams kp, const CUtensorMap& q64, const CUtensorMap& do64, cudaStream_t stream) {
  static bool dq_done[64] = {}, dense_done[64] = {}, varlen_done[64] = {};
  int rc = configure(diff_dq_kernel<D>, DqCfg<D>::kSmemBytes, dq_done);
  if (rc == FA_OK) rc = configure(diff_dkdv_kernel<D, false>, DkvCfg<D>::kSmemBytes, dense_done);
  if (rc == FA_OK) rc = configure(diff_dkdv_kernel<D, true>, DkvCfg<D>::kSmemBytes, varlen_done);
  if (rc != FA_OK) return rc;
  const bool varlen = kp.cu_seqlens_q != nullptr;
  DiffKernelParams kk = kp;
  kk.tm_q = q64, kk.tm_do = do64;
  kk.items_x = (b.seqlen_k + kBlock - 1) / kBlock;
  kk.section_rows = section_rows(b.is_causal != 0, b.seqlen_q, b.seqlen_k, static_cast<int64_t>(4 * D) * kp.group);
  rc = launch_persistent(varlen ? diff_dkdv_kernel<D, true> : diff_dkdv_kernel<D, false>, kk,
                         varlen ? static_cast<int64_t>(b.h_k) * (b.total_k / kBlock + b.b) : static_cast<int64_t>(kk.items_x) * b.h_k * b.b,
                         kDkvThreads, DkvCfg<D>::kSmemBytes, stream);
  if (rc != FA_OK) return rc;
  kp.items_x = (b.seqlen_q + kBlock - 1) / kBlock;
  kp.section_rows = section_rows(b.is_causal != 0, b.seqlen_q, b.seqlen_k, 4 * D);
  return launch_persistent(diff_dq_kernel<D>, kp,
                           varlen ? static_cast<int64_t>(b.h) * (b.total_q / kBlock + b.b) : static_cast<int64_t>(kp.items_x) * b.h * b.b,
                           kDiffThreads, DqCfg<D>::kSmemBytes, stream);
}

}  // namespace
}  // namespace fa

extern "C" size_t fa_diff_bwd_workspace_bytes(const FaDiffBwdParams* p) {
  using namespace fa;
  if (p == nullptr || p->base.b < 1 || p->base.h < 1 || p->base.seqlen_q < 1 || p->base.total_q < 0) return 0;
  return stats_bytes(p->base) + ext_bytes(p->base) + align256(static_cast<size_t>(p->base.h) * sizeof(float));
}

extern "C" int fa_diff_bwd(const FaDiffBwdParams* p, fa_stream_t stream_) {
  using namespace fa;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  FA_CHECK_ARG(p != nullptr, "fa_diff_bwd: params is NULL");
  const FaBwdParams& b = p->base;
  FA_CHECK_ARG(b.q && b.k && b.v && b.o && p->o2 && b.dout && b.lse && b.dq && b.dk && b.dv && p->dlam,
               "fa_diff_bwd: q, k, v, o, o2, dout, lse, dq, dk, dv, dlam must be non-NULL");
  if (b.d != 64 && b.d != 128) return set_error(FA_ERR_UNSUPPORTED, "fa_diff_bwd: head_dim must be 64 or 128");
  FA_CHECK_ARG(b.b >= 1 && b.h >= 1 && b.h_k >= 1 && b.h % b.h_k == 0, "fa_diff_bwd: bad b / h / h_k");
  FA_CHECK_ARG(b.seqlen_q >= 1 && b.seqlen_k >= 1, "fa_diff_bwd: bad sequence lengths");
  FA_CHECK_ARG((b.cu_seqlens_q == nullptr) == (b.cu_seqlens_k == nullptr), "fa_diff_bwd: cu_seqlens_q and cu_seqlens_k go together");
  FA_CHECK_ARG(b.lse_row_stride >= b.seqlen_q, "fa_diff_bwd: lse_row_stride is smaller than seqlen_q");
  FA_CHECK_ARG(b.is_causal >= 0 && b.is_causal <= 2 && (b.is_causal != 2 || b.cu_seqlens_q == nullptr), "fa_diff_bwd: bad is_causal");
  FA_CHECK_ARG((b.flags & ~FA_BWD_ZERO_UNUSED_ROWS) == 0, "fa_diff_bwd: flags must be 0 or FA_BWD_ZERO_UNUSED_ROWS");
  int rc = check_weights(p->weights, b.h, b.softmax_scale, "fa_diff_bwd");
  if (rc != FA_OK) return rc;
  const bool varlen = b.cu_seqlens_q != nullptr;
  {
    const void* ptrs[] = {b.o, p->o2, b.dout, b.dq, b.dk, b.dv};
    for (const void* x : ptrs) FA_CHECK_ARG(aligned16(x), "fa_diff_bwd: o, o2, dout, dq, dk, dv must be 16-byte aligned");
    const int64_t strides[] = {b.o_row_stride, b.o_head_stride, p->o2_row_stride, p->o2_head_stride, b.do_row_stride, b.do_head_stride,
                               b.dq_row_stride, b.dq_head_stride, b.dk_row_stride, b.dk_head_stride, b.dv_row_stride, b.dv_head_stride};
    for (int64_t s : strides) FA_CHECK_ARG(s % 8 == 0, "fa_diff_bwd: strides must be multiples of 8 elements");
    const int64_t batch_strides[] = {b.o_batch_stride, p->o2_batch_stride, b.do_batch_stride, b.dq_batch_stride, b.dk_batch_stride, b.dv_batch_stride};
    for (int64_t s : batch_strides) FA_CHECK_ARG(varlen || s % 8 == 0, "fa_diff_bwd: batch strides must be multiples of 8 elements");
  }
  if (b.workspace == nullptr || b.workspace_bytes < fa_diff_bwd_workspace_bytes(p))
    return set_error(FA_ERR_WORKSPACE, "fa_diff_bwd: workspace smaller than fa_diff_bwd_workspace_bytes()");
  FA_CHECK_ARG((reinterpret_cast<uintptr_t>(b.workspace) & 255) == 0, "fa_diff_bwd: workspace must be 256-byte aligned");
  rc = check_device_sm100();
  if (rc != FA_OK) return rc;

  DiffKernelParams kp = {};
  CUtensorMap q64, do64;
  const int64_t q_rows = varlen ? b.total_q : b.seqlen_q, k_rows = varlen ? b.total_k : b.seqlen_k, nb = varlen ? 1 : b.b;
  FA_CHECK_ARG(q_rows >= 1 && k_rows >= 1, "fa_diff_bwd: empty q or k");
  const int64_t ext_rows = all_stat_tiles(b) * kStatRows;
  FA_CHECK_ARG(ext_rows < (1ll << 31), "fa_diff_bwd: too many rows");
  auto map = [&](CUtensorMap* to, const void* x, int heads, int64_t rows, int64_t hs, int64_t rs, int64_t bs, int box, const char* what) {
    if (rc == FA_OK) rc = make_tensor_map_4d(to, x, b.d, heads, rows, nb, hs, rs, bs, box, what);
  };
  map(&kp.tm_q, b.q, b.h, q_rows, b.q_head_stride, b.q_row_stride, b.q_batch_stride, kBlock, "fa_diff_bwd: q");
  map(&q64, b.q, b.h, q_rows, b.q_head_stride, b.q_row_stride, b.q_batch_stride, kQRows, "fa_diff_bwd: q");
  map(&kp.tm_do, b.dout, b.h, q_rows, b.do_head_stride, b.do_row_stride, b.do_batch_stride, kBlock, "fa_diff_bwd: dout");
  map(&do64, b.dout, b.h, q_rows, b.do_head_stride, b.do_row_stride, b.do_batch_stride, kQRows, "fa_diff_bwd: dout");
  map(&kp.tm_k, b.k, b.h_k, k_rows, b.k_head_stride, b.k_row_stride, b.k_batch_stride, kBlock, "fa_diff_bwd: k");
  map(&kp.tm_v, b.v, b.h_k, k_rows, b.v_head_stride, b.v_row_stride, b.v_batch_stride, kBlock, "fa_diff_bwd: v");
  if (rc != FA_OK) return rc;

  DiffPreParams pp = {};
  pp.o = static_cast<const __half*>(b.o), pp.o2 = static_cast<const __half*>(p->o2), pp.dout = static_cast<const __half*>(b.dout);
  pp.lse = b.lse;
  pp.stats = static_cast<float*>(b.workspace);
  pp.ext = reinterpret_cast<__half*>(static_cast<uint8_t*>(b.workspace) + stats_bytes(b));
  pp.inv_scale_log2 = 1.f / (b.softmax_scale * kLog2e);
  pp.o_batch_stride = b.o_batch_stride, pp.o_row_stride = b.o_row_stride, pp.o_head_stride = b.o_head_stride;
  pp.o2_batch_stride = p->o2_batch_stride, pp.o2_row_stride = p->o2_row_stride, pp.o2_head_stride = p->o2_head_stride;
  pp.do_batch_stride = b.do_batch_stride, pp.do_row_stride = b.do_row_stride, pp.do_head_stride = b.do_head_stride;
  pp.lse_row_stride = b.lse_row_stride;
  pp.h = b.h, pp.seqlen_q = b.seqlen_q, pp.sq_pad = round_up(b.seqlen_q, kBlock), pp.stat_tiles = static_cast<int>(stat_tiles(b)), pp.d = b.d;
  pp.weights = p->weights;
  pp.cu_seqlens_q = b.cu_seqlens_q;
  const bool clears = varlen && (b.flags & FA_BWD_ZERO_UNUSED_ROWS) != 0;
  pp.clear[0] = PackedRows{static_cast<__half*>(b.dq), b.dq_row_stride, b.dq_head_stride, b.total_q, b.h, b.d, b.cu_seqlens_q, b.b};
  pp.clear[1] = PackedRows{static_cast<__half*>(b.dk), b.dk_row_stride, b.dk_head_stride, b.total_k, b.h_k, b.d, b.cu_seqlens_k, b.b};
  pp.clear[2] = PackedRows{static_cast<__half*>(b.dv), b.dv_row_stride, b.dv_head_stride, b.total_k, b.h_k, b.d, b.cu_seqlens_k, b.b};
  pp.keys_written = round_up(b.seqlen_k, kBlock);
  pp.status = device_status_ptr();
  const int64_t pre_items = static_cast<int64_t>(pp.sq_pad / kPreRows) * b.h;
  const int items_per_block = 256 / (b.d / 8);
  int64_t pre_blocks = (pre_items + items_per_block - 1) / items_per_block;
  if (clears) {  // at least a block per SM for the unused rows
    const int sms = device_sm_count();
    if (sms <= 0) return set_error(FA_ERR_CUDA, "fa_diff_bwd: device attributes not available");
    pre_blocks = std::max<int64_t>(pre_blocks, (sms + b.b - 1) / b.b);
  }
  FA_CHECK_ARG(pre_blocks < (1ll << 31) && b.b <= 65535, "fa_diff_bwd: too many rows or sequences");
  const dim3 grid_pre(static_cast<unsigned>(pre_blocks), 1, b.b);
  const auto preprocess = clears ? diff_preprocess_kernel<true> : diff_preprocess_kernel<false>;
  preprocess<<<grid_pre, 256, 0, stream>>>(pp);
  FA_CHECK_CUDA(cudaGetLastError());

  kp.dq = static_cast<__half*>(b.dq), kp.dk = static_cast<__half*>(b.dk), kp.dv = static_cast<__half*>(b.dv);
  kp.dq_batch_stride = b.dq_batch_stride, kp.dq_row_stride = b.dq_row_stride, kp.dq_head_stride = b.dq_head_stride;
  kp.dk_batch_stride = b.dk_batch_stride, kp.dk_row_stride = b.dk_row_stride, kp.dk_head_stride = b.dk_head_stride;
  kp.dv_batch_stride = b.dv_batch_stride, kp.dv_row_stride = b.dv_row_stride, kp.dv_head_stride = b.dv_head_stride;
  kp.stats = pp.stats;
  rc = make_tensor_map_4d(&kp.tm_ext, pp.ext, kExtColumns, 1, ext_rows, 1, kExtColumns, kExtColumns, 0, kQRows, "fa_diff_bwd: workspace");
  if (rc != FA_OK) return rc;
  kp.stat_tiles = pp.stat_tiles;
  kp.seqlen_q = b.seqlen_q, kp.seqlen_k = b.seqlen_k, kp.h = b.h, kp.h_k = b.h_k, kp.group = b.h / b.h_k, kp.b = b.b;
  kp.scale = b.softmax_scale, kp.scale_log2 = b.softmax_scale * kLog2e;
  kp.is_causal = b.is_causal, kp.causal_shift = b.causal_shift;
  kp.cu_seqlens_q = b.cu_seqlens_q, kp.cu_seqlens_k = b.cu_seqlens_k;
  kp.weights = p->weights;
  const bool joins = p->weights.count == 1 && b.h > 1;
  kp.head_dlam = joins ? reinterpret_cast<float*>(static_cast<uint8_t*>(b.workspace) + stats_bytes(b) + ext_bytes(b)) : nullptr;
  kp.dlam = p->dlam;
  kp.status = device_status_ptr();
  rc = b.d == 128 ? launch<128>(b, kp, q64, do64, stream) : launch<64>(b, kp, q64, do64, stream);
  if (rc != FA_OK || !joins) return rc;
  join_dlam_kernel<<<1, 32, 0, stream>>>(kp.head_dlam, b.h, p->dlam, p->weights.is_half);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}
