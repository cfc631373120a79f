// Launcher of the split-KV log-sum-exp merge, shared by fa_combine() and fa_kvcache().
#pragma once

#include "common.h"

namespace fa {

int launch_combine(const float* o_accum, const float* lse_accum, void* o, float* lse, int64_t rows,
                   int num_splits, int h, int seqlen_q, int d, int64_t o_batch_stride,
                   int64_t o_row_stride, int64_t o_head_stride, cudaStream_t stream, bool overlap = false);

// Differential attention: h counts two rows per query head, 2 * head + map, in rows, lse and the partials; o has h / 2 heads.
// Launched overlapping the kernel before.  chunk_at: see DiffSplits; kWholeChunk: there is nothing to merge.
int launch_diff_combine(const float* o_accum, const float* lse_accum, void* o, float* lse, int64_t rows,
                        int num_splits, int h, int seqlen_q, int d, int64_t o_batch_stride, int64_t o_row_stride, int64_t o_head_stride,
                        const FaDiffWeights& weights, const int* chunk_at, cudaStream_t stream);

}  // namespace fa
