// Differential attention, O = (A_1 - lam_h A_2) V with A_m = softmax(scale Q_m K_m^T), on the attention kernels.
//
// A query row whose other half of d is zero has the scores of one map: [q_1, 0] . [k_1, k_2] = q_1 . k_1.  So the two maps of a
// head are two query heads of the same KV head, and what is left is to lay the queries out that way and to subtract.  In the
// backward dO of the second map is -lam_h dO; dK and dV are sums over the query heads of a group in any case, and the halves of dK
// come from the halves of the padded queries.
#include <algorithm>

#include "diff.cuh"
#include "fwd.h"
#define FA_WAIT_INLINE
#include "ptx.cuh"

namespace fa {
namespace {

constexpr int kThreads = 256;

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// (batches, rows, heads, d) through strides; packed tensors are one batch
struct View {
  __half* base;
  int64_t batch_stride, row_stride, head_stride;
  __device__ __forceinline__ uint4* at(int64_t batch, int64_t row, int head, int unit) const {
    return reinterpret_cast<uint4*>(base + batch * batch_stride + row * row_stride + head * head_stride + unit * 8);
  }
};

struct SplitParams {
  View q, o, o2, dout;               // dout.base == nullptr: forward
  __half *q_maps, *o_maps, *do_maps; // (batches, rows, 2 h, d)
  FaDiffWeights weights;
  int64_t units;                     // batches * rows * h * (d / 8)
  int rows, h, unit_bits;
};

struct Place {
  int64_t batch, row;
  int head, unit;
};
__device__ __forceinline__ Place place_of(int64_t idx, int rows, int h, int unit_bits) {
  Place p;
  p.unit = static_cast<int>(idx) & ((1 << unit_bits) - 1);
  const int64_t rest = idx >> unit_bits, r = rest / h;
  p.head = static_cast<int>(rest - r * h);
  p.batch = r / rows;
  p.row = r - p.batch * rows;
  return p;
}

__device__ __forceinline__ uint4 scaled(uint4 x, float f, const uint4* add) {
  const __half2* h = reinterpret_cast<const __half2*>(&x);
  uint4 out;
  uint32_t* to = &out.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v = __half22float2(h[i]);
    v.x *= f, v.y *= f;
    if (add != nullptr) {
      const float2 a = __half22float2(reinterpret_cast<const __half2*>(add)[i]);
      v.x += a.x, v.y += a.y;
    }
    to[i] = pack_half2(v.x, v.y);
  }
  return out;
}

__global__ void __launch_bounds__(kThreads) split_kernel(const __grid_constant__ SplitParams p) {
  const int units = 1 << p.unit_bits;
  for (int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; idx < p.units; idx += static_cast<int64_t>(gridDim.x) * kThreads) {
    const Place at = place_of(idx, p.rows, p.h, p.unit_bits);
    const int64_t to = ((idx >> p.unit_bits) * 2 << p.unit_bits) + at.unit;  // map 1; map 2 is `units` further
    const uint4 zero = make_uint4(0, 0, 0, 0), q = *p.q.at(at.batch, at.row, at.head, at.unit);
    const bool first = 2 * at.unit < units;
    uint4* q_maps = reinterpret_cast<uint4*>(p.q_maps);
    q_maps[to] = first ? q : zero;
    q_maps[to + units] = first ? zero : q;
    if (p.dout.base == nullptr) continue;
    const float lam = weight_of(p.weights, at.head);
    const uint4 o = *p.o.at(at.batch, at.row, at.head, at.unit), o2 = *p.o2.at(at.batch, at.row, at.head, at.unit);
    const uint4 d = *p.dout.at(at.batch, at.row, at.head, at.unit);
    uint4 *o_maps = reinterpret_cast<uint4*>(p.o_maps), *do_maps = reinterpret_cast<uint4*>(p.do_maps);
    o_maps[to] = scaled(o2, lam, &o);
    o_maps[to + units] = o2;
    do_maps[to] = d;
    do_maps[to + units] = scaled(d, -lam, nullptr);
  }
}

// O and, where asked for, A_2 V from the outputs of the two maps (o2.base may be null)
struct JoinParams {
  const __half* o_maps;
  View o, o2;
  FaDiffWeights weights;
  int64_t units;
  int rows, h, unit_bits;
};
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ JoinParams p) {
  const int units = 1 << p.unit_bits;
  for (int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; idx < p.units; idx += static_cast<int64_t>(gridDim.x) * kThreads) {
    const Place at = place_of(idx, p.rows, p.h, p.unit_bits);
    const int64_t from = ((idx >> p.unit_bits) * 2 << p.unit_bits) + at.unit;
    const uint4 o1 = reinterpret_cast<const uint4*>(p.o_maps)[from], o2 = reinterpret_cast<const uint4*>(p.o_maps)[from + units];
    *p.o.at(at.batch, at.row, at.head, at.unit) = scaled(o2, -weight_of(p.weights, at.head), &o1);
    if (p.o2.base != nullptr) *p.o2.at(at.batch, at.row, at.head, at.unit) = o2;
  }
}

View view(const void* base, int64_t batch_stride, int64_t row_stride, int64_t head_stride) {
  return View{static_cast<__half*>(const_cast<void*>(base)), batch_stride, row_stride, head_stride};
}

int blocks_for(int64_t units) { return static_cast<int>(std::min<int64_t>((units + kThreads - 1) / kThreads, 148 * 16)); }

bool whole_units(std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  return true;
}

struct Rows {
  int64_t batches, rows;
  int64_t units(int h, int d) const { return batches * rows * h * (d / 8); }
  size_t map_bytes(int h, int d) const { return align256(static_cast<size_t>(units(h, d)) * 2 * 16); }
};
template <class P>
Rows rows_of(const P& p) {
  return p.cu_seqlens_q ? Rows{1, p.total_q} : Rows{p.b, p.seqlen_q};
}

template <class P>
bool plausible(const P& p) {
  return (p.d == 64 || p.d == 128) && p.b >= 1 && p.h >= 1 && p.h_k >= 1 && p.h % p.h_k == 0 && p.seqlen_q >= 1 && p.h < (1 << 29);
}

int split(const SplitParams& sp, cudaStream_t stream) {
  split_kernel<<<blocks_for(sp.units), kThreads, 0, stream>>>(sp);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}
int join(const JoinParams& jp, cudaStream_t stream) {
  join_kernel<<<blocks_for(jp.units), kThreads, 0, stream>>>(jp);
  FA_CHECK_CUDA(cudaGetLastError());
  return FA_OK;
}

}  // namespace
}  // namespace fa

extern "C" int fa_diff_fwd(const FaDiffFwdParams* p, fa_stream_t stream) {
  using namespace fa;
  FA_CHECK_ARG(p != nullptr, "fa_diff_fwd: params is NULL");
  const FaFwdParams& b = p->base;
  FA_CHECK_ARG(b.q && b.k && b.v && b.o && b.lse, "fa_diff_fwd: q, k, v, o, lse must be non-NULL");
  if (b.d != 64 && b.d != 128) return set_error(FA_ERR_UNSUPPORTED, "fa_diff_fwd: head_dim must be 64 or 128");
  FA_CHECK_ARG(plausible(b), "fa_diff_fwd: bad b / h / h_k / seqlen_q");
  int rc = check_weights(p->weights, b.h, "fa_diff_fwd");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(aligned16(p->o2) && whole_units({p->o2_batch_stride, p->o2_row_stride, p->o2_head_stride}),
               "fa_diff_fwd: o2 must be 16-byte aligned with strides that are multiples of 8 elements");
  return run_fwd(&b, 0, static_cast<cudaStream_t>(stream), false, false, p);
}

extern "C" size_t fa_diff_kvcache_workspace_bytes(const FaDiffKvcacheParams* p) {
  using namespace fa;
  if (p == nullptr || !plausible(p->base)) return 0;
  FaKvcacheParams f = p->base;
  f.h *= 2;
  return 2 * Rows{f.b, f.seqlen_q}.map_bytes(p->base.h, f.d) + fa_kvcache_workspace_bytes(&f);
}

extern "C" int fa_diff_kvcache(const FaDiffKvcacheParams* p, int32_t* verdict, int32_t token, fa_stream_t stream_) {
  using namespace fa;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  FA_CHECK_ARG(p != nullptr, "fa_diff_kvcache: params is NULL");
  const FaKvcacheParams& b = p->base;
  FA_CHECK_ARG(b.q && b.o && b.lse, "fa_diff_kvcache: q, o, lse must be non-NULL");
  if (b.d != 64 && b.d != 128) return set_error(FA_ERR_UNSUPPORTED, "fa_diff_kvcache: head_dim must be 64 or 128");
  FA_CHECK_ARG(plausible(b), "fa_diff_kvcache: bad b / h / h_k / seqlen_q");
  int rc = check_weights(p->weights, b.h, "fa_diff_kvcache");
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(aligned16(b.q) && aligned16(b.o) &&
                   whole_units({b.q_batch_stride, b.q_row_stride, b.q_head_stride, b.o_batch_stride, b.o_row_stride, b.o_head_stride}),
               "fa_diff_kvcache: q and o must be 16-byte aligned with strides that are multiples of 8 elements");
  const size_t need = fa_diff_kvcache_workspace_bytes(p);
  if (p->base.workspace == nullptr || b.workspace_bytes < need)
    return set_error(FA_ERR_WORKSPACE, "fa_diff_kvcache: workspace smaller than fa_diff_kvcache_workspace_bytes()");
  FA_CHECK_ARG((reinterpret_cast<uintptr_t>(b.workspace) & 255) == 0, "fa_diff_kvcache: workspace must be 256-byte aligned");
  rc = check_device_sm100();
  if (rc != FA_OK) return rc;
  const Rows r{b.b, b.seqlen_q};
  const size_t map_bytes = r.map_bytes(b.h, b.d);
  const int unit_bits = b.d == 128 ? 4 : 3;
  uint8_t* ws = static_cast<uint8_t*>(b.workspace);
  SplitParams sp = {};
  sp.q = view(b.q, b.q_batch_stride, b.q_row_stride, b.q_head_stride);
  sp.q_maps = reinterpret_cast<__half*>(ws);
  __half* o_maps = reinterpret_cast<__half*>(ws + map_bytes);
  sp.units = r.units(b.h, b.d);
  sp.rows = b.seqlen_q, sp.h = b.h, sp.unit_bits = unit_bits;
  rc = split(sp, stream);
  if (rc != FA_OK) return rc;
  FaKvcacheParams f = b;
  f.q = sp.q_maps, f.o = o_maps, f.h = 2 * b.h;
  f.q_head_stride = f.o_head_stride = b.d;
  f.q_row_stride = f.o_row_stride = static_cast<int64_t>(2) * b.h * b.d;
  f.q_batch_stride = f.o_batch_stride = f.q_row_stride * b.seqlen_q;
  f.workspace = need > 2 * map_bytes ? ws + 2 * map_bytes : nullptr;
  f.workspace_bytes = need - 2 * map_bytes;
  rc = verdict != nullptr ? fa_kvcache_checked(&f, verdict, token, stream) : fa_kvcache(&f, stream);
  if (rc != FA_OK) return rc;
  return join(JoinParams{o_maps, view(b.o, b.o_batch_stride, b.o_row_stride, b.o_head_stride), View{nullptr, 0, 0, 0}, p->weights, sp.units,
                         b.seqlen_q, b.h, unit_bits},
              stream);
}
