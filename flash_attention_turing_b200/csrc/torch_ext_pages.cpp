// PyTorch binding of the page functions (fa_pages_*): tensors are checked here, outputs and scratch memory come from torch's
// allocator, and the call goes to the current stream of the tables' device.
#include "torch_common.h"

#include <vector>

namespace {

void check_int32(const at::Tensor& t, const at::Device& device, int64_t dim, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == device, name, " must be a CUDA tensor on the device of the others");
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be a torch.int32 tensor");
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, dim == 1 ? " dimension" : " dimensions");
}

// cache_seqlens may be undefined where the lengths are not looked at
FaPageTables tables(const at::Tensor& block_table, const at::Tensor& cache_seqlens, const at::Tensor& page_refs) {
  TORCH_CHECK(block_table.is_cuda(), "block_table must be a CUDA tensor");
  const at::Device device = block_table.device();
  check_int32(block_table, device, 2, "block_table");
  if (cache_seqlens.defined()) {
    check_int32(cache_seqlens, device, 1, "cache_seqlens");
    TORCH_CHECK(cache_seqlens.size(0) == block_table.size(0), "cache_seqlens must have shape [batch_size]");
    TORCH_CHECK(cache_seqlens.is_contiguous(), "cache_seqlens must be contiguous");
  }
  check_int32(page_refs, device, 1, "page_refs");
  TORCH_CHECK(block_table.stride(1) == 1 || block_table.size(1) <= 1, "block_table must have contiguous last dimension");
  TORCH_CHECK(page_refs.is_contiguous(), "page_refs must be contiguous");
  TORCH_CHECK(block_table.numel() < INT32_MAX && page_refs.numel() < INT32_MAX, "too many pages");
  TORCH_CHECK(block_table.size(0) <= 1 || block_table.stride(0) >= block_table.size(1), "block_table must not overlap itself");
  FaPageTables t = {};
  t.block_table = block_table.data_ptr<int>();
  t.cache_seqlens = cache_seqlens.defined() ? cache_seqlens.data_ptr<int>() : nullptr;
  t.page_refs = page_refs.data_ptr<int>();
  t.rows = block_table.size(0), t.columns = block_table.size(1), t.num_pages = page_refs.size(0);
  t.row_stride = t.rows <= 1 ? t.columns : block_table.stride(0);
  return t;
}

struct Caches {
  std::vector<void*> base;
  std::vector<int64_t> page_stride;
  FaPageCaches c = {};
  int64_t pages = 0, page_size = 0;
  at::Device device = at::kCUDA;

  explicit Caches(const std::vector<at::Tensor>& caches) {
    TORCH_CHECK(!caches.empty(), "caches must hold at least one tensor");
    const at::Tensor& first = caches[0];
    TORCH_CHECK(first.is_cuda() && first.dim() >= 2, "caches must be CUDA tensors of shape [num_pages, page_size, ...]");
    device = first.device();
    pages = first.size(0), page_size = first.size(1);
    TORCH_CHECK(pages < INT32_MAX && page_size < INT32_MAX, "too many pages");
    base.reserve(caches.size()), page_stride.reserve(caches.size());
    int64_t elements = 1;
    for (int64_t i = 1; i < first.dim(); ++i) elements *= first.size(i);
    c.page_bytes = elements * first.element_size();
    TORCH_CHECK(c.page_bytes % 16 == 0, "the bytes of a page must be a multiple of 16");
    for (const at::Tensor& t : caches) {
      TORCH_CHECK(t.device() == device && t.dim() == first.dim() && t.size(0) == pages && t.size(1) == page_size &&
                      t.numel() == first.numel() && t.element_size() == first.element_size(),
                  "caches must have the same device, shape and element size");
      if (!t.is_contiguous()) {
        int64_t stride = 1;
        for (int64_t i = t.dim() - 1; i >= 1; --i) {
          TORCH_CHECK(t.size(i) == 1 || t.stride(i) == stride, "a page must be contiguous in every cache");
          stride *= t.size(i);
        }
        TORCH_CHECK(pages <= 1 || t.stride(0) >= elements, "pages of a cache must not overlap");
      }
      const int64_t bytes = pages <= 1 ? c.page_bytes : t.stride(0) * t.element_size();
      TORCH_CHECK(bytes % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "pages must be aligned to 16 bytes");
      base.push_back(t.data_ptr());
      page_stride.push_back(bytes);
    }
    c.base = base.data(), c.page_stride = page_stride.data();
    c.count = static_cast<int32_t>(base.size());
  }
  bool empty() const { return pages == 0 || c.page_bytes == 0; }
};

struct Scratch {  // none where no bytes are wanted
  at::Tensor memory;
  void* data = nullptr;
  size_t bytes;
  Scratch(size_t wanted, const at::Tensor& like) : bytes(wanted) {
    if (wanted > 0) memory = scratch(wanted, like), data = memory.data_ptr();
  }
};

at::Tensor flags(int64_t n, const at::Tensor& like) { return torch::empty({n}, like.options().dtype(at::kBool)); }
uint8_t* flag_ptr(const at::Tensor& t) { return reinterpret_cast<uint8_t*>(t.data_ptr<bool>()); }

at::Tensor pages_reserve(at::Tensor block_table, at::Tensor cache_seqlens, at::Tensor page_refs, c10::optional<at::Tensor> new_tokens,
                         int64_t new_tokens_all, int64_t page_size) {
  const FaPageTables t = tables(block_table, cache_seqlens, page_refs);
  TORCH_CHECK(page_size >= 1 && page_size < INT32_MAX, "page_size must be positive");
  TORCH_CHECK(new_tokens_all >= 0 && new_tokens_all < INT32_MAX, "new_tokens must be non-negative");
  const int* tokens = nullptr;
  if (new_tokens.has_value()) {
    check_int32(*new_tokens, block_table.device(), 1, "new_tokens");
    TORCH_CHECK(new_tokens->size(0) == t.rows && new_tokens->is_contiguous(), "new_tokens must have shape [batch_size] and be contiguous");
    tokens = new_tokens->data_ptr<int>();
  }
  c10::cuda::CUDAGuard guard(block_table.device());
  at::Tensor granted = flags(t.rows, block_table);
  if (t.rows == 0) return granted;
  TORCH_CHECK(t.columns >= 1 && t.num_pages >= 1, "block_table and page_refs must not be empty");
  const Scratch ws(fa_pages_reserve_workspace_bytes(&t), block_table);
  check_rc(fa_pages_reserve(&t, tokens, static_cast<int32_t>(new_tokens_all), static_cast<int32_t>(page_size), flag_ptr(granted),
                            ws.data, ws.bytes, current_stream()),
           "fa_pages_reserve");
  return granted;
}

void check_list(const at::Tensor& t, const at::Device& device, const char* name) {
  check_int32(t, device, 1, name);
  TORCH_CHECK(t.is_contiguous() && t.numel() < INT32_MAX, name, " must be contiguous");
}

at::Tensor pages_fork(std::vector<at::Tensor> caches, at::Tensor block_table, at::Tensor cache_seqlens, at::Tensor page_refs,
                      at::Tensor parents, at::Tensor children) {
  const Caches c(caches);
  const FaPageTables t = tables(block_table, cache_seqlens, page_refs);
  TORCH_CHECK(c.device == block_table.device() && c.pages == t.num_pages, "caches and page_refs must have the same device and number of pages");
  check_list(parents, c.device, "parents");
  check_list(children, c.device, "children");
  TORCH_CHECK(parents.numel() == children.numel(), "parents and children must have the same length");
  c10::cuda::CUDAGuard guard(c.device);
  at::Tensor granted = flags(parents.numel(), parents);
  if (parents.numel() == 0) return granted;
  if (t.rows == 0 || t.columns == 0 || c.empty()) return granted.zero_();
  const int32_t n = static_cast<int32_t>(parents.numel());
  const Scratch ws(fa_pages_fork_workspace_bytes(&t, &c.c, n), block_table);
  check_rc(fa_pages_fork(&t, &c.c, parents.data_ptr<int>(), children.data_ptr<int>(), n, static_cast<int32_t>(c.page_size),
                         flag_ptr(granted), ws.data, ws.bytes, current_stream()),
           "fa_pages_fork");
  return granted;
}

void pages_free(at::Tensor block_table, at::Tensor cache_seqlens, at::Tensor page_refs, at::Tensor rows) {
  const FaPageTables t = tables(block_table, cache_seqlens, page_refs);
  check_list(rows, block_table.device(), "rows");
  if (rows.numel() == 0 || t.rows == 0 || t.columns == 0 || t.num_pages == 0) return;
  c10::cuda::CUDAGuard guard(block_table.device());
  check_rc(fa_pages_free(&t, rows.data_ptr<int>(), static_cast<int32_t>(rows.numel()), current_stream()), "fa_pages_free");
}

at::Tensor pages_compact(std::vector<at::Tensor> caches, at::Tensor block_table, at::Tensor page_refs) {
  const Caches c(caches);
  const FaPageTables t = tables(block_table, at::Tensor(), page_refs);
  TORCH_CHECK(c.device == block_table.device() && c.pages == t.num_pages, "caches and page_refs must have the same device and number of pages");
  c10::cuda::CUDAGuard guard(c.device);
  at::Tensor live = torch::empty({1}, page_refs.options());
  if (t.rows == 0 || t.columns == 0 || c.empty()) return live.zero_();
  const Scratch ws(fa_pages_workspace_bytes(t.rows, t.num_pages, 0), block_table);
  check_rc(fa_pages_compact(&t, &c.c, live.data_ptr<int>(), ws.data, ws.bytes, current_stream()), "fa_pages_compact");
  return live;
}

at::Tensor pages_copy(std::vector<at::Tensor> caches, at::Tensor src, at::Tensor dst) {
  const Caches c(caches);
  check_list(src, c.device, "src");
  check_list(dst, c.device, "dst");
  TORCH_CHECK(src.numel() == dst.numel(), "src and dst must have the same length");
  c10::cuda::CUDAGuard guard(c.device);
  at::Tensor done = flags(src.numel(), src);
  if (src.numel() == 0) return done;
  if (c.empty()) return done.zero_();
  const int32_t n = static_cast<int32_t>(src.numel());
  const Scratch ws(fa_pages_copy_workspace_bytes(&c.c, static_cast<int32_t>(c.pages), n), src);
  check_rc(fa_pages_copy(&c.c, static_cast<int32_t>(c.pages), src.data_ptr<int>(), dst.data_ptr<int>(), n, flag_ptr(done),
                         ws.data, ws.bytes, current_stream()),
           "fa_pages_copy");
  return done;
}

}  // namespace

void bind_pages(py::module_& m) {
  m.def("pages_reserve", &pages_reserve, "Pages for the next tokens of every row; which rows have them");
  m.def("pages_fork", &pages_fork, "Rows that share the pages of others; which entries were done");
  m.def("pages_free", &pages_free, "Rows give their pages back");
  m.def("pages_compact", &pages_compact, "Pages in use come first; how many they are");
  m.def("pages_copy", &pages_copy, "Copies pages in every cache; which entries were done");
}
