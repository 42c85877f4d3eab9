// C ABI of the pages of a KV cache (see include/fa4_nvfp4.h): argument validation and launches.  Host code only; the kernels live in
// kv_pages.cuh.
#include "kv_pages.cuh"
#include "launch.cuh"

#include <algorithm>

using namespace fa4;
using namespace fa4::pages;

namespace {

int validate_pages(const fa4_kv_pages* k) {
  if (k == nullptr) return -FA4_E_NULL;
  if (k->struct_size != sizeof(fa4_kv_pages)) return -FA4_E_STRUCT;
  if (!k->table || !k->refs) return -FA4_E_NULL;
  if (k->B <= 0 || k->pages_per_seq <= 0 || k->num_pages <= 0 || k->page_size <= 0) return -FA4_E_SHAPE;
  // positions are 32-bit, a bit of a page number is a mark
  if ((int64_t)k->pages_per_seq * k->page_size > 0x7ffffc00ll || k->num_pages > 0x3fffffff) return -FA4_E_TOO_LARGE;
  return 0;
}
Book book_of(const fa4_kv_pages* k) {
  Book b = {};
  b.table = k->table;
  b.refs = k->refs;
  b.B = k->B; b.width = k->pages_per_seq; b.num_pages = k->num_pages; b.page_size = k->page_size;
  b.div_page = make_fastdiv((uint32_t)k->page_size);
  b.status = k->status;
  b.epoch = next_launch_epoch();
  // A few hundred numbers are one CTA's.  us, one / eight: 4 rows of 15 pages, pool of 92 6.1 / 7.4, 128 of 18, 1315 14.2 / 8.8, 256 of 66, 11761 28 / 9.9.
  b.ctas = (int64_t)k->B * k->pages_per_seq + k->num_pages <= 1024 ? 1 : kCluster;
  return b;
}
int check_work(const void* work, uint64_t bytes, int64_t words) {
  if (work == nullptr) return -FA4_E_NULL;
  if (!aligned16(work)) return -FA4_E_ALIGN;
  return bytes < (uint64_t)words * 4 ? -FA4_E_TOO_LARGE : 0;
}

}  // namespace

extern "C" int64_t fa4_kv_pages_resize_workspace_bytes(const fa4_kv_pages* k) {
  if (int e = validate_pages(k)) return e;
  if (k->B > kRows) return -FA4_E_TOO_LARGE;
  return resize_words(k->B, k->num_pages) * 4;
}
extern "C" int fa4_kv_pages_resize_ex(const fa4_kv_pages* k, const int32_t* held, const int32_t* wanted, int32_t* pairs, int32_t* granted, void* workspace,
                                      uint64_t workspace_bytes, void* cuda_stream) {
  const int64_t need = fa4_kv_pages_resize_workspace_bytes(k);
  if (need < 0) return (int)need;
  if (!held || !wanted || !pairs) return -FA4_E_NULL;
  if (int e = check_work(workspace, workspace_bytes, need / 4)) return e;
  ResizeParams p = {book_of(k), held, wanted, pairs, granted, static_cast<int32_t*>(workspace)};
  return launch_pdl_cluster((unsigned)p.book.ctas, resize_kernel, dim3((unsigned)p.book.ctas), kThreads, 0, static_cast<cudaStream_t>(cuda_stream), p);
}
extern "C" int fa4_kv_pages_resize(const fa4_kv_pages* k, const int32_t* held, const int32_t* wanted, int32_t* pairs, void* workspace,
                                   uint64_t workspace_bytes, void* cuda_stream) {
  return fa4_kv_pages_resize_ex(k, held, wanted, pairs, nullptr, workspace, workspace_bytes, cuda_stream);
}

extern "C" int fa4_kv_pages_fork(const fa4_kv_pages* k, const int32_t* held, const int32_t* parents, int32_t rows, int32_t* new_table,
                                 int32_t* new_held, void* cuda_stream) {
  if (int e = validate_pages(k)) return e;
  if (!held || !parents || !new_table || !new_held) return -FA4_E_NULL;
  if (rows <= 0) return -FA4_E_SHAPE;
  if ((int64_t)rows + k->B > 0x7fffffffll || (int64_t)rows * k->B > 0x3fffffffll) return -FA4_E_TOO_LARGE;
  ForkParams p = {book_of(k), held, parents, new_table, new_held, rows};
  return launch_pdl(fork_kernel, dim3((unsigned)(rows + k->B)), kForkThreads, 0, static_cast<cudaStream_t>(cuda_stream), p);
}

extern "C" int64_t fa4_kv_pages_compact_workspace_bytes(const fa4_kv_pages* k) {
  if (int e = validate_pages(k)) return e;
  return compact_words(k->num_pages) * 4;
}
extern "C" int fa4_kv_pages_compact(const fa4_kv_pages* k, int32_t* pairs, int32_t* used, void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
  const int64_t need = fa4_kv_pages_compact_workspace_bytes(k);
  if (need < 0) return (int)need;
  if ((!pairs && k->num_pages > 1) || !used) return -FA4_E_NULL;
  if (int e = check_work(workspace, workspace_bytes, need / 4)) return e;
  CompactParams p = {book_of(k), pairs, used, static_cast<int32_t*>(workspace)};
  return launch_pdl_cluster((unsigned)p.book.ctas, compact_kernel, dim3((unsigned)p.book.ctas), kThreads, 0, static_cast<cudaStream_t>(cuda_stream), p);
}

extern "C" int fa4_kv_pages_copy(const fa4_kv_copy* c, void* cuda_stream) {
  if (c == nullptr) return -FA4_E_NULL;
  if (c->struct_size != sizeof(fa4_kv_copy)) return -FA4_E_STRUCT;
  if (!c->pairs) return -FA4_E_NULL;
  if (c->num_pairs <= 0 || c->num_pages <= 0 || c->num_tensors <= 0 || c->num_tensors > kTensors) return -FA4_E_SHAPE;
  PagedTensor all[kTensors];
  int64_t flat_bytes = 0;                     // of a page, in tensors whose pages lie in one piece
  auto flat = [](const PagedTensor& t) { return t.log_piece == 4 && t.row == t.pieces; };
  for (int i = 0; i < c->num_tensors; ++i) {
    const fa4_kv_paged& s = c->tensors[i];
    if (!s.base) return -FA4_E_NULL;
    if (s.row_bytes <= 0 || s.rows_inner <= 0 || s.rows_outer <= 0) return -FA4_E_SHAPE;
    // strides of what there is one of are never used
    const int64_t inner = s.rows_inner > 1 ? s.stride_inner : 0, outer = s.rows_outer > 1 ? s.stride_outer : 0, page = c->num_pages > 1 ? s.stride_page : 0;
    if (inner < 0 || outer < 0 || page < 0) return -FA4_E_STRIDE;
    const uint64_t bits = (uint64_t)(uintptr_t)s.base | (uint64_t)s.row_bytes | (uint64_t)inner | (uint64_t)outer | (uint64_t)page;
    const int log_piece = (bits & 15u) == 0 ? 4 : (bits & 3u) == 0 ? 2 : 0;
    if (s.row_bytes > 0x7fffffffll || s.rows_inner > 0x7fffffffll || s.rows_outer > 0x7fffffffll) return -FA4_E_TOO_LARGE;
    const int64_t rows = s.rows_inner * s.rows_outer, row = s.row_bytes >> log_piece;
    if (rows > 0x3fffffffll || rows * row > 0x3fffffffll) return -FA4_E_TOO_LARGE;
    PagedTensor& t = all[i];
    t.base = static_cast<uint8_t*>(s.base);
    t.page = page; t.inner = inner; t.outer = outer;
    t.pieces = (int)(rows * row);
    t.log_piece = log_piece;
    t.row = (int)row;
    t.rows_inner = (int)s.rows_inner;
    t.div_row = make_fastdiv((uint32_t)row);
    t.div_inner = make_fastdiv((uint32_t)s.rows_inner);
    if (flat(t)) flat_bytes += (int64_t)t.pieces * 16;
  }
  // From 64 MB on (the pairs that are none among them, which only the device can tell) by bulk copies, the rest of the tensors by a launch of its own.
  const bool bulk = flat_bytes * c->num_pairs >= (64ll << 20);
  CopyParams parts[2] = {};
  for (const bool by_bulk : {true, false}) {
    CopyParams& p = parts[by_bulk ? 0 : 1];
    p.pairs = c->pairs;
    p.n = c->num_pairs; p.num_pages = c->num_pages;
    int64_t tasks = 0;
    for (int i = 0; i < c->num_tensors; ++i) {
      if ((bulk && flat(all[i])) != by_bulk) continue;
      const int64_t per = by_bulk ? kBulkBytes / 16 : kCopyThreads * kCopyPieces;
      p.first[p.tensors] = (int)tasks;
      p.t[p.tensors++] = all[i];
      tasks += (all[i].pieces + per - 1) / per;
    }
    p.first[p.tensors] = (int)tasks;
    p.div_tasks = make_fastdiv((uint32_t)tasks);
    p.tasks = tasks * c->num_pairs;
    if (p.tasks > 0x3fffffffll) return -FA4_E_TOO_LARGE;
    p.status = c->status;
    p.epoch = next_launch_epoch();
    p.budget_ns = kDefaultBudgetNs;
  }
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (parts[0].tensors > 0) {
    const unsigned grid = (unsigned)std::min<int64_t>(parts[0].tasks, kSms * kBulkCtas);
    if (int e = launch_pdl(copy_bulk_kernel, dim3(grid), 32, kBulkRequest, stream, parts[0])) return e;
  }
  if (parts[1].tensors == 0) return 0;
  const unsigned grid = (unsigned)std::min<int64_t>(parts[1].tasks, kSms * 8);
  return launch_pdl(copy_kernel, dim3(grid), kCopyThreads, 0, stream, parts[1]);
}
