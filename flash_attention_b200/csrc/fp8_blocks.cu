// C ABI of the choice of blocks in the 8-bit KV cache (see include/fa4_nvfp4.h): argument validation and launches of the index and of the
// choice.  Host code only; the kernels live in fp8_blocks.cuh, the attention over what is chosen in fp8_cache.cu.
#include "fp8_blocks.cuh"
#include "fp8_host.cuh"

#include <algorithm>

using namespace fa4;

namespace {

int validate_index(const fa4_fp8_cache* c, const fa4_fp8_index* x) {
  if (int e = validate_cache(c)) return e;
  if (x == nullptr) return -FA4_E_NULL;
  if (x->struct_size != sizeof(fa4_fp8_index)) return -FA4_E_STRUCT;
  if (!x->bounds || !x->scale) return -FA4_E_NULL;
  if (!aligned16(x->bounds)) return -FA4_E_ALIGN;
  return 0;
}

}  // namespace

extern "C" int fa4_fp8_cache_index(const fa4_fp8_cache* c, const fa4_fp8_index* x, const fa4_fp8_index_call* a, void* cuda_stream) {
  if (int e = validate_index(c, x)) return e;
  if (a == nullptr) return -FA4_E_NULL;
  if (a->struct_size != sizeof(fa4_fp8_index_call)) return -FA4_E_STRUCT;
  if (!a->seqlens) return -FA4_E_NULL;
  if (a->B <= 0 || a->S <= 0 || (c->page_table == nullptr && a->B > c->num_pages)) return -FA4_E_SHAPE;
  const int64_t capacity = (int64_t)c->pages_per_seq * c->page_size;
  // (a call for more tokens than fit: one block too many, which reports it)
  const int64_t blocks = std::min<int64_t>(((int64_t)a->S + c->block - 2) / c->block + 1, capacity / c->block + 1), units = blocks * a->B * c->Hkv;
  if (units > 0x3fffffffll) return -FA4_E_TOO_LARGE;
  IndexParams p = {};
  p.k = static_cast<const uint8_t*>(c->k);
  p.k_page = c->k_stride_page; p.k_tok = c->k_stride_token; p.k_head = c->k_stride_head;
  p.k_scale = c->k_scale;
  p.bounds = static_cast<int8_t*>(x->bounds);
  p.scale = x->scale;
  p.seqlens = a->seqlens;
  p.fresh = a->seqused_new;
  p.table = c->page_table;
  p.S = a->S; p.Hkv = c->Hkv;
  p.log_block = log2_of(c->block);
  p.num_pages = c->num_pages; p.page_size = c->page_size; p.pages_per_seq = c->pages_per_seq;
  p.blocks = (int)blocks;
  p.units = (int)units;
  p.div_hkv = make_fastdiv((uint32_t)c->Hkv);
  p.div_blocks = make_fastdiv((uint32_t)blocks);
  p.div_page = make_fastdiv((uint32_t)c->page_size);
  p.status = a->status;
  p.epoch = next_launch_epoch();
  const dim3 grid((unsigned)((units + kIndexWarps - 1) / kIndexWarps));
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  return c->D == 128 ? launch_pdl(fp8_index_kernel<128>, grid, kIndexWarps * 32, 0, stream, p)
                     : launch_pdl(fp8_index_kernel<64>, grid, kIndexWarps * 32, 0, stream, p);
}

extern "C" int fa4_fp8_cache_select(const fa4_fp8_cache* c, const fa4_fp8_index* x, const fa4_fp8_select* a, void* cuda_stream) {
  if (int e = validate_index(c, x)) return e;
  if (a == nullptr) return -FA4_E_NULL;
  if (a->struct_size != sizeof(fa4_fp8_select)) return -FA4_E_STRUCT;
  if (!a->q || !a->seqused_k || !a->blocks) return -FA4_E_NULL;
  if (a->B <= 0 || a->Sq <= 0 || a->Hq <= 0 || a->Hq % c->Hkv != 0) return -FA4_E_SHAPE;
  if (c->page_table == nullptr && a->B > c->num_pages) return -FA4_E_SHAPE;
  if (a->num_blocks <= 0 || a->query_block <= 0 || a->front_blocks < 0 || a->recent_blocks < 1) return -FA4_E_SHAPE;
  const int64_t rows = std::min(a->query_block, a->Sq), group = a->Hq / c->Hkv;
  // what is chosen always has to fit: the front, and from the first row's block back and up to the last one's
  const int64_t always = (int64_t)a->front_blocks + a->recent_blocks + (rows + c->block - 2) / c->block;
  if (always > a->num_blocks) return -FA4_E_SHAPE;
  const int64_t strides[] = {a->q_stride_b, a->q_stride_s, a->q_stride_h};
  for (int64_t s : strides)
    if ((s & 7) != 0) return -FA4_E_STRIDE;
  if (!aligned16(a->q)) return -FA4_E_ALIGN;
  const int64_t query_blocks = ((int64_t)a->Sq + a->query_block - 1) / a->query_block, units = query_blocks * a->B * c->Hkv,
                blocks = (int64_t)c->pages_per_seq * c->page_size / c->block;
  // (sums of a query block are 32-bit; a unit's scores stay in shared memory)
  if (units > 0x0fffffffll || rows * group > 32768 || blocks > kSelectBlocks || (int64_t)c->num_pages * (c->page_size / c->block) > 0x7fffffffll) return -FA4_E_TOO_LARGE;
  SelectParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_b = a->q_stride_b; p.q_s = a->q_stride_s; p.q_h = a->q_stride_h;
  p.bounds = static_cast<const int8_t*>(x->bounds);
  p.scale = x->scale;
  p.used = a->seqused_k;
  p.fresh = a->seqused_q;
  p.table = c->page_table;
  p.blocks = a->blocks;
  p.Sq = a->Sq; p.Hkv = c->Hkv; p.group = (int)group;
  p.log_block = log2_of(c->block);
  p.num_pages = c->num_pages; p.page_size = c->page_size; p.pages_per_seq = c->pages_per_seq;
  p.capacity = c->pages_per_seq * c->page_size;
  p.chosen = a->num_blocks; p.query_block = (int)rows; p.query_blocks = (int)query_blocks;
  p.front = a->front_blocks; p.recent = a->recent_blocks;
  p.div_hkv = make_fastdiv((uint32_t)c->Hkv);
  p.div_query_blocks = make_fastdiv((uint32_t)query_blocks);
  p.div_page = make_fastdiv((uint32_t)c->page_size);
  p.div_group = make_fastdiv((uint32_t)group);
  p.status = a->status;
  p.epoch = next_launch_epoch();
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const uint32_t smem = (uint32_t)blocks * 4;
  // Few units of many blocks: several CTAs a unit.
  p.parts = 1;
  while (p.parts < 8 && units * p.parts * 2 <= kSms && blocks / (p.parts * 2) >= 256) p.parts *= 2;
  auto launch = [&](auto kernel) -> int {
    if (int e = ensure_smem(kernel, kSelectBlocks * 4)) return e;
    return launch_pdl_cluster((unsigned)p.parts, kernel, dim3((unsigned)(units * p.parts)), kSelectThreads, smem, stream, p);
  };
  if (p.parts > 1) return c->D == 128 ? launch(fp8_select_kernel<128, true>) : launch(fp8_select_kernel<64, true>);
  return c->D == 128 ? launch(fp8_select_kernel<128, false>) : launch(fp8_select_kernel<64, false>);
}
