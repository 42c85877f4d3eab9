// C ABI of the 8-bit KV cache (see include/fa4_nvfp4.h): argument validation and launches of the append and
// of the attention over it.  Host code only; the kernels live in the .cuh files.
#include "fp8_prefill.cuh"
#include "launch.cuh"

#include <algorithm>
#include <cmath>
#include <numeric>
#include <type_traits>

namespace {

using namespace fa4;

// Shape, strides and alignment of a cache.  Touches no CUDA API.
int validate_cache(const fa4_fp8_cache* c) {
  if (c == nullptr) return -FA4_E_NULL;
  if (c->struct_size != sizeof(fa4_fp8_cache)) return -FA4_E_STRUCT;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return -FA4_E_NULL;
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return -FA4_E_SHAPE;
  if (c->num_pages <= 0 || c->page_size <= 0 || c->page_size % c->block != 0 || c->Hkv <= 0) return -FA4_E_SHAPE;
  if (c->D != 64 && c->D != 128) return -FA4_E_SHAPE;
  if (c->pages_per_seq <= 0 || (c->page_table == nullptr && c->pages_per_seq != 1)) return -FA4_E_SHAPE;
  // positions are 32-bit
  if ((int64_t)c->pages_per_seq * c->page_size > 0x7ffffc00ll) return -FA4_E_TOO_LARGE;
  const int64_t strides[] = {c->k_stride_page, c->k_stride_token, c->k_stride_head,
                             c->v_stride_page, c->v_stride_token, c->v_stride_head};
  for (int64_t s : strides)
    if (s <= 0 || (s & 15) != 0) return -FA4_E_STRIDE;
  if (!aligned16(c->k) || !aligned16(c->v)) return -FA4_E_ALIGN;
  return 0;
}

int log2_of(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

}  // namespace

extern "C" int fa4_fp8_cache_append(const fa4_fp8_cache* c, const fa4_fp8_append* a, void* cuda_stream) {
  if (int e = validate_cache(c)) return e;
  if (a == nullptr) return -FA4_E_NULL;
  if (a->struct_size != sizeof(fa4_fp8_append)) return -FA4_E_STRUCT;
  if (!a->k || !a->v || !a->seqlens) return -FA4_E_NULL;
  if (a->B <= 0 || a->S <= 0 || (c->page_table == nullptr && a->B > c->num_pages)) return -FA4_E_SHAPE;
  const bool rotate = a->cos != nullptr;
  if ((a->sin != nullptr) != rotate) return -FA4_E_NULL;
  if (rotate && (a->rotary_dim <= 0 || a->rotary_dim % 16 != 0 || a->rotary_dim > c->D || a->rotary_rows <= 0)) return -FA4_E_SHAPE;
  if (rotate && (!aligned16(a->cos) || !aligned16(a->sin))) return -FA4_E_ALIGN;
  const bool with_q = a->q != nullptr;
  if (with_q && (!rotate || a->q_out == nullptr)) return -FA4_E_NULL;
  if (with_q && (a->Hq <= 0 || a->Hq > 0xffff)) return -FA4_E_SHAPE;
  const int64_t strides[] = {a->k_stride_b, a->k_stride_s, a->k_stride_h, a->v_stride_b, a->v_stride_s, a->v_stride_h,
                             with_q ? a->q_stride_b : 0, with_q ? a->q_stride_s : 0, with_q ? a->q_stride_h : 0};
  for (int64_t s : strides)
    if ((s & 7) != 0) return -FA4_E_STRIDE;
  if (!aligned16(a->k) || !aligned16(a->v) || (with_q && (!aligned16(a->q) || !aligned16(a->q_out)))) return -FA4_E_ALIGN;
  const int64_t blocks = ((int64_t)a->S + c->block - 2) / c->block + 1, units = blocks * a->B * c->Hkv * 2;
  if (units > 0x3fffffffll || (int64_t)a->B * a->S * (with_q ? a->Hq : 1) > 0x0fffffffll) return -FA4_E_TOO_LARGE;

  AppendParams p = {};
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.k_b = a->k_stride_b; p.k_s = a->k_stride_s; p.k_h = a->k_stride_h;
  p.v_b = a->v_stride_b; p.v_s = a->v_stride_s; p.v_h = a->v_stride_h;
  p.q_b = a->q_stride_b; p.q_s = a->q_stride_s; p.q_h = a->q_stride_h;
  p.kc = static_cast<uint8_t*>(c->k);
  p.vc = static_cast<uint8_t*>(c->v);
  p.kc_page = c->k_stride_page; p.kc_tok = c->k_stride_token; p.kc_head = c->k_stride_head;
  p.vc_page = c->v_stride_page; p.vc_tok = c->v_stride_token; p.vc_head = c->v_stride_head;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  p.seqlens = a->seqlens;
  p.fresh = a->seqused_new;
  p.table = c->page_table;
  p.cos = a->cos;
  p.sin = a->sin;
  p.rotary_dim = rotate ? a->rotary_dim : 0;
  p.rotary_rows = a->rotary_rows;
  p.rotary_bf16 = a->rotary_bf16;
  p.interleaved = a->interleaved;
  p.B = a->B; p.S = a->S; p.Hq = a->Hq; p.Hkv = c->Hkv; p.D = c->D;
  p.log_block = log2_of(c->block);
  p.num_pages = c->num_pages; p.page_size = c->page_size; p.pages_per_seq = c->pages_per_seq;
  p.blocks = (int)blocks;
  p.div_blocks = make_fastdiv((uint32_t)blocks);
  p.div_hkv2 = make_fastdiv((uint32_t)c->Hkv * 2u);
  p.div_page = make_fastdiv((uint32_t)c->page_size);
  p.div_s = make_fastdiv((uint32_t)a->S);
  p.status = a->status;
  p.epoch = next_launch_epoch();
  // q: four heads of a row to a thread, which share the angles, where one head each would be more threads than the SMs hold at once.  us, one /
  // four, 32 heads: 2 x 8192 tokens 99 / 87, 2 x 2048 25.1 / 23.5; but 64 x 1 2.89 / 2.98, 6 x 777 of 16 heads (D = 64) 7.2 / 7.4.
  const int64_t chunks = c->D / 16, q_items = with_q ? (int64_t)a->B * a->S * a->Hq * chunks : 0;
  p.q_heads = q_items > kSms * 2048 ? 4 : 1;
  p.q_head_groups = with_q ? (a->Hq + p.q_heads - 1) / p.q_heads : 1;
  p.div_groups = make_fastdiv((uint32_t)p.q_head_groups);
  const int64_t q_threads = with_q ? (int64_t)a->B * a->S * p.q_head_groups * chunks : 0;
  p.units = (int)units;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  // pieces of 16 elements that a unit may have
  const int64_t pieces = std::min<int64_t>(a->S, c->block) * chunks;
  auto launch = [&](auto kernel, int threads, int64_t ctas) -> int {
    p.kv_ctas = (int)ctas;
    return launch_pdl(kernel, dim3((unsigned)(ctas + (q_threads + threads - 1) / threads)), (unsigned)threads, 0, stream, p);
  };
  // About four rows a thread: what a unit costs a thread once (its place, the scale) is as much as a row's 16 elements.  us, 2 x 8192 tokens of 8
  // heads without q, blocks of 16 / 32 / 64 tokens: a row a thread (two for 64) 56 / 54 / 43, four 40 / 38 / 38.
  if (pieces <= 32) return launch(fp8_append_kernel<32, false>, 128, (units + 3) / 4);
  if (pieces <= 128) return launch(fp8_append_kernel<32, true>, 128, (units + 3) / 4);
  if (pieces <= 256) return launch(fp8_append_kernel<64, true>, 64, units);
  if (pieces <= 512) return launch(fp8_append_kernel<128, true>, 128, units);
  return launch(fp8_append_kernel<256, true>, 256, units);
}

namespace {

// Factors of the scores: in log2 units softmax_scale * log2 e, or with a soft cap cap * log2 e tanh((q . k) * softmax_scale / cap).
struct ScoreFactors {
  float sl2, cap_in, cap_out;
};
ScoreFactors factors_of(const fa4_fp8_fwd* f) {
  constexpr float kLog2e = 1.4426950408889634f;
  return {f->softmax_scale * kLog2e, f->softcap > 0.f ? f->softmax_scale / f->softcap : 0.f, f->softcap * kLog2e};
}

int validate_fwd(const fa4_fp8_cache* c, const fa4_fp8_fwd* f) {
  if (int e = validate_cache(c)) return e;
  if (f == nullptr) return -FA4_E_NULL;
  if (f->struct_size != sizeof(fa4_fp8_fwd)) return -FA4_E_STRUCT;
  if (!f->q || !f->out || !f->seqused_k) return -FA4_E_NULL;
  if (f->B <= 0 || f->Sq <= 0 || f->Hq <= 0 || f->Hq % c->Hkv != 0) return -FA4_E_SHAPE;
  if (c->page_table == nullptr && f->B > c->num_pages) return -FA4_E_SHAPE;
  if (!(f->softmax_scale > 0.f) || !(f->softcap >= 0.f) || f->num_splits < 0 || f->num_splits > 128) return -FA4_E_SHAPE;
  const ScoreFactors by = factors_of(f);
  if (!std::isfinite(by.sl2) || !std::isfinite(by.cap_out) || (f->softcap > 0.f && !std::isnormal(by.cap_in))) return -FA4_E_SHAPE;
  // (tiles of all sequences and heads are counted in 32 bits)
  if ((int64_t)f->B * c->Hkv * ((int64_t)c->pages_per_seq * c->page_size / 128 + 1) > 0x3fffffffll) return -FA4_E_TOO_LARGE;
  if ((int64_t)f->B * f->Sq * f->Hq > 0x0fffffffll || f->B > 65535) return -FA4_E_TOO_LARGE;
  if ((int64_t)f->B * c->Hkv * std::max(1, f->num_splits) > 0x7fffffffll) return -FA4_E_TOO_LARGE;       // (CTAs)
  const int64_t strides[] = {f->q_stride_b, f->q_stride_s, f->q_stride_h, f->o_stride_b, f->o_stride_s, f->o_stride_h};
  for (int64_t s : strides)
    if ((s & 7) != 0) return -FA4_E_STRIDE;
  if (!aligned16(f->q) || !aligned16(f->out)) return -FA4_E_ALIGN;
  return 0;
}

}  // namespace

namespace {

// The most tiles of 128 keys that `tokens` rows of a sequence one behind the other may see.
int64_t most_tiles(const fa4_fp8_cache* c, const fa4_fp8_fwd* f, int64_t tokens) {
  const int64_t all = ((int64_t)c->pages_per_seq * c->page_size + 127) / 128;
  if (f->window_left < 0) return all;
  const bool open = f->window_right < 0 && !f->causal;         // (to the right)
  return open ? all : std::min(all, ((int64_t)f->window_left + std::max(0, f->window_right) + tokens + 126) / 128 + 1);
}

// How a call is run.
struct Fp8Plan {
  bool decode;
  int rows;          // decode: rows that the kernel is built for
  int bundle;        // decode: kv heads side by side
  int row_tiles, cta_rows;   // many rows: tiles of 128 or 256
  int splits;        // 0: shares dealt on the device
  int64_t slots;     // of partial results, and their rows
  int64_t slot_rows;
};
// Rows of a CTA and splits of the kernel for many rows.  Chosen splits: 256 rows, whatever the batch.  CTAs that are more than the SMs: 256 rows, one
// split.  Else what takes the least time by these figures (us): a CTA 10 with 128 rows and 13 with 256, a step of 128 keys 2.0 and 1.85 (the softmax of one tile
// wait for the products more often), a merge 5 and the partial results, written and read once at 4 TB/s.  Measured, 128 rows / 256 rows / 256 in two
// splits, D = 128: 333 rows of 16 heads on as many keys 13.3 / 16.6 / 21.3, 512 of 32 heads on 1024 keys 21.2 / 25.4 / 31.7, on 4096 keys
// 56.4 / 68.2 / 54.0, three sequences of 333 rows of 16 heads on up to 2048 keys 39.3 / 40.6 / 40.2.
// The steps are those of a table that is full: the lengths are on the device.  In front of a table for 16 times its keys the first call takes 21.2, as if split.
void plan_many(const fa4_fp8_cache* c, const fa4_fp8_fwd* f, Fp8Plan* plan) {
  const int group = f->Hq / c->Hkv, chosen = f->num_splits;
  const int64_t rows = (int64_t)f->Sq * group, units = (int64_t)c->Hkv * f->B, values = (int64_t)f->B * f->Sq * f->Hq * c->D;
  double least = 0;
  for (const int cta_rows : {256, 128}) {
    const int64_t row_tiles = (rows + cta_rows - 1) / cta_rows, room = kSms / (units * row_tiles),
                  tiles = most_tiles(c, f, std::min<int64_t>(f->Sq, (cta_rows - 1) / group + 2));
    if (cta_rows == 128 && (room == 0 || chosen > 0)) break;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>({128, room, tiles / 2}));
    for (int64_t splits = chosen > 0 ? chosen : 1; splits <= (chosen > 0 ? chosen : most); ++splits) {
      const double merge = splits == 1 ? 0. : 5. + (double)(splits * values) * 8 / 4e6;
      const double us = (cta_rows == 256 ? 13. : 10.) + (cta_rows == 256 ? 1.85 : 2.) * (double)((tiles + splits - 1) / splits) + merge;
      if (plan->cta_rows == 0 || us < least) {
        least = us;
        plan->cta_rows = cta_rows;
        plan->row_tiles = (int)row_tiles;
        plan->splits = (int)splits;
      }
    }
  }
}
Fp8Plan plan_fwd(const fa4_fp8_cache* c, const fa4_fp8_fwd* f) {
  Fp8Plan plan = {};
  const int64_t rows = (int64_t)f->Sq * (f->Hq / c->Hkv), units = (int64_t)c->Hkv * f->B;
  // us, decode kernel / kernel for many rows: 8 sequences of five rows of 32 heads over up to 4099 keys 21 / 44, 32 of eight over up to 8192 75 / 225.
  // So the change is a step: the decode kernel's tensor memory and registers end at 32 rows, and 36 to 64 rows take 227 (128 rows 168, 256 rows 210), 44 on
  // the shorter ones.
  plan.decode = rows <= 32;
  if (plan.decode) {
    plan.rows = rows <= 16 ? 16 : 32;
    plan.splits = f->num_splits;
    // Dealing the shares and merging the pieces costs about as much as ten tiles.  us, dealt / a CTA a unit: 128 units of a window of nine
    // tiles, head dim 64 19.0 / 12.6, 8 units of seven tiles 10.5 / 9.2; but 256 units of up to 64 tiles 57.6 / 71.1.
    if (plan.splits == 0 && units <= kSms && most_tiles(c, f, f->Sq) <= 10) plan.splits = 1;
    // (us, up to 8 / 4 heads side by side, which are 144 / 148 CTAs: 32 sequences of up to 8192 keys 55 / 60, drafted tokens on pages of 16 29 / 32.5)
    for (plan.bundle = std::min(8, c->Hkv); c->Hkv % plan.bundle != 0;) --plan.bundle;
    plan.slots = plan.splits == 0 ? 2 * kSms : plan.splits == 1 ? 0 : units * plan.splits;
    plan.slot_rows = rows;
  } else {
    plan_many(c, f, &plan);
    plan.slots = plan.splits == 1 ? 0 : plan.splits;
    plan.slot_rows = (int64_t)f->B * f->Sq * f->Hq;
  }
  return plan;
}
// Values, then sums, then (dealt) the pieces of the units.
int64_t workspace_of(const fa4_fp8_cache* c, const fa4_fp8_fwd* f, const Fp8Plan& plan) {
  const int64_t values = plan.slots * plan.slot_rows;
  return values * (c->D + 1) * 4 + (plan.decode && plan.splits == 0 ? (values % 2) * 4 + (int64_t)f->B * c->Hkv * 8 : 0);
}

// The pool as (D, token of a page, head, page) bytes.
bool encode_pool(CUtensorMap* m, const fa4_fp8_cache* c, const void* base, int64_t page, int64_t token, int64_t head, int box) {
  const uint64_t dims[4] = {(uint64_t)c->D, (uint64_t)c->page_size, (uint64_t)c->Hkv, (uint64_t)c->num_pages};
  const uint64_t strides[3] = {(uint64_t)token, (uint64_t)head, (uint64_t)page};
  const uint32_t boxes[4] = {(uint32_t)c->D, (uint32_t)box, 1, 1};
  return encode_u8_4d(m, base, dims, strides, boxes, c->D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace

extern "C" int64_t fa4_fp8_cache_fwd_workspace_bytes(const fa4_fp8_cache* c, const fa4_fp8_fwd* f) {
  if (int e = validate_fwd(c, f)) return e;
  return workspace_of(c, f, plan_fwd(c, f));
}

extern "C" int fa4_fp8_cache_fwd(const fa4_fp8_cache* c, const fa4_fp8_fwd* f, void* cuda_stream) {
  if (int e = validate_fwd(c, f)) return e;
  const Fp8Plan plan = plan_fwd(c, f);
  const int64_t bytes = workspace_of(c, f, plan);
  if (bytes > 0 && f->workspace == nullptr) return -FA4_E_NULL;
  if (bytes > 0 && !aligned16(f->workspace)) return -FA4_E_ALIGN;
  if (bytes > 0 && f->workspace_bytes < (uint64_t)bytes) return -FA4_E_TOO_LARGE;
  Fp8Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(f->q);
  p.out = static_cast<__nv_bfloat16*>(f->out);
  p.lse = f->lse;
  p.q_b = f->q_stride_b; p.q_s = f->q_stride_s; p.q_h = f->q_stride_h;
  p.o_b = f->o_stride_b; p.o_s = f->o_stride_s; p.o_h = f->o_stride_h;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  p.used = f->seqused_k;
  p.fresh = f->seqused_q;
  p.table = c->page_table;
  p.sink = f->sink;
  p.num_splits = plan.splits;
  p.o_partial = static_cast<float*>(f->workspace);
  p.lse_partial = bytes > 0 ? p.o_partial + plan.slots * plan.slot_rows * c->D : nullptr;
  p.pieces = bytes > 0 ? reinterpret_cast<int2*>(p.lse_partial + (plan.slots * plan.slot_rows + 1) / 2 * 2) : nullptr;
  p.unit_rows = f->Sq * (f->Hq / c->Hkv);
  p.bundle = plan.decode ? plan.bundle : 1;
  p.bundles = c->Hkv / p.bundle;
  p.row_tiles = plan.row_tiles;
  p.cta_rows = plan.cta_rows;
  // (a contiguous cache has no page borders: what lies behind its end is read as zeros)
  p.box = c->page_table == nullptr ? 128 : std::gcd(c->page_size, 128);
  p.B = f->B; p.Sq = f->Sq; p.Hq = f->Hq; p.Hkv = c->Hkv; p.group = f->Hq / c->Hkv; p.D = c->D;
  p.log_block = log2_of(c->block);
  p.num_pages = c->num_pages; p.page_size = c->page_size; p.pages_per_seq = c->pages_per_seq;
  p.capacity = c->pages_per_seq * c->page_size;
  p.div_page = make_fastdiv((uint32_t)c->page_size);
  p.div_group = make_fastdiv((uint32_t)p.group);
  p.div_hq = make_fastdiv((uint32_t)f->Hq);
  p.div_sq = make_fastdiv((uint32_t)f->Sq);
  const ScoreFactors by = factors_of(f);
  p.sl2 = by.sl2;
  p.cap_in = by.cap_in;
  p.cap_out = by.cap_out;
  p.win_left = f->window_left;
  p.win_right = f->causal && f->window_right < 0 ? 0 : f->window_right;
  p.status = f->status;
  p.epoch = next_launch_epoch();
  p.budget_ns = f->wait_budget_ns ? f->wait_budget_ns : kDefaultBudgetNs;
  CUtensorMap tm_k, tm_v;
  if (!encode_pool(&tm_k, c, c->k, c->k_stride_page, c->k_stride_token, c->k_stride_head, p.box) ||
      !encode_pool(&tm_v, c, c->v, c->v_stride_page, c->v_stride_token, c->v_stride_head, p.box))
    return -FA4_E_TENSORMAP;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const bool cap = f->softcap > 0.f;
  const int64_t rows = (int64_t)f->B * f->Sq * f->Hq;
  const unsigned merge_grid = (unsigned)((rows + kFp8CombineWarps - 1) / kFp8CombineWarps);
  if (plan.decode) {
    const int64_t grid = plan.splits == 0 ? kSms / plan.bundle * plan.bundle : (int64_t)plan.splits * c->Hkv * f->B;
    p.div_groups = make_fastdiv((uint32_t)(kSms / plan.bundle));
    auto launch = [&](auto form) -> int {
      using F = decltype(form);
      return launch_pdl(fp8_decode_kernel<F>, dim3((unsigned)grid), F::kThreads, F::kRequest, stream, tm_k, tm_v, p);
    };
    using fp8d::Form;
    auto launch_rows = [&](auto capped) -> int {
      constexpr bool kCap = decltype(capped)::value;
      if (c->D == 128) return plan.rows == 16 ? launch(Form<128, 16, kCap>{}) : launch(Form<128, 32, kCap>{});
      return plan.rows == 16 ? launch(Form<64, 16, kCap>{}) : launch(Form<64, 32, kCap>{});
    };
    const int rc = cap ? launch_rows(std::true_type{}) : launch_rows(std::false_type{});
    if (rc != 0 || plan.splits == 1) return rc;
    return launch_pdl(fp8_merge_kernel, dim3(merge_grid), kFp8CombineWarps * 32, 0, stream, p);
  }
  // (a launch needs the registers that the kernel's budget counts on: see ensure_kernel)
  auto launch_many = [&](auto kernel, uint32_t smem) -> int {
    if (int e = ensure_kernel(kernel, smem, fp8p::kRegsLaunch)) return e;
    return launch_pdl(kernel, dim3((unsigned)((int64_t)plan.row_tiles * c->Hkv * f->B * plan.splits)), fp8p::kThreads, smem, stream, tm_k, tm_v, p);
  };
  const int rc = c->D == 128 ? (cap ? launch_many(fp8_prefill_kernel<128, true>, fp8p::Layout<128>::kRequest)
                                    : launch_many(fp8_prefill_kernel<128, false>, fp8p::Layout<128>::kRequest))
                             : (cap ? launch_many(fp8_prefill_kernel<64, true>, fp8p::Layout<64>::kRequest)
                                    : launch_many(fp8_prefill_kernel<64, false>, fp8p::Layout<64>::kRequest));
  if (rc != 0 || plan.splits == 1) return rc;
  return launch_pdl(fp8_combine_kernel, dim3(merge_grid), kFp8CombineWarps * 32, 0, stream, p);
}
