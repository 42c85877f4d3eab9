// Attention over the 8-bit KV cache for many query rows (pieces of prompts).
//
// With a tile of query rows the products are bound by the tensor cores, so keys and values are turned into fp16 once for 256 rows
// (two tiles of 128 rows, of all query heads of a kv head: row r = token r / group, head r % group) and everything runs as
// kind::f16 products, in which an e4m3 value, a bf16 query (times a power of two) and their products are exact.
//
//   S (128 rows x 128 keys) = Q . K^T,    O (128 rows x D) += W . V,    W = 2^(t - m) vs / vs_max * 2^6 as fp16, from tensor memory
//
// t is the score in log2 units, m a row's reference, which follows the maximum when it falls behind by more than 8 (then O
// is multiplied); vs / vs_max the scale of a block of values over the largest that this CTA meets, so a weight is below 2^16
// and has its eleven bits down to 2^-20 of that; the row sum takes the weight without vs, in fp32.
//
// Warps: 0-3 and 4-7 the softmax of a tile each (thread = row), 8-11 turn K and V tiles into fp16 (cvt.f16x2.e4m3x2 runs at 64 a clock and
// beside the exponentials: a step of 128 keys takes 256 clocks of it, the exponentials of 256 rows 2048), 12 and 14 load,
// 13 issues the products: W V of a step and Q K^T of the next one for one tile while the other tile's softmax runs.  Tensor memory: S 2 x 128
// columns, in whose place W is written, O 2 x D.  Every wait is bounded (those of the softmax warps, which
// leave no registers for a call, by the issuer's: see mbar_wait_flag); a warp whose wait ran out goes on without waiting.
#pragma once
#include "fp8_decode.cuh"

namespace fa4 {
namespace fp8p {

enum Site { kRawFullS = 140, kRawFreeS, kHalfFullS, kHalfFreeS, kSFullS, kPFullS, kODoneS, kQReadyS };

// Registers: 512 threads launch with 128; the softmax takes what the others give back.
constexpr int kThreads = 512, kRegsLaunch = 128, kRegsSoftmax = 192, kRegsConvert = 64, kRegsService = 64;
static_assert(2 * kRegsSoftmax + kRegsConvert + kRegsService <= 4 * kRegsLaunch, "register budget of the 8-bit prefill kernel");

template <int kD>
struct Layout {
  static constexpr uint32_t kHalf = 128 * 128;                       // 128 rows x 64 fp16
  static constexpr uint32_t kTile16 = kHalf * (kD / 64), kTile8 = 128 * kD;
  static constexpr uint32_t kOffQ = 0, kOffK = 2 * kTile16, kOffV = kOffK + 2 * kTile16, kOffRawK = kOffV + 2 * kTile16,
                            kOffRawV = kOffRawK + kTile8, kOffSc = kOffRawV + kTile8,   // scales of 16 keys: 4 steps x (8 of K, 8 of V)
      kOffBar = kOffSc + 4 * 64;
  static constexpr uint32_t kRawKFull = 0, kRawKFree = 1, kRawVFull = 2, kRawVFree = 3, kKFull = 4 /* 2 */, kKFree = 6, kVFull = 8,
                            kVFree = 10, kSFull = 12, kPFull = 14, kODone = 16, kQReady = 17, kDrain = 18, kBars = 19;
  static constexpr uint32_t kOffMisc = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr uint32_t kRequest = kOffMisc + 32 + sizeof(WaitCtx) + 1024;
  static_assert(kRequest <= 227 * 1024, "shared memory of the 8-bit prefill kernel");
};
constexpr uint32_t kColS = 0, kColO = 256;

// K-major rows of 64 fp16 (128 bytes, 128-byte swizzle, groups of eight rows 1024 bytes apart).  Read MN-major the same groups
// are eight steps of the contraction, and the next 64 of the other side lie 16 KB on.
__device__ __forceinline__ uint64_t half_desc(uint32_t saddr) { return make_smem_desc(saddr, 128 * 128, 1024, kSwizzle128); }
// Instruction descriptor of kind::f16, fp16 x fp16, fp32 accumulator.
__host__ __device__ constexpr uint32_t make_idesc_f16(uint32_t m, uint32_t n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four e4m3 bytes as two pairs of fp16.
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  uint2 r;
  asm("{\n"
      ".reg .b16 l, h;\n"
      "mov.b32 {l, h}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n"
      "}\n"
      : "=r"(r.x), "=r"(r.y)
      : "r"(w));
  return r;
}

// One tile of 128 rows of kD bytes (as TMA leaves it, swizzled over a row) into halves of 64 fp16, by four warps.  A warp
// takes eight rows' 64 bytes at a time: four lanes a row, and the rows of eight lanes that access memory together lie so that reads
// and writes fall into different banks (the second of two rows writes its pieces in the other order).  Rows outside
// [row_lo, row_hi) become zeros.
template <int kD>
__device__ __forceinline__ void widen_tile(const uint8_t* raw, uint8_t* to, int warp, int lane, int row_lo, int row_hi) {
  const int c = lane & 3, second = (lane >> 2) & 1, q = lane >> 3;
  const int in8 = kD == 128 ? q + 4 * second : 2 * q + second;
#pragma unroll
  for (int k = 0; k < kD / 16; ++k) {                       // 128 rows x kD / 64 halves by 4 warps of 8 rows
    const int item = k * 4 + warp, half = item & (kD / 64 - 1), r = item / (kD / 64) * 8 + in8;
    const uint4 u = *reinterpret_cast<const uint4*>(raw + fp8d::row_piece<kD>(r, half * 4 + c));
    uint4 a, b;
    const uint2 w0 = widen4(u.x), w1 = widen4(u.y), w2 = widen4(u.z), w3 = widen4(u.w);
    a = make_uint4(w0.x, w0.y, w1.x, w1.y);
    b = make_uint4(w2.x, w2.y, w3.x, w3.y);
    if (r < row_lo || r >= row_hi) a = b = make_uint4(0u, 0u, 0u, 0u);
    uint8_t* dst = to + half * (128 * 128);
    *reinterpret_cast<uint4*>(dst + fp8d::sw128_offset(r, 2 * c + second)) = second ? b : a;
    *reinterpret_cast<uint4*>(dst + fp8d::sw128_offset(r, 2 * c + 1 - second)) = second ? a : b;
  }
}

}  // namespace fp8p

template <int kD, bool kCap>
__global__ void __launch_bounds__(fp8p::kThreads, 1)
fp8_prefill_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ Fp8Params p) {
  using namespace fp8p;
  using L = Layout<kD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](uint32_t idx) -> uint32_t { return base + L::kOffBar + 8u * idx; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::kOffMisc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gbase + L::kOffMisc + 4);
  uint32_t* s_top = reinterpret_cast<uint32_t*>(gbase + L::kOffMisc + 8);
  WaitCtx& wc = *reinterpret_cast<WaitCtx*>(gbase + L::kOffMisc + 32);
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  // row tiles from the last one on (with a causal mask the longest comes first), the kv heads and sequences of one next to each other
  int w = blockIdx.x;
  const int split = w % p.num_splits;
  w /= p.num_splits;
  const int hk = w % p.Hkv;
  w /= p.Hkv;
  const int b = w % p.B, r_first = (p.row_tiles - 1 - w / p.B) * 256;
  pdl_wait();
  const SeqLens len = lens_of(p, b);
  const int R = min(256, len.sq * p.group - r_first);
  if (R <= 0) return;
  const int lo_all = seen_by(p, len.sk, len.sq, fast_div(r_first, p.div_group)).x,
            hi_all = seen_by(p, len.sk, len.sq, fast_div(r_first + R - 1, p.div_group)).y;
  const int t_first = lo_all >> 7, t_total = hi_all > lo_all ? ((hi_all + 127) >> 7) - t_first : 0;
  const int per = (t_total + p.num_splits - 1) / p.num_splits;
  const int t0 = t_first + min(split * per, t_total), n = min(t_first + t_total - t0, per);
  const int tiles = R > 128 ? 2 : 1;
  if (tid == 0) {
    *s_abort = 0u;
    *s_top = 0u;
    wc = WaitCtx{s_abort, p.status, p.budget_ns, p.epoch};
    mbar_init(bar(L::kRawKFull), 2);         // the copies' bytes, and the scales
    mbar_init(bar(L::kRawVFull), 1);
    mbar_init(bar(L::kRawKFree), 4);
    mbar_init(bar(L::kRawVFree), 4);
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(L::kKFull + s), 4);
      mbar_init(bar(L::kVFull + s), 4);
      mbar_init(bar(L::kKFree + s), 1);
      mbar_init(bar(L::kVFree + s), 1);
      mbar_init(bar(L::kSFull + s), 1);
      mbar_init(bar(L::kPFull + s), 4);
    }
    mbar_init(bar(L::kODone), 1);
    mbar_init(bar(L::kQReady), 8);
    mbar_init(bar(L::kDrain), 1);
    fence_barrier_init();
  }
  if (warp == 12 && lane == 0) tma_prefetch_desc(&tm_k);
  if (warp == 14 && lane == 0) tma_prefetch_desc(&tm_v);
  if (warp == 13) {
    tmem_alloc(base + L::kOffMisc, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  // the largest scale of values among this CTA's keys
  const int first_key = max(lo_all, t0 << 7), end_key = min(hi_all, (t0 + n) << 7);
  {
    uint32_t top = 0u;
    for (int64_t blk = (first_key >> p.log_block) + tid; (blk << p.log_block) < end_key && n > 0; blk += kThreads) {
      const int key = (int)(blk << p.log_block), pg = fast_div(key, p.div_page), off = key - pg * p.page_size;
      const int page = p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b;
      if (page >= 0 && page < p.num_pages)
        top = max(top, __float_as_uint(p.v_scale[((int64_t)page * (p.page_size >> p.log_block) + (off >> p.log_block)) * p.Hkv + hk]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0 && top > 0u) atomicMax(s_top, top);
  }
  __syncthreads();
  // 2^6 / its power of two, and back (1 and 1 where it is no ordinary number)
  const uint32_t top_e = *s_top >> 23;
  const bool ordinary = top_e >= 20 && top_e <= 240;
  const float vs_up = ordinary ? __uint_as_float((254u + 6u - top_e) << 23) : 1.f, vs_down = ordinary ? __uint_as_float((top_e - 6u) << 23) : 1.f;
  bool ok = true;

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsService));
    if (warp == 12 || warp == 14) {
      // ============================================ loaders ======================================
      // (as in the decode kernel: lane g and g + 8 have keys 16 g .. 16 g + 15 of a step)
      const bool is_k = warp == 12;
      const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
      const float* scales = lane < 8 ? p.k_scale : p.v_scale;
      const uint32_t full = bar(is_k ? L::kRawKFull : L::kRawVFull), free = bar(is_k ? L::kRawKFree : L::kRawVFree);
      const uint32_t tile = base + (is_k ? L::kOffRawK : L::kOffRawV);
      float* s_scale = reinterpret_cast<float*>(gbase + L::kOffSc);
      auto key_of = [&](int i) { return ((t0 + i) << 7) + 16 * (lane & 7); };
      auto live = [&](int i) { return lane < 16 && i < n && key_of(i) < hi_all && key_of(i) + 16 > lo_all; };
      auto look_up = [&](int i) -> int2 {
        int2 at = make_int2(-1, 0);
        if (live(i)) {
          const int key = key_of(i), pg = fast_div(key, p.div_page);
          at = make_int2(p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b, key - pg * p.page_size);
        }
        return at;
      };
      auto scale_at = [&](int2 at) -> float {
        return is_k && at.x >= 0 && at.x < p.num_pages
                   ? scales[((int64_t)at.x * (p.page_size >> p.log_block) + (at.y >> p.log_block)) * p.Hkv + hk] * (lane < 8 ? 1.f : vs_up) : 0.f;
      };
      int2 at = look_up(0), at1 = look_up(1);
      float sc = scale_at(at);
      int i = 0;
      for (; i < n; ++i) {
        const int2 at2 = look_up(i + 2);
        const float sc1 = scale_at(at1);
        if (i > 0 && ok) ok = mbar_wait_relaxed<512>(free, (i - 1) & 1, wc, kRawFreeS);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t seen = __ballot_sync(0xffffffffu, live(i)) & 0xffu;
        const int per_box = p.box >> 4;
        const uint32_t in_box = (seen >> lane) & ((1u << per_box) - 1u);
        const bool mine = lane < 8 && (lane & (per_box - 1)) == 0 && in_box != 0u;
        const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) mbar_arrive_expect_tx(full, boxes * (uint32_t)p.box * kD);
        __syncwarp();
        const int src = mine ? lane + __ffs(in_box) - 1 : lane;
        const int page = __shfl_sync(0xffffffffu, at.x, src & 31), off = __shfl_sync(0xffffffffu, at.y, src & 31) - 16 * (src - lane);
        if (mine) {
          const bool fine = page >= 0 && page < p.num_pages;
          if (!fine) report_bad_index(p.status, p.epoch, kPageSite);
          tma_load_4d(tile + 16 * lane * kD, tm, full, 0, off, hk, fine ? page : p.num_pages);
        }
        if (is_k) {
          // (Q K^T of step i - 2 is done before this step is converted, and so the softmax of step i - 3: four slots are enough)
          if (lane < 16) s_scale[(i & 3) * 16 + lane] = sc;
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
        }
        at = at1; at1 = at2; sc = sc1;
      }
      if (!ok && i > 0 && lane == 0) {
        const uint64_t begun = globaltimer_ns();
        while (!mbar_try_wait(full, (i - 1) & 1) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
      }
    } else if (warp == 13) {
      // ============================================ products =====================================
      if (elect_one() && n > 0) {
        constexpr uint32_t idesc_s = make_idesc_f16(128, 128, false), idesc_o = make_idesc_f16(128, kD, true);
        // (products run in the order they are issued: Q K^T of a tile's next step may overwrite the weights that W V in front of it reads)
        // (descriptors are moved, not made anew: see the issuers of the decode kernel)
        using fp8d::desc_at;
        const uint64_t dq = half_desc(base + L::kOffQ), dk = half_desc(base + L::kOffK), dv = half_desc(base + L::kOffV);
        auto score = [&](uint32_t t, uint32_t buf) {
          const uint64_t qt = desc_at(dq, t * L::kTile16), kt = desc_at(dk, buf * L::kTile16);
          const uint32_t to = tmem + kColS + 128 * t;
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks) {
            const uint32_t at = (ks >> 2) * L::kHalf + (ks & 3) * 32;
            mma_f16_ss(to, desc_at(qt, at), desc_at(kt, at), idesc_s, ks > 0);
          }
          tc_commit(bar(L::kSFull + t));
        };
        ok = mbar_wait(bar(L::kQReady), 0, wc, kQReadyS) && mbar_wait(bar(L::kKFull), 0, wc, kHalfFullS);
        if (ok) {
          tc_fence_after_sync();
          for (int t = 0; t < tiles; ++t) score(t, 0);
          tc_commit(bar(L::kKFree));
        }
        uint32_t buf = 0, parity = 0;          // of step i
#pragma unroll 1
        for (int i = 0; ok && i < n; ++i) {
          const bool more = i + 1 < n;
          ok = mbar_wait(bar(L::kVFull + buf), parity, wc, kHalfFullS);
          if (ok && more) ok = mbar_wait(bar(L::kKFull + (buf ^ 1u)), parity ^ buf, wc, kHalfFullS);
          const uint64_t vt = desc_at(dv, buf * L::kTile16);
#pragma unroll 1
          for (int t = 0; ok && t < tiles; ++t) {
            ok = mbar_wait(bar(L::kPFull + t), i & 1, wc, kPFullS);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t to = tmem + kColO + kD * t, w = tmem + kColS + 128 * t;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) mma_f16_ts(to, w + 8 * ks, desc_at(vt, 2048 * ks), idesc_o, i > 0 || ks > 0);
            if (more) score(t, buf ^ 1u);
          }
          if (ok) {
            tc_commit(bar(L::kVFree + buf));
            if (more) tc_commit(bar(L::kKFree + (buf ^ 1u)));
          }
          parity ^= buf;
          buf ^= 1u;
        }
        if (ok) {
          tc_commit(bar(L::kODone));
          ok = mbar_wait(bar(L::kODone), 0, wc, kODoneS);     // (for the softmax warps, which wait without a clock)
        }
        const uint64_t begun = globaltimer_ns();
        if (!ok) {
          tc_commit(bar(L::kDrain));
          while (!mbar_try_wait(bar(L::kDrain), 0) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
        }
      }
    }
  } else if (warp >= 8) {
    // ============================================ e4m3 -> fp16 ===================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    for (int i = 0; i < n; ++i) {
      const int key0 = (t0 + i) << 7;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const uint32_t full = bar(v ? L::kVFull : L::kKFull) + 8 * (i & 1);
        if (ok) ok = mbar_wait(bar(v ? L::kRawVFull : L::kRawKFull), i & 1, wc, kRawFullS);
        if (ok && i >= 2) ok = mbar_wait(bar(v ? L::kVFree : L::kKFree) + 8 * (i & 1), ((i >> 1) - 1) & 1, wc, kHalfFreeS);
        ok = __all_sync(0xffffffffu, ok);
        // (values that no row sees may be anything, and 0 * NaN is NaN)
        widen_tile<kD>(gbase + (v ? L::kOffRawV : L::kOffRawK), gbase + (v ? L::kOffV : L::kOffK) + (i & 1) * L::kTile16, warp - 8, lane,
                       v ? lo_all - key0 : 0, v ? hi_all - key0 : 128);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(v ? L::kRawVFree : L::kRawKFree));
          mbar_arrive(full);
        }
      }
    }
  } else {
    // ============================================ softmax ======================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int tile = warp >> 2, t = tid & 127, row = tile * 128 + t;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem + lanes + kColS + 128 * tile, tm_o = tmem + lanes + kColO + kD * tile;
    const int s = fast_div(r_first + row, p.div_group), h = hk * p.group + r_first + row - s * p.group;
    // ---- Q: the thread's row, times the power of two that brings its largest element to 128 .. 256
    float factor = 0.f;
    {
      uint8_t* qt = gbase + L::kOffQ + tile * L::kTile16;
      uint4 u[kD / 8];
      uint32_t top = 0u;
      const __nv_bfloat16* src = p.q + b * p.q_b + (int64_t)s * p.q_s + h * p.q_h;
#pragma unroll
      for (int c = 0; c < kD / 8; ++c) u[c] = row < R ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int c = 0; c < kD / 8; ++c) {
        const uint32_t w4[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max((w4[k] << 16) & 0x7fffffffu, w4[k] & 0x7fff0000u));
      }
      const int e = max((int)(top >> 23), 17);
      const float up = __uint_as_float((uint32_t)(254 + 7 - e) << 23), down = __uint_as_float((uint32_t)(e - 7) << 23);
      factor = (kCap ? p.cap_in : p.sl2) * down;
#pragma unroll
      for (int c = 0; c < kD / 8; ++c) {
        float x[8];
        unpack8(u[c], x);
        uint4 o = make_uint4(pack_f16x2(x[0] * up, x[1] * up), pack_f16x2(x[2] * up, x[3] * up), pack_f16x2(x[4] * up, x[5] * up),
                             pack_f16x2(x[6] * up, x[7] * up));
        if (top >= 0x7f800000u) o = make_uint4(0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u);   // (not finite: NaN whole)
        *reinterpret_cast<uint4*>(qt + (c >> 3) * L::kHalf + fp8d::sw128_offset(t, c & 7)) = o;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(L::kQReady));
    }
    int lo = 0, hi = 0;
    if (row < R) {
      const int2 see = seen_by(p, len.sk, len.sq, s);
      lo = see.x;
      hi = see.y;
    }
    float m_ref = -INFINITY;
    float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    if (tile < tiles) {
      for (int i = 0; i < n; ++i) {
        if (ok) ok = mbar_wait_flag(bar(L::kSFull + tile), i & 1, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after_sync();
        float x[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tm_s + 32 * c, reinterpret_cast<uint32_t*>(x + 32 * c));
        tc_wait_ld();
        const float4* sc4 = reinterpret_cast<const float4*>(gbase + L::kOffSc + (i & 3) * 64);
        const float4 ka = sc4[0], kb = sc4[1];
        const float ks[8] = {ka.x, ka.y, ka.z, ka.w, kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float2 f = make_float2(ks[g] * factor, ks[g] * factor);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float2 y = __fmul2_rn(make_float2(x[16 * g + 2 * j], x[16 * g + 2 * j + 1]), f);
            if constexpr (kCap) y = make_float2(p.cap_out * tanh_of(y.x), p.cap_out * tanh_of(y.y));
            x[16 * g + 2 * j] = y.x;
            x[16 * g + 2 * j + 1] = y.y;
          }
        }
        const int lo_in = lo - ((t0 + i) << 7), hi_in = hi - ((t0 + i) << 7);
        if (__any_sync(0xffffffffu, lo_in > 0 || hi_in < 128)) {
#pragma unroll
          for (int j = 0; j < 128; ++j) x[j] = j >= lo_in && j < hi_in ? x[j] : -INFINITY;
        }
        float top = fmaxf(x[0], x[1]);
#pragma unroll
        for (int j = 2; j < 128; j += 2) top = fmax3(top, x[j], x[j + 1]);
        // the reference follows when the row's weights would pass 2^8
        float fac = 1.f;
        const bool moved = top > m_ref + 8.f;
        if (moved) {
          fac = ex2_approx(m_ref - top);
          m_ref = top;
          l2[0].x *= fac; l2[0].y *= fac; l2[1].x *= fac; l2[1].y *= fac;
        }
        if (i > 0 && __any_sync(0xffffffffu, moved)) {
          // (the scores of this step are behind W V of the last one)
#pragma unroll 1
          for (int c = 0; c < kD / 16; ++c) {
            float o[16];
            dec::tmem_ld16(tm_o + 16 * c, reinterpret_cast<uint32_t*>(o));
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] *= fac;
            dec::tmem_st16(tm_o + 16 * c, reinterpret_cast<const uint32_t*>(o));
          }
        }
        const float ref = m_ref == -INFINITY ? 0.f : -m_ref;
        const float2 ref2 = make_float2(ref, ref);
        const float4 va = sc4[2], vb = sc4[3];
        const float vs[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pw[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int k = 32 * c + 2 * j;
            const float2 y = __fadd2_rn(make_float2(x[k], x[k + 1]), ref2);
            const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            l2[j & 1] = __fadd2_rn(l2[j & 1], e);
            const float2 wv = __fmul2_rn(e, make_float2(vs[k >> 4], vs[k >> 4]));
            pw[j] = pack_f16x2(wv.x, wv.y);
          }
          dec::tmem_st16(tm_s + 16 * c, pw);
        }
        tc_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::kPFull + tile));
      }
      // ---- the row's result
      if (n > 0) {
        if (ok) ok = mbar_wait_flag(bar(L::kODone), 0, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after_sync();
      }
      const float l = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
      const int64_t l_idx = ((int64_t)b * p.Hq + h) * p.Sq + s;
      const bool none = m_ref == -INFINITY && l == 0.f;
      const RowEnd end = finish_row(m_ref, l, p.sink, h);
      const bool direct = p.num_splits == 1;
      const int64_t rows = (int64_t)p.B * p.Sq * p.Hq, part = (int64_t)split * rows;
      const float scale = (direct ? end.factor : 1.f / l) * vs_down;
      if (ok && row < R) {
        if (direct && p.lse != nullptr) p.lse[l_idx] = end.lse;
        if (!direct) p.lse_partial[part + ((int64_t)b * p.Sq + s) * p.Hq + h] = none ? -INFINITY : m_ref + log2f(l);
      }
#pragma unroll 1
      for (int c = 0; c < kD / 32; ++c) {
        float o[32];
        if (n > 0) {
          tmem_ld32(tm_o + 32 * c, reinterpret_cast<uint32_t*>(o));
          tc_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0.f;
        }
        if (!ok || row >= R) {
        } else if (direct) {
          uint4* dst = reinterpret_cast<uint4*>(p.out + b * p.o_b + (int64_t)s * p.o_s + h * p.o_h + 32 * c);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[j] = make_uint4(pack_bf16x2(o[8 * j] * scale, o[8 * j + 1] * scale), pack_bf16x2(o[8 * j + 2] * scale, o[8 * j + 3] * scale),
                                pack_bf16x2(o[8 * j + 4] * scale, o[8 * j + 5] * scale), pack_bf16x2(o[8 * j + 6] * scale, o[8 * j + 7] * scale));
        } else if (!none) {
          float4* dst = reinterpret_cast<float4*>(p.o_partial + (part + ((int64_t)b * p.Sq + s) * p.Hq + h) * kD + 32 * c);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j] * scale, o[4 * j + 1] * scale, o[4 * j + 2] * scale, o[4 * j + 3] * scale);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace fa4
