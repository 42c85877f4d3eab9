// Attention over the 8-bit KV cache for many query rows (pieces of prompts).
//
//   S (128 rows x 128 keys) = Q . K^T  in e4m3: the keys as they are loaded, a bf16 query as two e4m3 rows (see the decode kernel)
//   O (128 rows x D) += W . V          in fp16: values widened to fp16 (exact), weights from tensor memory
//
// W = 2^(t - v) vs 2^6 with t the score in log2 units, vs the scale of the key's block of values and v a row's reference, which follows the row's largest
// t + log2 vs when it falls behind by more than 8 (then O is multiplied): a weight is 2^14 at most and has its eleven bits down to 2^-20 of that
// reference, whatever values the rows beside it see.  Two e4m3 rows would not do here: O stays in tensor memory, so the reference is one of all
// keys so far, and what lies 2^13 below it would lose its bits.  The row sum takes 2^(t - m) in fp32, m a reference of the scores alone.
//
// A CTA has two tiles of 128 rows (row r = token r / group, head r % group of a kv head), a softmax warpgroup each (thread = row).  The scores of a
// tile have two halves of 64 columns, which the steps take in turn: the upper scores (keys 64-127) come first, the lower ones to the same columns when
// those are in registers, the weights of both where the lower scores were.  Meanwhile the next step's upper scores go to the other half.  So the softmax finds
// its next scores waiting (with one product of 128 columns it waited 1500 of 4000 clocks for W V and Q K^T: 294 us for the first call below), and no product
// overwrites weights that another one may still read (Q K^T behind W V by issue alone 236 us, upper scores always in the same half and W V waited for 254-267).
//
// What bounds it: no unit alone.  A step of 256 rows x 128 keys takes about 3400 clocks: the exponentials 2048, the products 2560 (Q K^T in halves of 64
// columns 48 clocks an instruction, bound by shared memory), 1800 issue slots a scheduler, in chains between two warps of a scheduler.  D = 128, B = 1:
// 1024 rows of 32 heads on 16384 keys 241 us back to back (162 at the measured rate of bf16 products), tensor pipe 60 %, exponential unit 60 %, issue slots
// 53 % busy; 8192 rows of 64 heads on as many keys, causal, 975 us at first and 1110 under the power cap
// (669, or 793 at the sustained rate).  A CTA's start and end take 12000 clocks, 8000 of them Q.
// Tried on a form of 238 us: exponentials by polynomials, one in eight 253, one in four 261 (more instructions between the others); the logarithm of a value
// scale in the exponents where a half has one 248; the lower scores loaded in front of the upper exponentials or between them 282, 247.
//
// Over chosen blocks (kBlocks) the CTA's rows are those of one query block, its keys the blocks of that one's list one behind the other (see the decode kernel).  2048 rows of 32 heads, 64 rows
// choose 64 blocks of 64: 169 us, two rounds of CTAs of 32 steps; a step 4000 clocks, since chosen blocks differ in level and the references of some row move in most of them.
//
// Warps: 0-3 and 4-7 softmax, 8-11 widen the tiles of V (cvt.f16x2.e4m3x2 runs at 64 a clock beside the exponentials), 12 and 14 load, 13 issues
// the products.  Every wait is bounded (those of the softmax warps, which leave no registers for a call, by the issuer's: see mbar_wait_flag); a warp
// whose wait ran out goes on without waiting.
#pragma once
#include "fp8_decode.cuh"

namespace fa4 {
namespace fp8p {

enum Site { kKFullS = 140, kKFreeS, kRawFullS, kRawFreeS, kHalfFullS, kHalfFreeS, kUFreeS, kPFullS, kODoneS, kQReadyS, kPvDoneS };

// Registers: 512 threads launch with 128; the softmax takes what the others give back.
constexpr int kThreads = 512, kRegsLaunch = 128, kRegsSoftmax = 192, kRegsConvert = 64, kRegsService = 64;
static_assert(2 * kRegsSoftmax + kRegsConvert + kRegsService <= 4 * kRegsLaunch, "register budget of the 8-bit prefill kernel");
constexpr uint32_t kHalf = 128 * 128;                                // 128 rows x 64 fp16

template <int kD>
struct Layout {
  static constexpr int kStagesK = 3, kStagesV = 2;                   // tiles of bytes
  // (Q K^T of step i is done before its place is loaded anew; the softmax is at step i - 1 then, and a batch of scales four ahead)
  static constexpr int kScales = kStagesK + 6;
  static constexpr uint32_t kTile16 = kHalf * (kD / 64), kTile8 = 128 * kD;
  static constexpr uint32_t kOffQ = 0 /* 2 tiles x (q1, q2) */, kOffK = 4 * kTile8, kOffRawV = kOffK + kStagesK * kTile8,
                            kOffV = kOffRawV + kStagesV * kTile8, kOffSc = kOffV + 2 * kTile16, kOffBox = kOffSc + kScales * 96, kOffRow = kOffBox + 512 /* factor of a row's scores */,
                            kOffBar = kOffRow + 256 * 4;
  static constexpr uint32_t kKFull = 0, kKFree = kKFull + kStagesK, kRawFull = kKFree + kStagesK, kRawFree = kRawFull + kStagesV,
                            kVFull = kRawFree + kStagesV, kVFree = kVFull + 2, kUFull = kVFree + 2, kLFull = kUFull + 2, kUFree = kLFull + 2,
                            kPFull = kUFree + 2, kPvDone = kPFull + 2, kODone = kPvDone + 2, kQReady = kODone + 1, kDrain = kQReady + 1,
                            kBars = kDrain + 1;
  static constexpr uint32_t kOffMisc = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr uint32_t kRequest = kOffMisc + 32 + sizeof(WaitCtx) + 1024;
  static_assert(kRequest <= 227 * 1024, "shared memory of the 8-bit prefill kernel");
};
constexpr uint32_t kColS = 0, kColO = 256;

// A widened tile: halves of 64 columns, rows of 128 bytes (128-byte swizzle, groups of eight rows 1024 bytes apart).  Read MN-major the groups
// are eight steps of the contraction, and the next 64 columns lie a half on.
__device__ __forceinline__ uint64_t half_desc(uint32_t saddr) { return make_smem_desc(saddr, kHalf, 1024, kSwizzle128); }
// Instruction descriptor of kind::f16, fp16 x fp16, fp32 accumulator.
__host__ __device__ constexpr uint32_t make_idesc_f16(uint32_t m, uint32_t n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
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
// The smaller of two, NaN if one is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
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

// x to cap * tanh(x).  While no score of the warp's 64 keys is beyond 0.5 (a cap lies well above what scores mostly are), tanh x / x is a polynomial in
// x^2 through its values at the four Chebyshev nodes of [0, 0.5^2]: off by 6e-7 of the value, and
// without the two special functions of tanh_of, which with the weight's own would bound the kernel.  Three sequences of up to 333 rows on up to 2048 keys,
// in a kernel that takes 49.6 now: tanh_of alone 56 us, six nodes of [0, 0.75^2] 49.1, four 46.7.
__device__ __forceinline__ void cap_scores(float (&x)[64], float cap) {
  float far = fabsf(x[0]);
#pragma unroll
  for (int j = 1; j < 63; j += 2) far = fmax3(far, fabsf(x[j]), fabsf(x[j + 1]));
  far = fmaxf(far, fabsf(x[63]));
  if (__any_sync(0xffffffffu, far > 0.5f)) {
#pragma unroll
    for (int j = 0; j < 64; ++j) x[j] = cap * tanh_of(x[j]);
  } else {
    constexpr float kC[4] = {0.99999945f, -0.33326284f, 0.13189939f, -0.044392738f};
    float2 c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = make_float2(cap * kC[k], cap * kC[k]);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float2 v = make_float2(x[2 * j], x[2 * j + 1]), z = __fmul2_rn(v, v);
      float2 y = c[3];
#pragma unroll
      for (int k = 2; k >= 0; --k) y = __ffma2_rn(y, z, c[k]);
      y = __fmul2_rn(y, v);
      x[2 * j] = y.x;
      x[2 * j + 1] = y.y;
    }
  }
}

}  // namespace fp8p

// kBlocks: over the blocks that the row tile's query block has chosen.
template <int kD, bool kCap, bool kBlocks = false>
__global__ void __launch_bounds__(fp8p::kThreads, 1)
fp8_prefill_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ Fp8Params p) {
  using namespace fp8p;
  using fp8d::desc_at;
  using fp8d::Ring;
  using L = Layout<kD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](uint32_t idx) -> uint32_t { return base + L::kOffBar + 8u * idx; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::kOffMisc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gbase + L::kOffMisc + 4);
  WaitCtx& wc = *reinterpret_cast<WaitCtx*>(gbase + L::kOffMisc + 32);
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  // row tiles from the last one on (with a causal mask the longest comes first), the kv heads and sequences of one next to each other
  int w = blockIdx.x;
  const int split = w % p.num_splits;
  w /= p.num_splits;
  const int hk = w % p.Hkv;
  w /= p.Hkv;
  const int v = w % p.seqs, r_first = (p.row_tiles - 1 - w / p.seqs) * p.cta_rows;
  const QueryBlock place = query_block_of<kBlocks>(p, v);
  const int b = place.b, q0 = place.q0;                 // sequence, and row of the call that the unit's first one is
  pdl_wait();
  const SeqLens len = unit_lens<kBlocks>(p, v);
  const int R = min(p.cta_rows, len.sq * p.group - r_first);
  if (R <= 0) return;
  const int s_first = fast_div(r_first, p.div_group), s_last = fast_div(r_first + R - 1, p.div_group);
  int lo_all = 0, hi_all;
  const int32_t* list = nullptr;
  if constexpr (kBlocks) {
    list = list_of(p, v, hk);
    hi_all = keys_in_front(p, list, len.sk + s_last + 1);
  } else {
    lo_all = seen_by(p, len.sk, len.sq, s_first).x;
    hi_all = seen_by(p, len.sk, len.sq, s_last).y;
  }
  const int t_first = lo_all >> 7, t_total = hi_all > lo_all ? ((hi_all + 127) >> 7) - t_first : 0;
  const int per = (t_total + p.num_splits - 1) / p.num_splits;
  const int t0 = t_first + min(split * per, t_total), n = min(t_first + t_total - t0, per);
  const int tiles = R > 128 ? 2 : 1;
  if (tid == 0) {
    *s_abort = 0u;
    wc = WaitCtx{s_abort, p.status, p.budget_ns, p.epoch};
    for (int s = 0; s < L::kStagesK; ++s) {
      mbar_init(bar(L::kKFull + s), 1);
      mbar_init(bar(L::kKFree + s), 1);
    }
    for (int s = 0; s < L::kStagesV; ++s) {
      mbar_init(bar(L::kRawFull + s), 1);
      mbar_init(bar(L::kRawFree + s), 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(L::kVFull + s), 4);
      mbar_init(bar(L::kVFree + s), 1);
      mbar_init(bar(L::kUFull + s), 1);
      mbar_init(bar(L::kLFull + s), 1);
      mbar_init(bar(L::kUFree + s), 4);
      mbar_init(bar(L::kPFull + s), 4);
      mbar_init(bar(L::kPvDone + s), 1);
    }
    mbar_init(bar(L::kODone), 1);
    mbar_init(bar(L::kQReady), 12);
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
  bool ok = true;
  if (warp < 12) {
    // ---- Q by all but the service warps, a row's pieces of eight elements by neighbouring lanes: a row as two e4m3 rows, times the
    //      power of two that brings its largest element to 128 .. 256.  All on their way at once, to where V's widened tiles
    //      will be (one after another from registers took 14000 clocks).
    constexpr int kPieces = kD / 8;
    float* s_row = reinterpret_cast<float*>(gbase + L::kOffRow);
#pragma unroll 4
    for (int i = tid; i < p.cta_rows * kPieces; i += 384) {
      const int r = i / kPieces, ch = i % kPieces, s = fast_div(r_first + r, p.div_group), h = hk * p.group + r_first + r - s * p.group;
      const __nv_bfloat16* src = r < R ? p.q + b * p.q_b + (int64_t)(q0 + s) * p.q_s + h * p.q_h + 8 * ch : p.q;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + L::kOffV + 16 * i), "l"(src), "r"(r < R ? 16 : 0) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // (two pieces at a time: 2048 rows over chosen blocks 172 -> 169 us, 1024 rows on 16384 keys 244 -> 241; four 174, 242)
#pragma unroll 2
    for (int i = tid; i < p.cta_rows * kPieces; i += 384) {
      const int r = i / kPieces, ch = i % kPieces;
      const uint4 u = *reinterpret_cast<const uint4*>(gbase + L::kOffV + 16 * i);
      float x[8], y[8];
      unpack8(u, x);
      uint32_t top = 0u;                      // (bit patterns: NaN is the largest)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < kPieces; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int e = max((int)(top >> 23), 17);
      const float up = __uint_as_float((uint32_t)(254 + 7 - e) << 23), down = __uint_as_float((uint32_t)(e - 7) << 23);
      const bool fine = top < 0x7f800000u;                   // (a row that is not finite becomes NaN whole)
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= up;
      uint2 q1 = make_uint2(pack4_e4m3(x[0], x[1], x[2], x[3]), pack4_e4m3(x[4], x[5], x[6], x[7]));
      unpack4_e4m3(q1.x, y);
      unpack4_e4m3(q1.y, y + 4);
      const uint2 q2 = make_uint2(pack4_e4m3(x[0] - y[0], x[1] - y[1], x[2] - y[2], x[3] - y[3]),
                                  pack4_e4m3(x[4] - y[4], x[5] - y[5], x[6] - y[6], x[7] - y[7]));
      if (!fine) q1 = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
      uint8_t* to = gbase + L::kOffQ + 2 * (r >> 7) * L::kTile8 + fp8d::row_piece<kD>(r & 127, ch >> 1) + (ch & 1) * 8;
      *reinterpret_cast<uint2*>(to) = q1;
      *reinterpret_cast<uint2*>(to + L::kTile8) = q2;
      if (ch == 0) s_row[r] = (kCap ? p.cap_in : p.sl2) * down;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(L::kQReady));
    asm volatile("bar.sync 1, 384;" ::: "memory");             // (the factors of the rows)
  }

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsService));
    if (warp == 12) {
      fp8d::Feeder<kD, L::kStagesK, L::kScales, true, kBlocks> feed;
      feed.tm = &tm_k;
      feed.full0 = bar(L::kKFull);
      feed.free0 = bar(L::kKFree);
      feed.part = 0u;
      feed.tiles = base + L::kOffK;
      feed.ring = gbase + L::kOffK;
      feed.scales = reinterpret_cast<float*>(gbase + L::kOffSc);
      feed.box = reinterpret_cast<int2*>(gbase + L::kOffBox);
      feed.site = {kKFreeS, kKFullS};
      feed.piece(p, wc, n, t0, b, hk, lo_all, hi_all, list);
      feed.drain();
    } else if (warp == 14) {
      fp8d::Feeder<kD, L::kStagesV, L::kScales, false, kBlocks> feed;
      feed.tm = &tm_v;
      feed.full0 = bar(L::kRawFull);
      feed.free0 = bar(L::kRawFree);
      feed.part = 0u;
      feed.tiles = base + L::kOffRawV;
      feed.ring = gbase + L::kOffRawV;
      feed.scales = nullptr;
      feed.box = reinterpret_cast<int2*>(gbase + L::kOffBox) + 32;
      feed.site = {kRawFreeS, kRawFullS};
      feed.piece(p, wc, n, t0, b, hk, lo_all, hi_all, list);
      feed.drain();
    } else if (warp == 13) {
      // ============================================ products =====================================
      // (Products are ordered by issue only where they share an accumulator and a shape: what is overwritten is waited for.
      // Descriptors are moved, not made anew: see the issuers of the decode kernel.)
      if (elect_one() && n > 0) {
        constexpr uint32_t idesc_s = fp8d::make_idesc_e4m3(128, 64, false), idesc_o = make_idesc_f16(128, kD, true);
        const uint64_t dq = fp8d::tile_desc<kD>(base + L::kOffQ), dk = fp8d::tile_desc<kD>(base + L::kOffK), dv = half_desc(base + L::kOffV);
        // scores of tile t, upper or lower keys of the K tile at place `at`, to a half of its columns
        auto score = [&](uint32_t t, uint32_t at, bool upper, uint32_t half) {
          const uint64_t qt = desc_at(dq, 2 * t * L::kTile8), kt = desc_at(dk, at * L::kTile8 + (upper ? 64 * kD : 0));
          const uint32_t to = tmem + kColS + 128 * t + 64 * half;
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks)
            fp8d::mma_e4m3(to, desc_at(qt, ks / (kD / 32) * L::kTile8 + 32 * (ks % (kD / 32))), desc_at(kt, 32 * (ks % (kD / 32))), idesc_s, ks > 0);
          tc_commit(bar((upper ? L::kUFull : L::kLFull) + t));
        };
        Ring<L::kStagesK> kk;
        ok = mbar_wait(bar(L::kQReady), 0, wc, kQReadyS) && mbar_wait(bar(L::kKFull), 0, wc, kKFullS);
        if (ok) {
          tc_fence_after_sync();
          for (int t = 0; t < tiles; ++t) score(t, 0, true, 1);
          for (int t = 0; t < tiles; ++t) score(t, 0, false, 0);
          tc_commit(bar(L::kKFree));
          kk.next();
        }
        uint32_t buf = 0, parity = 0;          // of V of step i
#pragma unroll 1
        for (int i = 0; ok && i < n; ++i) {
          const bool more = i + 1 < n;
          const uint32_t half = (i + 1) & 1;   // of step i + 1
          // (what is most often there already is asked for at once: a wait of its own costs 110 clocks even then)
          if (more) {
            // what was in that half: the upper scores of step 0, the weights of step i - 1
            const uint32_t two = tiles - 1, gone = bar(i == 0 ? L::kUFree : L::kPvDone), site = i == 0 ? kUFreeS : kPvDoneS, phase = i == 0 ? 0 : half;
            const bool kf = mbar_poll(bar(L::kKFull + kk.at), kk.parity), vf = mbar_poll(bar(L::kVFull + buf), parity),
                       g0 = mbar_poll(gone, phase), g1 = mbar_poll(gone + 8 * two, phase);
            if (!(kf && vf && g0 && g1))
              ok = mbar_wait(bar(L::kKFull + kk.at), kk.parity, wc, kKFullS) && mbar_wait(bar(L::kVFull + buf), parity, wc, kHalfFullS) &&
                   mbar_wait(gone, phase, wc, site) && mbar_wait(gone + 8 * two, phase, wc, site);
            if (!ok) break;
            tc_fence_after_sync();
#pragma unroll 1
            for (int t = 0; t < tiles; ++t) score(t, kk.at, true, half);
          } else {
            ok = mbar_wait(bar(L::kVFull + buf), parity, wc, kHalfFullS);
          }
          const uint64_t vt = desc_at(dv, buf * L::kTile16);
#pragma unroll 1
          for (int t = 0; ok && t < tiles; ++t) {
            ok = mbar_wait(bar(L::kPFull + t), i & 1, wc, kPFullS);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t to = tmem + kColO + kD * t, from = tmem + kColS + 128 * t + 64 * (i & 1);
            // (the weights of the upper keys come first)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) mma_f16_ts(to, from + 8 * ks, desc_at(vt, 2048 * (ks ^ 4)), idesc_o, i > 0 || ks > 0);
            tc_commit(bar(L::kPvDone + t));
            if (more) {
              // (the softmax takes the upper scores as soon as it has handed its weights on)
              ok = mbar_wait(bar(L::kUFree + t), half, wc, kUFreeS);
              if (!ok) break;
              tc_fence_after_sync();
              score(t, kk.at, false, half);
            }
          }
          if (ok) {
            tc_commit(bar(L::kVFree + buf));
            if (more) {
              tc_commit(bar(L::kKFree + kk.at));
              kk.next();
            }
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
    // ============================================ V: e4m3 -> fp16 ================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    Ring<L::kStagesV> raw;
    Ring<2> to;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int key0 = (t0 + i) << 7;
      if (ok) ok = mbar_wait(bar(L::kRawFull + raw.at), raw.parity, wc, kRawFullS);
      if (ok && i >= 2) ok = mbar_wait(bar(L::kVFree + to.at), to.parity ^ 1u, wc, kHalfFreeS);
      ok = __all_sync(0xffffffffu, ok);
      // (values that no row sees may be anything, and 0 * NaN is NaN)
      widen_tile<kD>(gbase + L::kOffRawV + raw.at * L::kTile8, gbase + L::kOffV + to.at * L::kTile16, warp - 8, lane, lo_all - key0, hi_all - key0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(L::kRawFree + raw.at));
        mbar_arrive(bar(L::kVFull + to.at));
      }
      raw.next();
      to.next();
    }
  } else {
    // ============================================ softmax ======================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int tile = warp >> 2, t = tid & 127, row = tile * 128 + t;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem + lanes + kColS + 128 * tile, tm_o = tmem + lanes + kColO + kD * tile;
    const int s = fast_div(r_first + row, p.div_group), h = hk * p.group + r_first + row - s * p.group;
    const float factor = reinterpret_cast<const float*>(gbase + L::kOffRow)[row];
    int lo = 0, hi = 0;
    if constexpr (kBlocks) {
      // (the tokens of the warp's rows, one after the other)
      const int s0 = fast_div(r_first + (row & ~31), p.div_group), s1 = min(fast_div(r_first + (row | 31), p.div_group), s_last);
#pragma unroll 1
      for (int at = s0; at <= s1; ++at) {
        const int keys = keys_in_front(p, list, len.sk + at + 1);
        if (at == s && row < R) hi = keys;
      }
    } else if (row < R) {
      const int2 see = seen_by(p, len.sk, len.sq, s);
      lo = see.x;
      hi = see.y;
    }
    float m_ref = -INFINITY, v_ref = -INFINITY, v_up = 0.f;     // references of the sum and of O; 2^(m_ref - v_ref + 6)
    float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    if (tile < tiles) {
      int slot = 0;
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const float* sc = reinterpret_cast<const float*>(gbase + L::kOffSc) + slot * 24;
        if (++slot == L::kScales) slot = 0;
        uint32_t wu[32];
        const uint32_t tm_half = tm_s + 64 * (i & 1);
        // 64 scores to weights (two to a word); `upper`: keys 64-127 of the step
        auto weights = [&](float (&x)[64], const bool upper, uint32_t (&pw)[32]) {
          const float4 ks = *reinterpret_cast<const float4*>(sc + (upper ? 4 : 0));
          float kf[4] = {ks.x * factor, ks.y * factor, ks.z * factor, ks.w * factor};
          const int key0 = ((t0 + i) << 7) + (upper ? 64 : 0), lo_in = lo - key0, hi_in = hi - key0;
          const bool part = __any_sync(0xffffffffu, lo_in > 0 || hi_in < 64);
          auto hide = [&](float as) {
#pragma unroll
            for (int j = 0; j < 64; ++j) x[j] = j >= lo_in && j < hi_in ? x[j] : as;
          };
          if constexpr (kCap) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float2 y = __fmul2_rn(make_float2(x[2 * j], x[2 * j + 1]), make_float2(kf[j >> 3], kf[j >> 3]));
              x[2 * j] = y.x;
              x[2 * j + 1] = y.y;
            }
            // (what a row does not see may be anything and has no say in how the others are capped)
            if (part) hide(0.f);
            cap_scores(x, p.cap_out);
          } else {
            // (the factors go into the exponents' multiply-add and the groups' maxima; 0 would make NaN of a masked score)
#pragma unroll
            for (int k = 0; k < 4; ++k) kf[k] = kf[k] == 0.f ? 1.17549435e-38f : kf[k];
          }
          if (part) hide(-INFINITY);
          const float4 lv4 = *reinterpret_cast<const float4*>(sc + 16 + (upper ? 4 : 0));
          const float lv[4] = {lv4.x, lv4.y, lv4.z, lv4.w};
          float top = -INFINITY, top_v = -INFINITY;             // of the scores; of the weights with the values' scales
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float m = fmaxf(x[16 * k], x[16 * k + 1]);
#pragma unroll
            for (int j = 2; j < 16; j += 2) m = fmax3(m, x[16 * k + j], x[16 * k + j + 1]);
            top = fmaxf(top, kCap ? m : m * kf[k]);
            top_v = fmaxf(top_v, kCap ? m + lv[k] : fmaf(m, kf[k], lv[k]));
          }
          // the references follow when the row's weights would pass 2^8, without or with the values' scales
          const bool moved = top > m_ref + 8.f || top_v > v_ref + 8.f;
          if (__any_sync(0xffffffffu, moved)) {
            float fac = 1.f;
            if (moved) {
              // (2^-120: the smallest scale of an append; below it, or at 0, the weights lose range, not v_up)
              const float m_new = fmaxf(m_ref, top), v_new = fmaxf(fmaxf(v_ref, top_v), m_new - 120.f), keep = ex2_approx(m_ref - m_new);
              fac = ex2_approx(v_ref - v_new);
              l2[0].x *= keep; l2[0].y *= keep; l2[1].x *= keep; l2[1].y *= keep;
              m_ref = m_new;
              v_ref = v_new;
              v_up = ex2_approx(m_new - v_new + 6.f);
            }
            if (i > 0) {
              // O, behind W V of the step before (whose end the barrier of the lower scores implies)
              if (upper) {
                if (ok) ok = mbar_wait_flag(bar(L::kPvDone + tile), (i - 1) & 1, s_abort);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after_sync();
              }
#pragma unroll 1
              for (int c = 0; c < kD / 16; ++c) {
                float o[16];
                dec::tmem_ld16(tm_o + 16 * c, reinterpret_cast<uint32_t*>(o));
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] *= fac;
                dec::tmem_st16(tm_o + 16 * c, reinterpret_cast<const uint32_t*>(o));
              }
              tc_wait_st();                // (the lower half may read them again)
            }
            if (!upper && fac != 1.f) {
              // the weights of the upper half were made under the old reference
              const __half2 f2 = __float2half2_rn(fac);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&wu[j]), f2);
                wu[j] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
          }
          const float ref = m_ref == -INFINITY ? 0.f : -m_ref;
          const float2 ref2 = make_float2(ref, ref);
          const float4 vs4 = *reinterpret_cast<const float4*>(sc + 8 + (upper ? 4 : 0));
          // (finite: a key whose score lies 2^100 lower has a weight of 0, whatever its scale)
          const float vs[4] = {min_nan(vs4.x * v_up, 3e38f), min_nan(vs4.y * v_up, 3e38f), min_nan(vs4.z * v_up, 3e38f), min_nan(vs4.w * v_up, 3e38f)};
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float2 xx = make_float2(x[2 * j], x[2 * j + 1]);
            const float2 y = kCap ? __fadd2_rn(xx, ref2) : __ffma2_rn(xx, make_float2(kf[j >> 3], kf[j >> 3]), ref2);
            const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            l2[j & 1] = __fadd2_rn(l2[j & 1], e);
            const float2 wv = __fmul2_rn(e, make_float2(vs[j >> 3], vs[j >> 3]));
            pw[j] = pack_f16x2(wv.x, wv.y);
          }
        };
        {
          if (ok) ok = mbar_wait_flag(bar(L::kUFull + tile), i & 1, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after_sync();
          float x[64];
          const uint32_t from = i == 0 ? tm_s + 64 : tm_half;
          tmem_ld32(from, reinterpret_cast<uint32_t*>(x));
          tmem_ld32(from + 32, reinterpret_cast<uint32_t*>(x + 32));
          tc_wait_ld();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::kUFree + tile));
          weights(x, true, wu);
        }
        {
          if (ok) ok = mbar_wait_flag(bar(L::kLFull + tile), i & 1, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after_sync();
          float x[64];
          uint32_t wl[32];
          tmem_ld32(tm_half, reinterpret_cast<uint32_t*>(x));
          tmem_ld32(tm_half + 32, reinterpret_cast<uint32_t*>(x + 32));
          tc_wait_ld();
          weights(x, false, wl);
          tmem_st32(tm_half, wu);
          tmem_st32(tm_half + 32, wl);
          tc_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::kPFull + tile));
        }
      }
      // ---- the row's result
      if (n > 0) {
        if (ok) ok = mbar_wait_flag(bar(L::kODone), 0, s_abort);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after_sync();
      }
      const float l = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
      const int64_t l_idx = ((int64_t)b * p.Hq + h) * p.Sq + q0 + s;
      const bool none = m_ref == -INFINITY && l == 0.f;
      const RowEnd end = finish_row(m_ref, l, p.sink, h);
      const bool direct = p.num_splits == 1;
      const int64_t rows = (int64_t)p.B * p.Sq * p.Hq, part = (int64_t)split * rows;
      // (2^(v_ref - m_ref - 6) in two steps: it may be as small as 2^-126 beside a large O)
      const float down = m_ref == -INFINITY ? 0.f : ex2_approx(0.5f * (v_ref - m_ref - 6.f)), scale = (direct ? end.factor : rcp_approx(l)) * down;
      if (ok && row < R) {
        if (direct && p.lse != nullptr) p.lse[l_idx] = end.lse;
        if (!direct) p.lse_partial[part + ((int64_t)b * p.Sq + q0 + s) * p.Hq + h] = none ? -INFINITY : m_ref + lg2_approx(l);
      }
      // Output rows go through the memory of the tile's Q (a warp's own 32 rows; every product is done), to be written by lanes side by side.
      uint8_t* stage = gbase + L::kOffQ + 2 * tile * L::kTile8 + (t & ~31) * (2 * kD);
      constexpr int kChunks = kD / 8;
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
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = o[j] * scale * down;
        if (direct) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(stage + lane * (2 * kD) + (((4 * c + j) ^ (lane & 7)) << 4)) =
                make_uint4(pack_bf16x2(o[8 * j], o[8 * j + 1]), pack_bf16x2(o[8 * j + 2], o[8 * j + 3]), pack_bf16x2(o[8 * j + 4], o[8 * j + 5]),
                           pack_bf16x2(o[8 * j + 6], o[8 * j + 7]));
        } else if (ok && row < R && !none) {
          float4* dst = reinterpret_cast<float4*>(p.o_partial + (part + ((int64_t)b * p.Sq + q0 + s) * p.Hq + h) * kD + 32 * c);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
      }
      if (direct && ok) {
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < kChunks; ++i) {
          const int rr = i * (32 / kChunks) + lane / kChunks, c = lane % kChunks, at = r_first + (row & ~31) + rr;
          const int ss = fast_div(at, p.div_group), hh = hk * p.group + at - ss * p.group;
          if ((row & ~31) + rr < R)
            *reinterpret_cast<uint4*>(p.out + b * p.o_b + (int64_t)(q0 + ss) * p.o_s + hh * p.o_h + 8 * c) =
                *reinterpret_cast<const uint4*>(stage + rr * (2 * kD) + ((c ^ (rr & 7)) << 4));
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
