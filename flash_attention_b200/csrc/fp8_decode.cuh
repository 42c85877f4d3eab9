// Attention over the 8-bit KV cache for a handful of query rows (up to 32 rows of all query heads of a kv head).
//
// The bytes go from HBM to the tensor core as they are: keys and values are the A operands of kind::f8f6f4 products,
// transposed (keys, then head dims on the 128 lanes, query rows on the N side), and nothing is converted.
//
//   S^T (128 keys x N) = K (128 x D e4m3, K-major as loaded) . Q^T,     O^T (D x N) = V^T (MN-major as loaded) . P^T
//
// A bf16 query has eight significant bits and an e4m3 value four, so a query row is TWO e4m3 rows: q = q1 + q2 / 16 with q1 =
// e4m3(q 2^c) and q2 = 16 (q 2^c - q1), which is exact for elements down to 2^-13 of the row's largest (2^c brings that to 128..256;
// smaller ones are off by 2^-20 of it).  Their scores are two columns of one product; S = S1 + S2 / 16.  The weights go the same
// way: w = (w1 + w2 / 16) / 256, within 2^-9 of w down to 2^-14 and 2^-22 below that.  w is softmax weight times value scale, over
// the largest of these that the row has in the TILE, not among all keys so far (a row whose first key outweighs the rest by 2^15 would
// round the rest to nothing): the product of a tile is read out of tensor memory and added to the row's sums in fp32 registers,
// 2 FMAs per row and thread.
//
// One CTA = (split, kv head, sequence): a contiguous share of the sequence's 128-key tiles.  Warps: softmax warpgroups first
// (strand w takes every kStrands-th tile; with more than 16 rows two warpgroups share a tile's rows), then the loaders of K
// and V, the issuers of the two products.  Every wait is bounded.  A warp whose wait ran out goes through the rest of its loop
// without waiting, so that the rendezvous of a warpgroup (bar.sync) always has all its threads.
#pragma once
#include "fp8_attn.cuh"
#include "attn_decode.cuh"   // the transpose of lane groups, tensor-memory loads of few columns

namespace fa4 {
namespace fp8d {

enum Site { kKFullS = 130, kKFreeS, kVFullS, kVFreeS, kSFullS, kSFreeS, kPFullS, kPvDoneS, kQReadyS };

// Byte offset of 16-byte piece `ch` of row `row` in a tile of 128-byte rows (128-byte swizzle) / 64-byte rows.
__device__ __forceinline__ uint32_t sw128_offset(uint32_t row, uint32_t ch) {
  return (row >> 3) * 1024u + (row & 7u) * 128u + ((ch ^ (row & 7u)) << 4);
}
template <int kD>
__device__ __forceinline__ uint32_t row_piece(uint32_t row, uint32_t ch) {
  return kD == 128 ? sw128_offset(row, ch) : sw64_offset(row, ch);
}
// Operand tiles of kD-byte rows, groups of eight rows one behind the other: K-major (rows are M or N, the contraction
// within a row) and MN-major (rows are the contraction) read the same memory.  With 64-byte rows a second chunk of the M side
// would lie LBO further; it is 0, so lanes 64-127 repeat lanes 0-63.
template <int kD>
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
  return make_smem_desc(saddr, 0, 8 * kD, kD == 128 ? kSwizzle128 : kSwizzle64);
}
// Instruction descriptor of kind::f8f6f4, e4m3 x e4m3, fp32 accumulator: [4,6) D format 1, [7,10) A and [10,13) B format 0,
// [15] A and [16] B MN-major, [17,23) N >> 3, [24,29) M >> 4.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(uint32_t m, uint32_t n, bool a_mn_major) {
  return (1u << 4) | (a_mn_major ? 1u << 15 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

// kRW: rows of a warpgroup; kHalves: warpgroups that share a tile's rows; kStages: K and V tiles in flight; kCtas: of an SM.
template <int kD_, int kRW_, int kHalves_, int kStrands_, int kStages_, int kCtas_>
struct Form {
  static constexpr int kD = kD_, kRW = kRW_, kHalves = kHalves_, kStrands = kStrands_, kStages = kStages_, kCtas = kCtas_;
  static constexpr int kR = kRW * kHalves, kN = 2 * kR, kGroups = kHalves * kStrands, kThreads = 128 * kGroups + 128;
  static constexpr uint32_t kTile = 128 * kD;
  // Scales of K and V come with K.  Its stage is free when the product is done, which is before the softmax has read them:
  // the tiles that a strand may still read (one each) keep theirs.
  static constexpr int kScales = kStages + kStrands;
  static constexpr uint32_t kOffK = 0, kOffV = kOffK + kStages * kTile, kOffQ = kOffV + kStages * kTile,
                            kOffP = kOffQ + (kN * kD + 1023) / 1024 * 1024,   // kStrands x (N rows x 128 keys)
      kOffSc = kOffP + kStrands * kN * 128,                                  // scales of 16 keys: 8 of K, 8 of V a tile
      kOffRed = kOffSc + kScales * 64,                                        // maxima: groups x 2 x 4 warps x rows
      kOffFac = kOffRed + kGroups * 2 * 4 * kRW * 8,                         // (keep, add): groups x 2 x rows
      kOffRow = kOffFac + kGroups * 2 * kRW * 8,                             // factor of a row's scores
      kOffSum = kOffRow + kR * 4,                                            // groups x 4 warps x rows: sums
      kOffRef = kOffSum + kGroups * 4 * kRW * 4,                             // groups x rows: last references
      kOffBar = (kOffRef + kGroups * kRW * 4 + 7) / 8 * 8;
  static constexpr uint32_t kKFull = 0, kKFree = kKFull + kStages, kVFull = kKFree + kStages, kVFree = kVFull + kStages,
                            kSFull = kVFree + kStages, kSFree = kSFull + kStrands, kPFull = kSFree + kStrands,
                            kPvDone = kPFull + kStrands, kQReady = kPvDone + kStrands, kDrain = kQReady + 1, kBars = kDrain + 2;
  static constexpr uint32_t kOffMisc = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr uint32_t kRequest = kOffMisc + 16 + sizeof(WaitCtx) + 1024;
  static_assert(kCtas * (kRequest + 1024) <= 228 * 1024, "shared memory of the decode kernel");
  static constexpr uint32_t kS = 0, kO = kStrands * kN, kUsed = 2 * kStrands * kN;
  static constexpr uint32_t kCols = kUsed <= 32 ? 32 : kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kCtas * kCols <= 512, "tensor memory of the decode kernel");
  // the strands' sums meet in the memory of the K ring
  static_assert(kR * kD * 4 * kStrands <= 2 * (int)kStages * (int)kTile, "merge of the strands");
};

}  // namespace fp8d

template <class F>
__global__ void __launch_bounds__(F::kThreads, F::kCtas)
fp8_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ Fp8Params p) {
  using namespace fp8d;
  using dec::tmem_ld_cols;
  constexpr int kD = F::kD, kRW = F::kRW, kR = F::kR, kN = F::kN, kStages = F::kStages, kStrands = F::kStrands, kHalves = F::kHalves,
                kGroups = F::kGroups;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](uint32_t idx) -> uint32_t { return base + F::kOffBar + 8u * idx; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + F::kOffMisc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gbase + F::kOffMisc + 4);
  WaitCtx& wc = *reinterpret_cast<WaitCtx*>(gbase + F::kOffMisc + 16);
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  const int split = blockIdx.x, hk = fast_div(blockIdx.y, p.div_row_tiles), b = blockIdx.z, r_first = (blockIdx.y - hk * p.row_tiles) * F::kR;
  constexpr int kLoadK = 4 * kGroups, kLoadV = kLoadK + 1, kIssueS = kLoadK + 2, kIssueO = kLoadK + 3;

  if (tid == 0) {
    *s_abort = 0u;
    wc = WaitCtx{s_abort, p.status, p.budget_ns, p.epoch};
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(F::kKFull + s), 2);    // the copies' bytes, and the scales
      mbar_init(bar(F::kVFull + s), 1);
      mbar_init(bar(F::kKFree + s), 1);
      mbar_init(bar(F::kVFree + s), 1);
    }
    for (int s = 0; s < kStrands; ++s) {
      mbar_init(bar(F::kSFull + s), 1);
      mbar_init(bar(F::kSFree + s), 4 * kHalves);
      mbar_init(bar(F::kPFull + s), 4 * kHalves);
      mbar_init(bar(F::kPvDone + s), 1);
    }
    mbar_init(bar(F::kQReady), 4 * kGroups);
    mbar_init(bar(F::kDrain), 1);
    mbar_init(bar(F::kDrain + 1), 1);
    fence_barrier_init();
  }
  if (warp == kLoadK && lane == 0) tma_prefetch_desc(&tm_k);
  if (warp == kLoadV && lane == 0) tma_prefetch_desc(&tm_v);
  if (warp == kIssueS) {
    tmem_alloc(base + F::kOffMisc, F::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  pdl_wait();
  const SeqLens len = lens_of(p, b);
  // the keys that some row sees, as tiles; this CTA's share of them
  const int R = max(0, min(F::kR, len.sq * p.group - r_first));      // live rows: row r = s * group + head in the group
  const int lo_all = seen_by(p, len.sk, len.sq, fast_div(r_first, p.div_group)).x,
            hi_all = R > 0 ? seen_by(p, len.sk, len.sq, fast_div(r_first + R - 1, p.div_group)).y : 0;
  const int t_first = lo_all >> 7, t_total = hi_all > lo_all ? ((hi_all + 127) >> 7) - t_first : 0;
  const int per = (t_total + p.num_splits - 1) / p.num_splits;
  const int t0 = t_first + min(split * per, t_total), n = min(t_first + t_total - t0, per);
  __syncthreads();
  tc_fence_after_sync();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == kLoadK || warp == kLoadV) {
    // ============================================ loaders ======================================
    // Lane g (and g + 8) looks up keys 16 g .. 16 g + 15 of a tile: their page two tiles ahead and, in the loader of K, the scale of their
    // keys (of their values) one tile ahead.  The lanes in front of a box issue its copy.  Boxes that no row sees are not
    // loaded, their entries of the table not read.
    const bool is_k = warp == kLoadK;
    const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
    const float* scales = lane < 8 ? p.k_scale : p.v_scale;
    const uint32_t full0 = is_k ? F::kKFull : F::kVFull, free0 = is_k ? F::kKFree : F::kVFree;
    const uint32_t tile0 = base + (is_k ? F::kOffK : F::kOffV);
    float* s_scale = reinterpret_cast<float*>(gbase + F::kOffSc);
    auto key_of = [&](int li) { return ((t0 + li) << 7) + 16 * (lane & 7); };
    auto live = [&](int li) { return lane < 16 && li < n && key_of(li) < hi_all && key_of(li) + 16 > lo_all; };
    // (page, first key of these 16 in it)
    auto look_up = [&](int li) -> int2 {
      int2 at = make_int2(-1, 0);
      if (live(li)) {
        const int key = key_of(li), pg = fast_div(key, p.div_page);
        at = make_int2(p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b, key - pg * p.page_size);
      }
      return at;
    };
    auto scale_at = [&](int2 at) -> float {
      return is_k && at.x >= 0 && at.x < p.num_pages
                 ? scales[((int64_t)at.x * (p.page_size >> p.log_block) + (at.y >> p.log_block)) * p.Hkv + hk] : 0.f;
    };
    int2 at = look_up(0), at1 = look_up(1);
    float sc = scale_at(at);
    int li = 0;
    for (; li < n; ++li) {
      const uint32_t st = li % kStages;
      const int2 at2 = look_up(li + 2);
      const float sc1 = scale_at(at1);
      if (li >= kStages && ok) ok = mbar_wait(bar(free0 + st), (li / kStages - 1) & 1, wc, is_k ? kKFreeS : kVFreeS);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // a box is loaded if any of its keys is seen
      const uint32_t seen = __ballot_sync(0xffffffffu, live(li)) & 0xffu;
      const int per_box = p.box >> 4;
      const bool mine = lane < 8 && (lane & (per_box - 1)) == 0 && ((seen >> lane) & ((1u << per_box) - 1u)) != 0u;
      const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_arrive_expect_tx(bar(full0 + st), boxes * (uint32_t)p.box * kD);
      __syncwarp();
      // (the keys in front of those that are seen have no page here: that of the box is the first one looked up)
      const uint32_t in_box = (seen >> lane) & ((1u << per_box) - 1u);
      const int src = mine ? lane + __ffs(in_box) - 1 : lane;
      const int page = __shfl_sync(0xffffffffu, at.x, src & 31), off = __shfl_sync(0xffffffffu, at.y, src & 31) - 16 * (src - lane);
      if (mine) {
        const bool fine = page >= 0 && page < p.num_pages;
        if (!fine) report_bad_index(p.status, p.epoch, kPageSite);
        tma_load_4d(tile0 + st * F::kTile + 16 * lane * kD, tm, bar(full0 + st), 0, hk, off, fine ? page : p.num_pages);
      }
      if (is_k) {
        // (those of V as logarithms: -inf where nothing is seen or the scale is 0)
        if (lane < 16) s_scale[li % F::kScales * 16 + lane] = lane < 8 ? sc : lg2_approx(sc);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(full0 + st));
      }
      at = at1; at1 = at2; sc = sc1;
    }
    if (!ok && lane == 0) {
      // bounded drain: let the copies on their way land before the CTA's memory is released
      const uint64_t begun = globaltimer_ns();
      for (int i = li > kStages ? li - kStages : 0; i < li; ++i)
        while (!mbar_try_wait(bar(full0 + i % kStages), (i / kStages) & 1) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
    }
  } else if (warp == kIssueS) {
    // ============================================ K . Q^T ======================================
    if (elect_one() && n > 0) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, kN, false);
      ok = mbar_wait(bar(F::kQReady), 0, wc, kQReadyS);
      for (int li = 0; ok && li < n; ++li) {
        const uint32_t st = li % kStages, sd = li % kStrands;
        ok = mbar_wait(bar(F::kKFull + st), (li / kStages) & 1, wc, kKFullS);
        if (ok && li >= kStrands) ok = mbar_wait(bar(F::kSFree + sd), (li / kStrands - 1) & 1, wc, kSFreeS);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int ks = 0; ks < kD / 32; ++ks)
          mma_e4m3(tmem + F::kS + sd * kN, tile_desc<kD>(base + F::kOffK + st * F::kTile + 32 * ks),
                   tile_desc<kD>(base + F::kOffQ + 32 * ks), idesc, ks > 0);
        tc_commit(bar(F::kKFree + st));
        tc_commit(bar(F::kSFull + sd));
      }
      if (!ok) {
        const uint64_t begun = globaltimer_ns();
        tc_commit(bar(F::kDrain));
        while (!mbar_try_wait(bar(F::kDrain), 0) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
      }
    }
  } else if (warp == kIssueO) {
    // ============================================ V^T . P^T ====================================
    constexpr uint32_t idesc = make_idesc_e4m3(128, kN, true);
    for (int li = 0; li < n; ++li) {
      const uint32_t st = li % kStages, sd = li % kStrands;
      const int key0 = (t0 + li) << 7;
      const bool lead = elect_one();
      if (lead) ok = mbar_wait(bar(F::kVFull + st), (li / kStages) & 1, wc, kVFullS);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (key0 < lo_all || key0 + 128 > hi_all) {
        // values that no row sees may be anything, and 0 * NaN is NaN
        __syncwarp();
        for (int r = lane; r < 128; r += 32)
          if (key0 + r < lo_all || key0 + r >= hi_all) {
            uint4* v = reinterpret_cast<uint4*>(gbase + F::kOffV + st * F::kTile + r * kD);
#pragma unroll
            for (int i = 0; i < kD / 16; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lead) {
        ok = mbar_wait(bar(F::kPFull + sd), (li / kStrands) & 1, wc, kPFullS);
        if (ok) {
          tc_fence_after_sync();
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma_e4m3(tmem + F::kO + sd * kN, tile_desc<kD>(base + F::kOffV + st * F::kTile + 32 * ks * kD),
                     tile_desc<128>(base + F::kOffP + sd * kN * 128 + 32 * ks), idesc, ks > 0);
          tc_commit(bar(F::kVFree + st));
          tc_commit(bar(F::kPvDone + sd));
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    if (!ok && elect_one()) {
      const uint64_t begun = globaltimer_ns();
      tc_commit(bar(F::kDrain + 1));
      while (!mbar_try_wait(bar(F::kDrain + 1), 0) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
    }
  } else {
    // ============================================ softmax ======================================
    const int wg = warp >> 2, wq = warp & 3, sd = wg / kHalves, half = wg % kHalves, t = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    float2* s_red = reinterpret_cast<float2*>(gbase + F::kOffRed) + wg * 2 * 4 * kRW;
    float2* s_fac = reinterpret_cast<float2*>(gbase + F::kOffFac) + wg * 2 * kRW;
    float* s_row = reinterpret_cast<float*>(gbase + F::kOffRow);

    // ---- Q^T: a row's pieces of eight elements by neighbouring lanes
    {
      constexpr int kPieces = kD / 8;
      for (int i = tid; i < kR * kPieces; i += 128 * kGroups) {
        const int r = i / kPieces, ch = i % kPieces;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (r < R) {
          const int s = fast_div(r_first + r, p.div_group), h = hk * p.group + r_first + r - s * p.group;
          u = *reinterpret_cast<const uint4*>(p.q + b * p.q_b + s * p.q_s + h * p.q_h + 8 * ch);
        }
        float x[8];
        unpack8(u, x);
        uint32_t top = 0u;                      // (bit patterns: NaN is the largest)
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < kPieces; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^c with largest * 2^c in [128, 256); a row that is not finite becomes NaN whole
        const int e = max((int)(top >> 23), 17);
        const float up = __uint_as_float((uint32_t)(254 + 7 - e) << 23), down = __uint_as_float((uint32_t)(e - 7) << 23);
        uint32_t w[4];
        if (top >= 0x7f800000u) {
          w[0] = w[1] = w[2] = w[3] = 0x7f7f7f7fu;
        } else {
          float y[8], rest[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= up;
          w[0] = pack4_e4m3(x[0], x[1], x[2], x[3]);
          w[1] = pack4_e4m3(x[4], x[5], x[6], x[7]);
          unpack4_e4m3(w[0], y);
          unpack4_e4m3(w[1], y + 4);
#pragma unroll
          for (int k = 0; k < 8; ++k) rest[k] = (x[k] - y[k]) * 16.f;
          w[2] = pack4_e4m3(rest[0], rest[1], rest[2], rest[3]);
          w[3] = pack4_e4m3(rest[4], rest[5], rest[6], rest[7]);
        }
        *reinterpret_cast<uint2*>(gbase + F::kOffQ + row_piece<kD>(r, ch >> 1) + (ch & 1) * 8) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(gbase + F::kOffQ + row_piece<kD>(kR + r, ch >> 1) + (ch & 1) * 8) = make_uint2(w[2], w[3]);
        if (ch == 0) s_row[r] = (p.cap_out != 0.f ? p.cap_in : p.sl2) * down;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(F::kQReady));
      // (the factors of the rows are read by all warps: they have met where all have arrived)
      ok = __all_sync(0xffffffffu, mbar_wait(bar(F::kQReady), 0, wc, kQReadyS));
    }
    // After the transpose below a thread has one row, and the kRW keys of its lane group.
    const int my = lane & (kRW - 1), row = half * kRW + my, grp = lane / kRW, key_in = wq * 32 + grp * kRW;
    int lo = 0, hi = 0;
    if (row < R) {
      const int2 see = seen_by(p, len.sk, len.sq, fast_div(r_first + row, p.div_group));
      lo = see.x;
      hi = see.y;
    }
    const float factor = s_row[row];
    float m_run = -INFINITY, l = 0.f, acc[kRW];
#pragma unroll
    for (int r = 0; r < kRW; ++r) acc[r] = 0.f;
    // O^T of the strand's last tile, into the sums
    auto take = [&](int u) {
      if (ok) ok = mbar_wait(bar(F::kPvDone + sd), u & 1, wc, kPvDoneS);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after_sync();
      float o1[kRW], o2[kRW];
      tmem_ld_cols<kRW>(tmem + lanes + F::kO + sd * kN + half * kRW, reinterpret_cast<uint32_t*>(o1));
      tmem_ld_cols<kRW>(tmem + lanes + F::kO + sd * kN + kR + half * kRW, reinterpret_cast<uint32_t*>(o2));
      tc_wait_ld();
      tc_fence_before_sync();
      const float2* fac = s_fac + (u & 1) * kRW;
#pragma unroll
      for (int r = 0; r < kRW; ++r) acc[r] = fmaf(acc[r], fac[r].x, fmaf(o2[r], 0.0625f, o1[r]) * fac[r].y);
    };
    int u = 0;
    for (int li = sd; li < n; li += kStrands, ++u) {
      // (only barriers of this strand are waited for: a stage's barrier may be two phases behind, and a wait on parities
      // does not tell that from done)
      const int key0 = (t0 + li) << 7;
      if (ok) ok = mbar_wait(bar(F::kSFull + sd), u & 1, wc, kSFullS);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after_sync();
      float x[kRW], lv;
      {
        float x2[kRW];
        tmem_ld_cols<kRW>(tmem + lanes + F::kS + sd * kN + half * kRW, reinterpret_cast<uint32_t*>(x));
        tmem_ld_cols<kRW>(tmem + lanes + F::kS + sd * kN + kR + half * kRW, reinterpret_cast<uint32_t*>(x2));
        tc_wait_ld();
        tc_fence_before_sync();
        // (the scales were there before the product: one barrier for both)
        const float* sc = reinterpret_cast<const float*>(gbase + F::kOffSc) + li % F::kScales * 16;
        const float ks = sc[t >> 4];
        lv = sc[8 + (key_in >> 4)];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(F::kSFree + sd));
#pragma unroll
        for (int r = 0; r < kRW; ++r) x[r] = fmaf(x2[r], 0.0625f, x[r]) * ks;
      }
      dec::lane_group_transpose<kRW>(x, lane);
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kRW; ++j) {
        const int key = key0 + key_in + j;
        x[j] = key >= lo && key < hi ? score_of(p, x[j], factor) : -INFINITY;
        top = fmaxf(top, x[j]);
      }
      float top_v = top + lv;              // of the weights with the values' scales
#pragma unroll
      for (int o = kRW; o < 32; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
      }
      float2* red = s_red + (u & 1) * 4 * kRW;
      if (lane < kRW) red[wq * kRW + lane] = make_float2(top, top_v);
      group_sync(1 + wg);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 of = red[k * kRW + my];
        top = fmaxf(top, of.x);
        top_v = fmaxf(top_v, of.y);
      }
      const float ref = top == -INFINITY ? 0.f : top, up = lv - (top_v == -INFINITY ? 0.f : top_v) + 8.f;
      const float m_new = fmaxf(m_run, top), keep = m_new == -INFINITY ? 0.f : ex2_approx(m_run - m_new),
                  add = m_new == -INFINITY ? 0.f : ex2_approx(top - m_new),
                  add_v = m_new == -INFINITY ? 0.f : ex2_approx(top_v - m_new);
      float w[kRW], sum = 0.f;
#pragma unroll
      for (int j = 0; j < kRW; ++j) {
        sum += ex2_approx(x[j] - ref);
        w[j] = ex2_approx(x[j] + up);
      }
      l = fmaf(l, keep, sum * add);
      m_run = m_new;
      // the sums of the tile before, and with them its P^T, are done with
      if (u > 0) take(u - 1);
      if (wq == 0 && lane < kRW) s_fac[(u & 1) * kRW + lane] = make_float2(keep, add_v * (1.f / 256.f));
      {
        uint8_t* pt = gbase + F::kOffP + sd * kN * 128;
        uint32_t w1[kRW / 4], w2[kRW / 4];
#pragma unroll
        for (int j = 0; j < kRW / 4; ++j) {
          float y[4];
          w1[j] = pack4_e4m3(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          unpack4_e4m3(w1[j], y);
          w2[j] = pack4_e4m3((w[4 * j] - y[0]) * 16.f, (w[4 * j + 1] - y[1]) * 16.f, (w[4 * j + 2] - y[2]) * 16.f,
                             (w[4 * j + 3] - y[3]) * 16.f);
        }
        uint8_t *a1 = pt + sw128_offset(row, key_in >> 4) + (key_in & 15), *a2 = pt + sw128_offset(kR + row, key_in >> 4) + (key_in & 15);
        if constexpr (kRW == 8) {
          *reinterpret_cast<uint2*>(a1) = make_uint2(w1[0], w1[1]);
          *reinterpret_cast<uint2*>(a2) = make_uint2(w2[0], w2[1]);
        } else {
          *reinterpret_cast<uint4*>(a1) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
          *reinterpret_cast<uint4*>(a2) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(F::kPFull + sd));
    }
    if (u > 0) {
      // (the factors of the last tile, written before its rendezvous... by one warp: meet once more)
      group_sync(1 + wg);
      take(u - 1);
    }
    // ---- the row's sum over its lanes and warps, then the strands
#pragma unroll
    for (int o = kRW; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float* s_sum = reinterpret_cast<float*>(gbase + F::kOffSum);
    float* s_ref = reinterpret_cast<float*>(gbase + F::kOffRef);
    if (lane < kRW) s_sum[(wg * 4 + wq) * kRW + lane] = l;
    if (wq == 0 && lane < kRW) s_ref[wg * kRW + lane] = m_run;
    auto all_groups = [] { asm volatile("bar.sync 15, %0;" ::"n"(128 * kGroups) : "memory"); };
    all_groups();                                                    // (every tile is done with: the rings are free)
    float* s_acc = reinterpret_cast<float*>(gbase + F::kOffK);       // strands x rows x kD
    if (t < kD) {
#pragma unroll
      for (int r = 0; r < kRW; ++r) s_acc[(sd * kR + half * kRW + r) * kD + t] = acc[r];
    }
    all_groups();
    // a warp a row, four elements a lane
    const bool whole = *s_abort == 0u;
#pragma unroll 1
    for (int r = warp; r < R && whole; r += 4 * kGroups) {
      const int hf = r / kRW, rw = r % kRW, col = 4 * lane;
      float m = -INFINITY, sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kStrands; ++k) m = fmaxf(m, s_ref[(k * kHalves + hf) * kRW + rw]);
#pragma unroll
      for (int k = 0; k < kStrands; ++k) {
        const int g = k * kHalves + hf;
        const float f = m == -INFINITY ? 1.f : ex2_approx(s_ref[g * kRW + rw] - m);
        const float* s4 = s_sum + g * 4 * kRW + rw;
        sum = fmaf(f, ((s4[0] + s4[kRW]) + s4[2 * kRW]) + s4[3 * kRW], sum);
        if (col < kD) {
          const float4 a = *reinterpret_cast<const float4*>(s_acc + (k * kR + r) * kD + col);
          o.x = fmaf(f, a.x, o.x); o.y = fmaf(f, a.y, o.y); o.z = fmaf(f, a.z, o.z); o.w = fmaf(f, a.w, o.w);
        }
      }
      const int s = fast_div(r_first + r, p.div_group), h = hk * p.group + r_first + r - s * p.group;
      const int64_t l_idx = ((int64_t)b * p.Hq + h) * p.Sq + s;
      if (p.num_splits == 1) {
        const RowEnd e = finish_row(m, sum, p.sink, h);
        if (col < kD)
          *reinterpret_cast<uint2*>(p.out + b * p.o_b + s * p.o_s + h * p.o_h + col) =
              make_uint2(pack_bf16x2(o.x * e.factor, o.y * e.factor), pack_bf16x2(o.z * e.factor, o.w * e.factor));
        if (lane == 0 && p.lse != nullptr) p.lse[l_idx] = e.lse;
      } else {
        const int64_t rows = (int64_t)p.B * p.Sq * p.Hq, part = (int64_t)split * rows;
        const bool none = m == -INFINITY && sum == 0.f;
        const float f = 1.f / sum;
        if (col < kD && !none)
          *reinterpret_cast<float4*>(p.o_partial + (part + ((int64_t)b * p.Sq + s) * p.Hq + h) * kD + col) =
              make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
        if (lane == 0) p.lse_partial[part + l_idx] = none ? -INFINITY : m + log2f(sum);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kIssueS) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, F::kCols);
  }
}

}  // namespace fa4
