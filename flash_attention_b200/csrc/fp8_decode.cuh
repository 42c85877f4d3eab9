// Attention over the 8-bit KV cache for a handful of query rows (up to 32 rows of all query heads of a kv head).
//
// The bytes go from HBM to the tensor core as they are: both products are kind::f8f6f4 and nothing of the cache is converted.
//
//   S (rows x 128 keys) = Q . K^T (K-major as loaded),     O^T (D x rows) = V^T (MN-major as loaded) . W^T
//
// A bf16 query has eight significant bits and an e4m3 value four, so a query row is two e4m3 rows, one behind the other along the
// contraction: q 2^c = q1 + q2 with q1 = e4m3(q 2^c), which is exact for elements down to 2^-10 of the row's largest (2^c brings that to
// 256 at most; smaller ones are off by 2^-18 of it).  The rows stand on the lanes of the A operand as often as they fit, so each of the four
// warps of a tile finds all of them in its lanes, and a thread has one row and 16 neighbouring keys (32 with more than 16 rows):
// nothing is transposed, and maxima take a shuffle and one exchange through shared memory.
//
// Weights are two e4m3 rows as well, w = (w1 + w2 / 16) / 256, as neighbouring columns of one product: within 2^-9 of w down to 2^-14 and
// 2^-22 below that.  w is softmax weight times value scale, over the largest of these that the row has in the TILE, not among all
// keys so far (a row whose first key outweighs the rest by 2^15 would round the rest to nothing): the product of a tile is read out of
// tensor memory and added to the row's sums in fp32 registers, two FMAs a row and thread, under a reference of all tiles so far.  The sum
// of the weights without the scales has one of its own.
//
// A CTA per SM works through its share of all tiles of the call: the lengths are on the device, and shares of equal size are what keeps HBM
// busy to the end.  Up to eight kv heads go side by side through the same tokens, a CTA each: theirs lie next to each other in memory
// (every head at its own place in the list: 4 x 65536 keys of 8 heads at 3.9 TB/s, HBM pages and translations missed).  A unit (sequence, kv head) that ends up in several CTAs is
// merged by fp8_merge_kernel.  With a split count of the caller's a CTA has one split of one unit.
//
// What bounds it (calls back to back): HBM in its steady part, 4 x 65536 keys of 8 heads 92 us (88 the kernel: 6.1 TB/s, 94 % of a measured copy; 82 at that
// rate; 112 in turn with other work).  Short calls pay
// about 14 us in front and behind: dealing 1.3, a chain of table, scales and copies, the products of the first and the last tile, the merge of
// pieces 3 to 4; 32 sequences of up to 8192 keys 55 us (38), 8 of five rows over up to 4099 keys with pages of 16 22 us (6).  A unit alone (one token over 777
// keys: eight CTAs of seven tiles) takes 9.6 us.
//
// Warps: kStrands softmax warpgroups, to which the tiles are dealt in turn, then the loaders of K and V and the issuers of the two products.  The
// loaders run ahead through the pieces of a CTA.  Every wait is bounded.  A warp whose wait ran out goes through the rest of its loops
// without waiting, so that the rendezvous of a warpgroup (bar.sync) always has all its threads.
#pragma once
#include "fp8_attn.cuh"
#include "attn_decode.cuh"   // tensor-memory loads of few columns

namespace fa4 {
namespace fp8d {

// Smallest share of a CTA, in tiles.
constexpr int kMinShare = 2;

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
// The same descriptor `bytes` further on.
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(desc));
  lo += bytes >> 4;
  asm("mov.b64 %0, {%1, %2};" : "=l"(desc) : "r"(lo), "r"(hi));
  return desc;
}
// A place in a ring of kN barriers and the parity of its present phase, without divisions.
template <int kN>
struct Ring {
  uint32_t at = 0, parity = 0;
  __device__ __forceinline__ void next() {
    if (++at == kN) {
      at = 0;
      parity ^= 1u;
    }
  }
};
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

// A warp that loads the tiles of keys or of values, as far ahead as its ring of kStages places allows.
//
// Four tiles at a time: lane 8 q + g looks up keys 16 g .. 16 g + 15 of the q-th, their page two batches ahead and, in the loader of
// K, the scales of their keys and values one batch ahead (a tile at a time, a CTA ran at a tile per memory latency).  What the copies need goes
// through shared memory to one thread, which issues them (with all lanes in that loop a tile took 900 clocks).  Boxes that no row
// sees are not loaded, their entries of the table not read.  The scales are written in front of the copies: the barrier of K's tile is
// theirs too.
struct FeederSites {
  uint32_t free, lands;      // where a wait may run out
};
// kLogs: behind the scales the logarithms of the values', to base 2.
template <int kD, int kStages, int kScales, bool kLogs = false>
struct Feeder {
  static constexpr uint32_t kTile = 128 * kD;
  static constexpr int kWords = kLogs ? 24 : 16;
  const CUtensorMap* tm;
  uint32_t full0, free0, part;      // barriers: of the ring's places; of a tile of values that are not all seen (0: such tiles are no matter)
  uint32_t tiles;                   // shared memory of the ring
  uint8_t* ring;                    //   the same, for plain stores
  float* scales;                    // kScales x (8 of K, 8 of V, logarithms of those), or null
  int2* box;                        // 32 places
  FeederSites site;
  Ring<kStages> st;                 // (of the issuing thread)
  bool first = true;                // round of the ring
  int issued = 0;                   // tiles so far (of the issuing thread)
  int slot = 0;                     // place of the next tile among the scales
  uint32_t parts = 0u;
  bool part_on_way = false;         // a tile that lands on `part` (of the issuing thread)

  // Tiles t0 .. t0 + n - 1 of kv head hk of sequence b, in which keys [lo, hi) are seen.  False: a wait ran out.
  __device__ __forceinline__ bool piece(const Fp8Params& p, const WaitCtx& wc, int n, int t0, int b, int hk, int lo, int hi) {
    const int lane = threadIdx.x & 31, per_box = p.box >> 4, gr = lane & 7;
    bool ok = true;
    // (page, first key of these 16 in it) for the batch from tile `li` on; key -1: no row sees them
    auto look_up = [&](int li) -> int2 {
      int2 at = make_int2(0, -1);
      const int mine = li + (lane >> 3), key = ((t0 + mine) << 7) + 16 * gr;
      if (mine < n && key < hi && key + 16 > lo) {
        const int pg = fast_div(key, p.div_page);
        at = make_int2(p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b, key - pg * p.page_size);
      }
      return at;
    };
    auto scales_at = [&](int2 at) -> float2 {
      if (scales == nullptr || at.y < 0 || at.x < 0 || at.x >= p.num_pages) return make_float2(0.f, 0.f);
      const int64_t i = ((int64_t)at.x * (p.page_size >> p.log_block) + (at.y >> p.log_block)) * p.Hkv + hk;
      return make_float2(p.k_scale[i], p.v_scale[i]);
    };
    int2 at = look_up(0), at1 = look_up(4);
    float2 sc = scales_at(at);
#pragma unroll 1
    for (int l0 = 0; l0 < n; l0 += 4) {
      // a box is loaded if any of its keys is seen; the keys in front of those have no page here: that of the box is the first one looked up
      const uint32_t seen = __ballot_sync(0xffffffffu, at.y >= 0);
      const uint32_t in_box = (seen >> lane) & ((1u << per_box) - 1u);
      const bool heads = (gr & (per_box - 1)) == 0 && in_box != 0u;
      const uint32_t boxes = __ballot_sync(0xffffffffu, heads);
      const int src = heads ? lane + __ffs(in_box) - 1 : lane;
      int page = __shfl_sync(0xffffffffu, at.x, src & 31);
      const int off = __shfl_sync(0xffffffffu, at.y, src & 31) - 16 * (src - lane);
      if (heads) {
        if (page < 0 || page >= p.num_pages) {
          report_bad_index(p.status, p.epoch, kPageSite);
          page = p.num_pages;                       // (reads as zeros)
        }
        box[lane] = make_int2(page, off);
      }
      const int end = min(4, n - l0);
      if (scales != nullptr && (lane >> 3) < end) {
        // (the scales of the batch, as far ahead of the softmax as the ring of them allows)
        int to = slot + (lane >> 3);
        to = (to >= kScales ? to - kScales : to) * kWords + gr;
        scales[to] = sc.x;
        scales[to + 8] = sc.y;
        if constexpr (kLogs) scales[to + 16] = lg2_approx(sc.y);
      }
      const int2 at2 = look_up(l0 + 8);
      const float2 sc1 = scales_at(at1);
      __syncwarp();
      // A tile of values that are not all seen (the first and the last of a unit may be) goes through a barrier of its own: the others may be
      // anything, and 0 * NaN is NaN, so they are made zeros before the tile is given on.
      auto in_part = [&](int q) { const int key0 = (t0 + l0 + q) << 7; return part != 0u && (key0 < lo || key0 + 128 > hi); };
      for (int q0 = 0; q0 < end && ok;) {
        int q1 = q0;
        while (q1 < end && !in_part(q1)) ++q1;
        const bool is_part = q1 < end;
        uint32_t last = 0u;                       // the last one's place
        const bool lead = elect_one();            // (the same lane each time)
        if (lead) {
#pragma unroll 1
          for (int q = q0; q < q1 + is_part; ++q) {
            const uint32_t lands = q < q1 ? full0 + 8 * st.at : part;
            if (!first) ok = mbar_wait_relaxed<256>(free0 + 8 * st.at, st.parity ^ 1u, wc, site.free);
            if (!ok) break;
            last = st.at;
            const uint32_t mine = (boxes >> (8 * q)) & 0xffu;
            mbar_arrive_expect_tx(lands, __popc(mine) * (uint32_t)p.box * kD);
            part_on_way = q == q1;
            ++issued;
            for (uint32_t m = mine; m != 0u; m &= m - 1u) {
              const int i = __ffs(m) - 1;
              const int2 from = box[8 * q + i];
              tma_load_4d(tiles + last * kTile + 16 * i * kD, tm, lands, 0, from.y, hk, from.x);
            }
            st.next();
            if (st.at == 0) first = false;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (is_part && ok) {
          ok = __all_sync(0xffffffffu, mbar_wait(part, parts, wc, site.lands));
          if (!ok) return false;
          part_on_way = false;
          parts ^= 1u;
          last = __shfl_sync(0xffffffffu, last, __ffs(__ballot_sync(0xffffffffu, lead)) - 1);
          const int key0 = (t0 + l0 + q1) << 7;
          for (int r = lane; r < 128; r += 32)
            if (key0 + r < lo || key0 + r >= hi) {
              uint4* v = reinterpret_cast<uint4*>(ring + last * kTile + r * kD);
#pragma unroll
              for (int i = 0; i < kD / 16; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
            }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full0 + 8 * last);
        }
        q0 = q1 + is_part;
      }
      if (!ok) return false;
      slot += end;
      if (slot >= kScales) slot -= kScales;
      at = at1; at1 = at2; sc = sc1;
    }
    return true;
  }
  // Before the CTA's memory is released: let the copies on their way land, within limits.  (Not only after a wait of this warp that ran
  // out: where another one's did, nobody else may have waited for the last tiles.)
  __device__ __forceinline__ void drain() const {
    if (!elect_one()) return;
    const uint64_t begun = globaltimer_ns();
    auto landed = [&](uint32_t bar, uint32_t parity) {
      while (!mbar_try_wait(bar, parity) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
    };
    if (part_on_way) landed(part, parts);
    for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i) landed(full0 + 8 * (i % kStages), (i / kStages) & 1);
  }
};

// kR: rows (16 or 32).
template <int kD_, int kR_, bool kCap_>
struct Form {
  static constexpr int kD = kD_, kR = kR_, kStrands = kR == 16 ? 3 : 2, kStages = kD == 128 ? 5 : 10, kThreads = 128 * kStrands + 128;
  static constexpr bool kCap = kCap_;
  static constexpr int kN = 2 * kR, kKeys = kR;       // keys of a thread: 128 lanes hold 128 / kR copies of the rows
  static constexpr uint32_t kTile = 128 * kD;
  // Scales of K and V come with K.  Its stage is free when the product is done, which is before the softmax has read them:
  // the tiles that a strand may still read (one each) keep theirs, beside a batch that is written at once.
  static constexpr int kScales = kStages + kStrands + 4;
  static constexpr uint32_t kOffK = 0, kOffV = kOffK + kStages * kTile, kOffQ = kOffV + kStages * kTile,   // q1, q2: 128 x kD
      kOffP = kOffQ + 2 * kTile,                                             // kStrands x (kN rows x 128 keys)
      kOffSc = kOffP + kStrands * kN * 128,                                  // scales of 16 keys: 8 of K, 8 of V a tile
      kOffBox = (kOffSc + kScales * 64 + 15) / 16 * 16,                                        // what the copies of a batch need: 2 x 32 (page, key in it)
      kOffRed = kOffBox + 512,                                       // maxima: strands x 2 x 4 warps x rows
      kOffFac = kOffRed + kStrands * 2 * 4 * kR * 8,                         // (keep, add): strands x 2 x rows
      kOffRow = kOffFac + kStrands * 2 * kR * 8,                             // factor of a row's scores
      kOffSum = kOffRow + kR * 4,                                            // strands x 4 warps x rows: sums
      kOffRef = (kOffSum + kStrands * 4 * kR * 4 + 7) / 8 * 8,                             // strands x rows: last references
      kOffBar = kOffRef + kStrands * kR * 8;
  static constexpr uint32_t kKFull = 0, kKFree = kKFull + kStages, kVFull = kKFree + kStages, kVFree = kVFull + kStages,
                            kSFull = kVFree + kStages, kSFree = kSFull + kStrands, kPFull = kSFree + kStrands,
                            kPvDone = kPFull + kStrands, kQReady = kPvDone + kStrands, kVPart = kQReady + 1, kDrain = kVPart + 1, kBars = kDrain + 2;
  static constexpr uint32_t kOffMisc = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr uint32_t kOffDeal = (kOffMisc + 16 + sizeof(WaitCtx) + 15) / 16 * 16;
  static constexpr uint32_t kRequest = kOffDeal + 64 + 1024;
  static_assert(kRequest <= 227 * 1024, "shared memory of the decode kernel");
  static constexpr uint32_t kS = 0, kO = kStrands * 128;
  static_assert(kO + kStrands * kN <= 512, "tensor memory of the decode kernel");
  // the strands' sums meet in the memory of Q
  static_assert(kR * kD * 4 * kStrands <= 2 * (int)kTile, "merge of the strands");
};

// A sequence as the kernel sees it: keys, query rows; the keys that some row sees, as tiles of 128.
struct Seq {
  int sk, sq, lo, hi, first, tiles;
};
__device__ __forceinline__ Seq seq_of(const Fp8Params& p, int sk, int sq) {
  Seq q;
  q.sk = sk;
  q.sq = sq;
  q.lo = seen_by(p, sk, sq, 0).x;
  q.hi = sq > 0 ? seen_by(p, sk, sq, sq - 1).y : 0;
  q.first = q.lo >> 7;
  q.tiles = q.hi > q.lo ? ((q.hi + 127) >> 7) - q.first : 0;
  return q;
}
// A unit's place in the list of all tiles: one that sees nothing takes a place too (its zeros are to be written), one without rows none.
__device__ __forceinline__ int cost_of(const Seq& q) { return q.sq == 0 ? 0 : max(q.tiles, 1); }

// The CTA's walk through its pieces: `bundle` heads of a sequence are worked on side by side by as many CTAs, so units of the walk are
// (sequence, bundle).  One warp finds the start and leaves it in shared memory; every warp walks on by itself, with the lengths of the next
// sequence on their way while a piece is worked on.
struct alignas(16) Walk {
  Seq cur;
  int b, hb, at, left;       // unit, first place of the piece in it, places of this CTA from there on
  int share;                 // places of a CTA
  int next_sk, next_sq;

  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ int places() const { return min(left, cost_of(cur) - at); }
  __device__ __forceinline__ int tiles() const { return min(places(), cur.tiles - at); }
  __device__ __forceinline__ void fetch(const Fp8Params& p) {
    if (left <= cost_of(cur) - at) return;                     // (the last piece)
    const SeqLens n = b + 1 < p.B ? lens_of(p, b + 1) : SeqLens{0, 0};
    next_sk = n.sk;
    next_sq = n.sq;
  }
  __device__ __forceinline__ void next(const Fp8Params& p) {
    left -= places();
    if (left <= 0) return;
    at = 0;
    if (++hb == p.bundles) {
      hb = 0;
      do {
        if (++b >= p.B) {
          left = 0;
          return;
        }
        cur = seq_of(p, next_sk, next_sq);
        fetch(p);
      } while (cost_of(cur) == 0);
    }
  }
};

// Where group `group` of CTAs (of as many as p.div_groups divides by) starts, by one warp.
__device__ __forceinline__ Walk deal_shares(const Fp8Params& p, int group, int lane) {
  Walk w = {};
  w.b = p.B;
  auto read = [&](int b0) {
    const SeqLens n = b0 + lane < p.B ? lens_of(p, b0 + lane) : SeqLens{0, 0};
    return seq_of(p, n.sk, n.sq);
  };
  const Seq first = read(0);
  int total = cost_of(first);
#pragma unroll 1
  for (int b0 = 32; b0 < p.B; b0 += 32) total += cost_of(read(b0));
  total = __reduce_add_sync(0xffffffffu, total) * p.bundles;
  const int groups = gridDim.x / p.bundle;
  w.share = max(fast_div(total + groups - 1, p.div_groups), kMinShare);
  const int from = group * w.share;
  if (from >= total) return w;
  int before = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const Seq q = b0 == 0 ? first : read(b0);
    int upto = cost_of(q) * p.bundles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    upto += before;
    const uint32_t hit = __ballot_sync(0xffffffffu, from < upto);
    if (hit != 0u) {
      const int l = __ffs(hit) - 1;
      w.b = b0 + l;
      w.cur = seq_of(p, __shfl_sync(0xffffffffu, q.sk, l), __shfl_sync(0xffffffffu, q.sq, l));
      const int c = cost_of(w.cur), into = from - (__shfl_sync(0xffffffffu, upto, l) - c * p.bundles);
      w.hb = p.bundles > 1 ? into / c : 0;
      w.at = into - w.hb * c;
      w.left = w.share;
      return w;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return w;
}

}  // namespace fp8d

template <class F>
__global__ void __launch_bounds__(F::kThreads, 1)
fp8_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ Fp8Params p) {
  using namespace fp8d;
  using dec::tmem_ld_cols;
  constexpr int kD = F::kD, kR = F::kR, kN = F::kN, kStages = F::kStages, kStrands = F::kStrands, kKeys = F::kKeys;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](uint32_t idx) -> uint32_t { return base + F::kOffBar + 8u * idx; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + F::kOffMisc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gbase + F::kOffMisc + 4);
  WaitCtx& wc = *reinterpret_cast<WaitCtx*>(gbase + F::kOffMisc + 16);
  Walk& s_walk = *reinterpret_cast<Walk*>(gbase + F::kOffDeal);
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  constexpr int kLoadK = 4 * kStrands, kLoadV = kLoadK + 1, kIssueS = kLoadK + 2, kIssueO = kLoadK + 3;

  if (tid == 0) {
    *s_abort = 0u;
    wc = WaitCtx{s_abort, p.status, p.budget_ns, p.epoch};
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(F::kKFull + s), 1);    // (the scales are written in front of the copies)
      mbar_init(bar(F::kVFull + s), 1);
      mbar_init(bar(F::kKFree + s), 1);
      mbar_init(bar(F::kVFree + s), 1);
    }
    for (int s = 0; s < kStrands; ++s) {
      mbar_init(bar(F::kSFull + s), 1);
      mbar_init(bar(F::kSFree + s), 4);
      mbar_init(bar(F::kPFull + s), 4);
      mbar_init(bar(F::kPvDone + s), 1);
    }
    mbar_init(bar(F::kQReady), 4 * kStrands);
    mbar_init(bar(F::kVPart), 1);
    mbar_init(bar(F::kDrain), 1);
    mbar_init(bar(F::kDrain + 1), 1);
    fence_barrier_init();
  }
  if (warp == kLoadK && lane == 0) tma_prefetch_desc(&tm_k);
  if (warp == kLoadV && lane == 0) tma_prefetch_desc(&tm_v);
  if (warp == kIssueS) {
    tmem_alloc(base + F::kOffMisc, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  pdl_wait();
  // CTA = group * bundle + head in the bundle; with a split count of the caller's, a group is one split of one unit
  const int group = blockIdx.x / p.bundle, in_bundle = blockIdx.x - group * p.bundle;
  if (warp == 0) {
    Walk w = {};
    if (p.num_splits > 0) {
      const int unit = group / p.num_splits, split = group - unit * p.num_splits;
      w.b = unit / p.bundles;
      w.hb = unit - w.b * p.bundles;
      const SeqLens len = lens_of(p, w.b);
      w.cur = seq_of(p, len.sk, len.sq);
      const int places = cost_of(w.cur);
      w.share = p.num_splits == 1 ? places : (places + p.num_splits - 1) / p.num_splits;
      w.at = split * w.share;
      w.left = max(0, min(w.share, places - w.at));
    } else {
      w = deal_shares(p, group, lane);
    }
    if (lane == 0) s_walk = w;
  }
  __syncthreads();
  tc_fence_after_sync();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  Walk walk = s_walk;
  walk.fetch(p);

  if (warp == kLoadK || warp == kLoadV) {
    // ============================================ loaders ======================================
    const bool is_k = warp == kLoadK;
    Feeder<kD, kStages, F::kScales> feed;
    feed.tm = is_k ? &tm_k : &tm_v;
    feed.full0 = bar(is_k ? F::kKFull : F::kVFull);
    feed.free0 = bar(is_k ? F::kKFree : F::kVFree);
    feed.part = is_k ? 0u : bar(F::kVPart);
    feed.tiles = base + (is_k ? F::kOffK : F::kOffV);
    feed.ring = gbase + (is_k ? F::kOffK : F::kOffV);
    feed.scales = is_k ? reinterpret_cast<float*>(gbase + F::kOffSc) : nullptr;
    feed.box = reinterpret_cast<int2*>(gbase + F::kOffBox) + (is_k ? 0 : 32);
    feed.site = is_k ? FeederSites{kKFreeS, kKFullS} : FeederSites{kVFreeS, kVFullS};
    for (; ok && walk.more(); walk.next(p))
      ok = feed.piece(p, wc, walk.tiles(), walk.cur.first + walk.at, walk.b, walk.hb * p.bundle + in_bundle, walk.cur.lo, walk.cur.hi);
    feed.drain();
  } else if (warp == kIssueS) {
    // ============================================ Q . K^T ======================================
    // (An issuing thread gets an instruction every eight clocks or so, its code never stays in the scheduler's cache beside the softmax
    // warps'.  With divisions for the ring places, descriptors made anew and votes in the loop the issuer of V^T W^T took 2000
    // clocks a tile and paced the kernel: 4 x 65536 keys 139 us.)
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, 128, false);
      const uint64_t dq = tile_desc<kD>(base + F::kOffQ), dk = tile_desc<kD>(base + F::kOffK);
      Ring<kStages> st;
      Ring<kStrands> sd;
      bool first = true;                    // round of the strands
      // (pieces without a tile have no Q: a phase of the barrier for each that has some)
      uint32_t piece = 0;
      for (; ok && walk.more(); walk.next(p)) {
        const int n = walk.tiles();
        if (n > 0) {
          ok = mbar_wait(bar(F::kQReady), piece, wc, kQReadyS);
          piece ^= 1u;
        }
#pragma unroll 1
        for (int li = 0; ok && li < n; ++li) {
          ok = mbar_wait(bar(F::kKFull + st.at), st.parity, wc, kKFullS);
          if (ok && !first) ok = mbar_wait(bar(F::kSFree + sd.at), sd.parity ^ 1u, wc, kSFreeS);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t kt = desc_at(dk, st.at * F::kTile);
          const uint32_t to = tmem + F::kS + 128 * sd.at;
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks)
            mma_e4m3(to, desc_at(dq, ks / (kD / 32) * F::kTile + 32 * (ks % (kD / 32))), desc_at(kt, 32 * (ks % (kD / 32))), idesc, ks > 0);
          tc_commit(bar(F::kKFree + st.at));
          tc_commit(bar(F::kSFull + sd.at));
          st.next();
          sd.next();
          if (sd.at == 0) first = false;
        }
      }
      // (every product is awaited before the CTA's memory is released, also where it was another role's wait that ran out)
      const uint64_t begun = globaltimer_ns();
      tc_commit(bar(F::kDrain));
      while (!mbar_try_wait(bar(F::kDrain), 0) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
    }
  } else if (warp == kIssueO) {
    // ============================================ V^T . W^T ====================================
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, kN, true);
      const uint64_t dv = tile_desc<kD>(base + F::kOffV), dw = tile_desc<128>(base + F::kOffP);
      Ring<kStages> st;
      Ring<kStrands> sd;
      for (; ok && walk.more(); walk.next(p)) {
        const int n = walk.tiles();
#pragma unroll 1
        for (int li = 0; li < n; ++li) {
          ok = mbar_wait(bar(F::kVFull + st.at), st.parity, wc, kVFullS) && mbar_wait(bar(F::kPFull + sd.at), sd.parity, wc, kPFullS);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t vt = desc_at(dv, st.at * F::kTile), wt = desc_at(dw, sd.at * kN * 128);
          const uint32_t to = tmem + F::kO + sd.at * kN;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) mma_e4m3(to, desc_at(vt, 32 * ks * kD), desc_at(wt, 32 * ks), idesc, ks > 0);
          tc_commit(bar(F::kVFree + st.at));
          tc_commit(bar(F::kPvDone + sd.at));
          st.next();
          sd.next();
        }
      }
      // (every product is awaited before the CTA's memory is released, also where it was another role's wait that ran out)
      const uint64_t begun = globaltimer_ns();
      tc_commit(bar(F::kDrain + 1));
      while (!mbar_try_wait(bar(F::kDrain + 1), 0) && globaltimer_ns() - begun < 50ull * 1000 * 1000) {}
    }
  } else {
    // ============================================ softmax ======================================
    const int sd = warp >> 2, wq = warp & 3, t = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    float2* s_red = reinterpret_cast<float2*>(gbase + F::kOffRed) + sd * 2 * 4 * kR;
    float2* s_fac = reinterpret_cast<float2*>(gbase + F::kOffFac) + sd * 2 * kR;
    float* s_row = reinterpret_cast<float*>(gbase + F::kOffRow);
    float* s_sum = reinterpret_cast<float*>(gbase + F::kOffSum);
    float2* s_ref = reinterpret_cast<float2*>(gbase + F::kOffRef);
    float* s_acc = reinterpret_cast<float*>(gbase + F::kOffQ);       // strands x rows x kD
    auto all_strands = [] { asm volatile("bar.sync 15, %0;" ::"n"(128 * kStrands) : "memory"); };
    const int my = lane & (kR - 1), grp = lane / kR, key_in = wq * 32 + grp * kKeys;
    int g = 0;
    bool again = false;
    for (int piece = 0; walk.more(); walk.next(p)) {
      if (again) all_strands();                                        // (the sums of the last piece are read: Q may be written)
      again = true;
      const Seq seq = walk.cur;
      const int n = walk.tiles(), t0 = seq.first + walk.at, b = walk.b, hk = walk.hb * p.bundle + in_bundle, R = seq.sq * p.group;
      // ---- Q: a row's pieces of eight elements by neighbouring lanes, to all copies of the row
      if (n > 0) {
        constexpr int kPieces = kD / 8;
        for (int i = tid; i < kR * kPieces; i += 128 * kStrands) {
          const int r = i / kPieces, ch = i % kPieces;
          uint4 u = make_uint4(0u, 0u, 0u, 0u);
          if (r < R) {
            const int s = fast_div(r, p.div_group), h = hk * p.group + r - s * p.group;
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
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] *= up;
            w[0] = pack4_e4m3(x[0], x[1], x[2], x[3]);
            w[1] = pack4_e4m3(x[4], x[5], x[6], x[7]);
            unpack4_e4m3(w[0], y);
            unpack4_e4m3(w[1], y + 4);
            w[2] = pack4_e4m3(x[0] - y[0], x[1] - y[1], x[2] - y[2], x[3] - y[3]);
            w[3] = pack4_e4m3(x[4] - y[4], x[5] - y[5], x[6] - y[6], x[7] - y[7]);
          }
#pragma unroll
          for (int k = 0; k < 128 / kR; ++k) {
            uint8_t* to = gbase + F::kOffQ + row_piece<kD>(k * kR + r, ch >> 1) + (ch & 1) * 8;
            *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2*>(to + F::kTile) = make_uint2(w[2], w[3]);
          }
          if (ch == 0) s_row[r] = (F::kCap ? p.cap_in : p.sl2) * down;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(F::kQReady));
        // (the factors of the rows are read by all warps: they have met where all have arrived)
        if (ok) ok = mbar_wait(bar(F::kQReady), piece++ & 1, wc, kQReadyS);
        ok = __all_sync(0xffffffffu, ok);
      }
      int lo = 0, hi = 0;
      if (my < R) {
        const int2 see = seen_by(p, seq.sk, seq.sq, fast_div(my, p.div_group));
        lo = see.x;
        hi = see.y;
      }
      // the keys that all rows see
      const int lo_in = seq.sq > 0 ? seen_by(p, seq.sk, seq.sq, seq.sq - 1).x : 0, hi_in = seen_by(p, seq.sk, seq.sq, 0).y;
      const float factor = s_row[my];
      float m_run = -INFINITY, v_run = -INFINITY, l = 0.f, acc[kR];    // largest score, and with its value scale
#pragma unroll
      for (int r = 0; r < kR; ++r) acc[r] = 0.f;
      // O^T of the strand's tile before, into the sums
      auto take = [&](int u) {
        if (ok) ok = mbar_wait(bar(F::kPvDone + sd), u & 1, wc, kPvDoneS);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after_sync();
        float o1[kR], o2[kR];
        tmem_ld_cols<kR>(tmem + lanes + F::kO + sd * kN, reinterpret_cast<uint32_t*>(o1));
        tmem_ld_cols<kR>(tmem + lanes + F::kO + sd * kN + kR, reinterpret_cast<uint32_t*>(o2));
        tc_wait_ld();
        tc_fence_before_sync();
        const float4* fac = reinterpret_cast<const float4*>(s_fac + (u & 1) * kR);
#pragma unroll
        for (int r = 0; r < kR; r += 2) {
          const float4 f = fac[r / 2];
          acc[r] = fmaf(acc[r], f.x, fmaf(o2[r], 0.0625f, o1[r]) * f.y);
          acc[r + 1] = fmaf(acc[r + 1], f.z, fmaf(o2[r + 1], 0.0625f, o1[r + 1]) * f.w);
        }
      };
      // this strand's tiles: those with running number sd, sd + kStrands, ... of the CTA
      // (and one round more, for the last tile's product)
      const int g0 = g, li0 = (sd + kStrands - g0 % kStrands) % kStrands, u0 = (g0 + li0) / kStrands;
#pragma unroll 1
      for (int li = li0, u = u0; li < n + kStrands; li += kStrands, ++u) {
        const bool live = li < n;
        const int key0 = (t0 + li) << 7;
        float x[kKeys], up[kKeys / 16], keep_v = 0.f, add_v = 0.f;
        if (live) {
        // (only barriers of this strand are waited for: a stage's barrier may be two phases behind, and a wait on parities
        // does not tell that from done)
        if (ok) ok = mbar_wait(bar(F::kSFull + sd), u & 1, wc, kSFullS);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after_sync();
        float ks[kKeys / 16], lv[kKeys / 16];
        {
          float y[32];
          tmem_ld32(tmem + lanes + F::kS + 128 * sd + 32 * wq, reinterpret_cast<uint32_t*>(y));
          tc_wait_ld();
          tc_fence_before_sync();
          // (the scales were there before the product: one barrier for both)
          const float* sc = reinterpret_cast<const float*>(gbase + F::kOffSc) + (g0 + li) % F::kScales * 16;
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i) {
            ks[i] = sc[(key_in >> 4) + i] * factor;
            lv[i] = lg2_approx(sc[8 + (key_in >> 4) + i]);       // (-inf where nothing is seen or the scale is 0)
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(F::kSFree + sd));
#pragma unroll
          for (int j = 0; j < kKeys; ++j) {
            x[j] = (kR == 16 && grp != 0 ? y[(16 + j) & 31] : y[j]) * ks[j / 16];
            if constexpr (F::kCap) x[j] = p.cap_out * tanh_of(x[j]);
          }
        }
        if (key0 < lo_in || key0 + 128 > hi_in) {
#pragma unroll
          for (int j = 0; j < kKeys; ++j) {
            const int key = key0 + key_in + j;
            x[j] = key >= lo && key < hi ? x[j] : -INFINITY;
          }
        }
        float top = -INFINITY, top_v = -INFINITY;     // of the scores; of the weights with the values' scales
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
          float m = fmaxf(x[16 * i], x[16 * i + 1]);
#pragma unroll
          for (int j = 2; j < 16; j += 2) m = fmax3(m, x[16 * i + j], x[16 * i + j + 1]);
          top = fmaxf(top, m);
          top_v = fmaxf(top_v, m + lv[i]);
        }
#pragma unroll
        for (int o = kR; o < 32; o <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
        }
        float2* red = s_red + (u & 1) * 4 * kR;
        if (lane < kR) red[wq * kR + lane] = make_float2(top, top_v);
        group_sync(1 + sd);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 of = red[k * kR + my];
          top = fmaxf(top, of.x);
          top_v = fmaxf(top_v, of.y);
        }
        const float ref = top == -INFINITY ? 0.f : top, ref_v = top_v == -INFINITY ? 0.f : top_v;
        const float m_new = fmaxf(m_run, top), base_m = m_new == -INFINITY ? 0.f : m_new, add = ex2_approx(top - base_m), keep = ex2_approx(m_run - base_m);
        // (the values' sums have a reference of their own: scales may be as far from 1 as fp32 reaches)
        const float v_new = fmaxf(v_run, top_v), base_v = v_new == -INFINITY ? 0.f : v_new;
        keep_v = ex2_approx(v_run - base_v);
        add_v = ex2_approx(top_v - base_v);
        v_run = v_new;
        // a weight times this is 256 at most (bounded for scales further apart than fp32 reaches)
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
          const float e = lv[i] + (ref - ref_v) + 8.f;
          up[i] = ex2_approx(e > 100.f ? 100.f : e);
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
          x[j] = ex2_approx(x[j] - ref);
          sum += x[j];
          x[j] *= up[j / 16];
        }
        l = fmaf(l, keep, sum * add);
        m_run = m_new;
        } else {
          if (u == u0) break;
          group_sync(1 + sd);         // (the factors of the last tile are written by one warp)
        }
        // the sums of the tile before, and with them its W^T, are done with
        if (u > u0) take(u - 1);
        if (!live) break;
        if (wq == 0 && lane < kR) s_fac[(u & 1) * kR + lane] = make_float2(keep_v, add_v * (1.f / 256.f));
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
          uint32_t w1[4], w2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float* w = x + 16 * i + 4 * j;
            float y[4];
            w1[j] = pack4_e4m3(w[0], w[1], w[2], w[3]);
            unpack4_e4m3(w1[j], y);
            w2[j] = pack4_e4m3((w[0] - y[0]) * 16.f, (w[1] - y[1]) * 16.f, (w[2] - y[2]) * 16.f, (w[3] - y[3]) * 16.f);
          }
          uint8_t* pt = gbase + F::kOffP + sd * kN * 128;
          *reinterpret_cast<uint4*>(pt + sw128_offset(my, (key_in >> 4) + i)) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
          *reinterpret_cast<uint4*>(pt + sw128_offset(kR + my, (key_in >> 4) + i)) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(F::kPFull + sd));
      }
      g += n;
      // ---- the row's sum over its lanes and warps, then the strands
#pragma unroll
      for (int o = kR; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (lane < kR) s_sum[(sd * 4 + wq) * kR + lane] = l;
      if (wq == 0 && lane < kR) s_ref[sd * kR + lane] = make_float2(m_run, v_run);
      all_strands();                                                   // (every product of the piece is done: Q is free)
      if (t < kD) {
#pragma unroll
        for (int r = 0; r < kR; ++r) s_acc[(sd * kR + r) * kD + t] = acc[r];
      }
      all_strands();
      // where the result goes: the output if the whole unit was this piece, else a slot of partial results
      const int places = cost_of(seq), unit = b * p.Hkv + hk;
      bool direct;
      int64_t slot;
      if (p.num_splits > 0) {
        direct = p.num_splits == 1;
        slot = (int64_t)unit * p.num_splits + group % p.num_splits;
      } else {
        direct = walk.places() == places;
        slot = 2 * (int64_t)blockIdx.x + (walk.at == 0 ? 1 : 0);
        if (tid == 0 && walk.at == 0) {
          const int share = s_walk.share, rest = places - walk.places();
          p.pieces[unit] = make_int2(blockIdx.x, 1 + (rest + share - 1) / share);
        }
      }
      // a warp a row, four elements a lane
      const bool whole = *s_abort == 0u;
#pragma unroll 1
      for (int r = warp; r < R && whole; r += 4 * kStrands) {
        const int col = 4 * lane;
        float m = -INFINITY, v = -INFINITY, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kStrands; ++k) {
          const float2 of = s_ref[k * kR + r];
          m = fmaxf(m, of.x);
          v = fmaxf(v, of.y);
        }
#pragma unroll
        for (int k = 0; k < kStrands; ++k) {
          const float2 of = s_ref[k * kR + r];
          const float f = m == -INFINITY ? 1.f : ex2_approx(of.x - m), fv = v == -INFINITY ? 1.f : ex2_approx(of.y - v);
          const float* s4 = s_sum + k * 4 * kR + r;
          sum = fmaf(f, ((s4[0] + s4[kR]) + s4[2 * kR]) + s4[3 * kR], sum);
          if (col < kD) {
            const float4 a = *reinterpret_cast<const float4*>(s_acc + (k * kR + r) * kD + col);
            o.x = fmaf(fv, a.x, o.x); o.y = fmaf(fv, a.y, o.y); o.z = fmaf(fv, a.z, o.z); o.w = fmaf(fv, a.w, o.w);
          }
        }
        // (2^(v - m) in two steps: the values' sum may be as large as that is small)
        const float by = v == -INFINITY ? 0.f : ex2_approx(0.5f * (v - m));
        if (direct) {
          const int s = fast_div(r, p.div_group), h = hk * p.group + r - s * p.group;
          const RowEnd e = finish_row(m, sum, p.sink, h);
          const float f = e.factor * by;
          if (col < kD)
            *reinterpret_cast<uint2*>(p.out + b * p.o_b + s * p.o_s + h * p.o_h + col) =
                make_uint2(pack_bf16x2(o.x * f * by, o.y * f * by), pack_bf16x2(o.z * f * by, o.w * f * by));
          if (lane == 0 && p.lse != nullptr) p.lse[((int64_t)b * p.Hq + h) * p.Sq + s] = e.lse;
        } else {
          const bool none = m == -INFINITY && sum == 0.f;
          const float f = rcp_approx(sum) * by;
          if (col < kD && !none)
            *reinterpret_cast<float4*>(p.o_partial + (slot * p.unit_rows + r) * kD + col) = make_float4(o.x * f * by, o.y * f * by, o.z * f * by, o.w * f * by);
          if (lane == 0) p.lse_partial[slot * p.unit_rows + r] = none ? -INFINITY : m + lg2_approx(sum);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kIssueS) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// The units that several CTAs had a piece of: a warp a row.
__global__ void __launch_bounds__(kFp8CombineWarps * 32) fp8_merge_kernel(const __grid_constant__ Fp8Params p) {
  const int lane = threadIdx.x & 31;
  const uint32_t r = blockIdx.x * kFp8CombineWarps + (threadIdx.x >> 5), rows = (uint32_t)p.B * p.Sq * p.Hq;
  pdl_wait();
  if (r >= rows) return;
  const int bs = fast_div((int)r, p.div_hq), h = (int)r - bs * p.Hq, b = fast_div(bs, p.div_sq), s = bs - b * p.Sq;
  const int hk = fast_div(h, p.div_group), row = s * p.group + h - hk * p.group, unit = b * p.Hkv + hk;
  // (asked for together; a sequence without rows has no pieces noted)
  const int rows_here = p.fresh != nullptr ? p.fresh[b] : p.Sq;
  const int2 at = p.num_splits == 0 ? p.pieces[unit] : make_int2(0, 0);
  if (s >= rows_here) return;
  int64_t first, step;
  int pieces = p.num_splits;
  if (pieces > 0) {
    // (the splits that have a part of the unit)
    first = (int64_t)unit * pieces;
    step = 1;
    const SeqLens len = lens_of(p, b);
    const int places = fp8d::cost_of(fp8d::seq_of(p, len.sk, len.sq)), per = (places + pieces - 1) / pieces;
    pieces = (places + per - 1) / per;
  } else {
    pieces = at.y;
    first = 2 * (int64_t)at.x;          // (a CTA has two slots: of the unit it begins in the middle of, of the one it leaves there)
    step = 2 * p.bundle;
  }
  if (p.num_splits == 0 && pieces <= 1) return;
  merge_row(p, b, s, h, lane, pieces, [&](int i) { return (first + i * step + (i == 0 && p.num_splits == 0 ? 1 : 0)) * p.unit_rows + row; });
}

}  // namespace fa4
