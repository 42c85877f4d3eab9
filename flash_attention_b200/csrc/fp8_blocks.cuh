// Choosing blocks of the 8-bit KV cache: the index of a cache (bounds of the keys of every block), and the blocks that queries choose by it.
//
//   index    of a block and kv head, over the tokens that are there:  u = 2^(e - 6), e the exponent of the largest |byte value|,
//            hi = ceil(max / u), lo = floor(min / u) of every channel (whole numbers up to 120),  scale = k_scale u
//   query    of Q rows one behind the other and the heads of a kv head: positive and negative parts of q 2^(14 - e) as whole numbers, summed
//            over rows and heads, then shifted to seven bits: p and n
//   score    scale * (sum_d p_d hi_d - n_d lo_d): up to those roundings the sum, over rows and heads, of the largest q . k that the
//            bounds of the block allow
//
// Everything up to the last product is a whole number below 2^24, so a score has one rounding and no order of summation: any split of
// the work, and any other program, finds the same blocks, ties (equal scores) included.
#pragma once
#include "fp8_append.cuh"

namespace fa4 {

struct IndexParams {
  const uint8_t* k;
  int64_t k_page, k_tok, k_head;     // bytes
  const float* k_scale;
  int8_t* bounds;                    // (pages, blocks of a page, Hkv, 2, D)
  float* scale;                      // (pages, blocks of a page, Hkv)
  const int32_t *seqlens, *fresh, *table;
  int S, Hkv, log_block, num_pages, page_size, pages_per_seq;
  int blocks, units;                 // that S tokens may touch; B * blocks * Hkv
  FastDiv div_hkv, div_blocks, div_page;
  uint32_t* status;
  uint32_t epoch;
};

constexpr int kIndexWarps = 4;

// A warp a block and kv head: kD / 16 lanes a row of 16-byte pieces, maxima and minima as pairs of fp16 (every e4m3 value is one).  It waits for loads: 111700 tokens of 8 heads,
// blocks of 64 (118 MB read and written) 26.3 us, 4.5 TB/s at 31 warps an SM, issue slots 47 % busy; eight rows of a lane on their way rather than four 28 (80 registers), warps that go on to a next block 31.5.
template <int kD>
__global__ void __launch_bounds__(kIndexWarps * 32) fp8_index_kernel(const __grid_constant__ IndexParams p) {
  constexpr int kChunks = kD / 16, kRows = 32 / kChunks;
  const int unit = blockIdx.x * kIndexWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  if (unit >= p.units) return;
  const int rest = fast_div(unit, p.div_hkv), head = unit - rest * p.Hkv, b = fast_div(rest, p.div_blocks), blk = rest - b * p.blocks;
  const int held = p.seqlens[b];
  int n = p.fresh != nullptr ? p.fresh[b] : p.S;
  n = n < 0 ? 0 : (n < p.S ? n : p.S);
  if (n == 0) return;
  if (held < 0) {
    if (lane == 0) report_bad_index(p.status, p.epoch, kPositionSite);
    return;
  }
  const int bt = 1 << p.log_block;
  const int64_t start = (int64_t)((held >> p.log_block) + blk) << p.log_block, end = (int64_t)held + n;
  if (start >= end) return;
  if (start >= (int64_t)p.pages_per_seq * p.page_size) {
    if (lane == 0) report_bad_index(p.status, p.epoch, kPositionSite);
    return;
  }
  const int pg = fast_div((int)start, p.div_page), off = (int)start - pg * p.page_size;
  const int page = p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b;
  if (page < 0 || page >= p.num_pages) {
    if (lane == 0) report_bad_index(p.status, p.epoch, kPageSite);
    return;
  }
  const int there = end - start < bt ? (int)(end - start) : bt, row0 = lane / kChunks, c = lane % kChunks;
  const uint8_t* src = p.k + page * p.k_page + off * p.k_tok + head * p.k_head + 16 * c;
  const __half2 inf = __float2half2_rn(INFINITY);
  __half2 hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi[i] = __hneg2(inf);
    lo[i] = inf;
  }
#pragma unroll 1
  for (int r0 = row0; r0 < there; r0 += 4 * kRows) {
    uint4 u[4];                                  // (on their way together)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (r0 + q * kRows < there) u[q] = *reinterpret_cast<const uint4*>(src + (r0 + q * kRows) * p.k_tok);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (r0 + q * kRows >= there) break;
      const uint32_t w[4] = {u[q].x, u[q].y, u[q].z, u[q].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x[2];
        asm("{\n"
            ".reg .b16 l, h;\n"
            "mov.b32 {l, h}, %2;\n"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n"
            "cvt.rn.f16x2.e4m3x2 %1, h;\n"
            "}\n"
            : "=r"(x[0]), "=r"(x[1])
            : "r"(w[i]));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const __half2 v = *reinterpret_cast<const __half2*>(&x[k]);
          hi[2 * i + k] = __hmax2_nan(hi[2 * i + k], v);       // (NaN stays in the maximum)
          lo[2 * i + k] = __hmin2(lo[2 * i + k], v);
        }
      }
    }
  }
#pragma unroll
  for (int o = kChunks; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      hi[i] = __hmax2_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
      lo[i] = __hmin2(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
    }
  float top = 0.f, up[16], down[16];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 a = __half22float2(hi[i]), z = __half22float2(lo[i]);
    up[2 * i] = a.x; up[2 * i + 1] = a.y; down[2 * i] = z.x; down[2 * i + 1] = z.y;
    bad = bad || a.x != a.x || a.y != a.y;
    top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(z.x), fabsf(z.y)));
  }
#pragma unroll
  for (int o = 1; o < kChunks; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  bad = __any_sync(0xffffffffu, bad);
  const int e = top > 0.f ? (int)(__float_as_uint(top) >> 23) - 127 : -9;
  const float inv = __uint_as_float((uint32_t)(127 + 6 - e) << 23), step = __uint_as_float((uint32_t)(127 - 6 + e) << 23);
  const int64_t at = ((int64_t)page * (p.page_size >> p.log_block) + (off >> p.log_block)) * p.Hkv + head;
  if (row0 == 0) {
    uint32_t w[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[0][i] = w[1][i] = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[0][i] |= (uint32_t)(uint8_t)__float2int_ru(up[4 * i + k] * inv) << (8 * k);
        w[1][i] |= (uint32_t)(uint8_t)__float2int_rd(down[4 * i + k] * inv) << (8 * k);
      }
      if (bad) w[0][i] = w[1][i] = 0u;
    }
    int8_t* to = p.bounds + at * (2 * kD) + 16 * c;
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
    *reinterpret_cast<uint4*>(to + kD) = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
  }
  if (lane == 0) p.scale[at] = bad ? __uint_as_float(0x7fffffffu) : __fmul_rn(p.k_scale[at], step);
}

// ---- the choice -------------------------------------------------------------------------------------------------

struct SelectParams {
  const __nv_bfloat16* q;
  int64_t q_b, q_s, q_h;             // elements
  const int8_t* bounds;
  const float* scale;
  const int32_t *used, *fresh, *table;
  int32_t* blocks;                   // (B, query blocks, Hkv, chosen)
  int Sq, Hkv, group, log_block, num_pages, page_size, pages_per_seq, capacity;
  int chosen, query_block, query_blocks, front, recent;
  int parts;                         // CTAs of a unit
  FastDiv div_hkv, div_query_blocks, div_page, div_group;
  uint32_t* status;
  uint32_t epoch;
};

constexpr int kSelectThreads = 512;
constexpr int kSelectBlocks = 53248;           // of a sequence: their scores are 208 KB

// Order of scores as whole numbers: the larger the score the larger the key; NaN as +inf, -0 as 0.
__device__ __forceinline__ uint32_t score_key(float s) {
  s = s != s ? INFINITY : s + 0.f;
  const uint32_t u = __float_as_uint(s);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kAlways = 0xffffffffu;      // (no score has it)

__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t rank, uint32_t v) {
  asm volatile(
      "{\n"
      ".reg .b32 a;\n"
      "mapa.shared::cluster.u32 a, %0, %1;\n"
      "st.shared::cluster.u32 [a], %2;\n"
      "}\n" ::"r"(addr), "r"(rank), "r"(v)
      : "memory");
}

// A unit (sequence, query block, kv head) is one CTA's, or (kParts) that of a cluster whose CTAs score a part of the blocks each and leave the keys
// with the first one, which chooses.
//
// Four lanes have a block, pieces of 16 bytes apart by four, so a warp's load covers eight blocks and a dot product takes two shuffles (16 lanes a block took four times the
// instructions: 2048 rows over 1024 blocks 25.7 -> 20.8 us).  The first bounds are on their way while the query is summed.  What bounds it: scattered pieces of 256 bytes in its middle (32 sequences of
// up to 512 blocks, 21 MB, 10.7 us back to back and 16 on a cold L2), else a chain of lengths, table, bounds, three passes over the keys and the list: 128 blocks 5.4 us.  Four sequences of 4096 blocks
// with a CTA a unit 24, as clusters of four 13.8.
template <int kD, bool kParts>
__global__ void __launch_bounds__(kSelectThreads, 2) fp8_select_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kWarps = kSelectThreads / 32, kPieces = kD / 8, kBins = 2048;
  extern __shared__ uint32_t s_key[];          // of the CTA's blocks: where their bounds are; then the keys
  __shared__ int s_sum[2 * kD], s_red[kWarps], s_count[2 * kWarps];
  __shared__ __align__(16) int s_hist[kBins];
  __shared__ __align__(16) int8_t s_q[2 * kD];
  __shared__ uint32_t s_range[2 * 8];          // smallest and largest key of a CTA's blocks
  __shared__ int s_bin[3];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = kParts ? blockIdx.x / p.parts : blockIdx.x, part = kParts ? blockIdx.x - unit * p.parts : 0;
  const int rest = fast_div(unit, p.div_hkv), head = unit - rest * p.Hkv, b = fast_div(rest, p.div_query_blocks),
            q0 = (rest - b * p.query_blocks) * p.query_block;
  // (the attention's CTAs may take an SM as soon as this one's leave it, and set themselves up; with clusters that delayed those: 13.8 -> 15.2 us)
  if constexpr (!kParts) pdl_trigger();
  pdl_wait();
  int sk = p.used[b], sq = p.fresh != nullptr ? p.fresh[b] : p.Sq;
  sk = sk < 0 ? 0 : (sk < p.capacity ? sk : p.capacity);
  sq = sq < 0 ? 0 : (sq < p.Sq ? sq : p.Sq);
  const int rows = max(0, min(sq - q0, p.query_block)), first = sk - sq + q0, end = rows > 0 ? max(0, first + rows) : 0;
  const int bt = 1 << p.log_block, n = (end + bt - 1) >> p.log_block;
  int32_t* out = p.blocks + (int64_t)unit * p.chosen;
  if (n <= p.chosen) {
    if (part == 0)
      for (int i = tid; i < p.chosen; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int per = kParts ? ((n + p.parts - 1) / p.parts + 31) & ~31 : n, b0 = part * per, b1 = min(n, b0 + per);
  // ---- where the bounds are
  for (int j = b0 + tid; j < b1; j += kSelectThreads) {
    const int at = j << p.log_block, pg = fast_div(at, p.div_page), off = at - pg * p.page_size;
    const int page = p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b;
    const bool fine = page >= 0 && page < p.num_pages;
    if (!fine) report_bad_index(p.status, p.epoch, kPageSite);
    s_key[j] = fine ? (uint32_t)(page * (p.page_size >> p.log_block) + (off >> p.log_block)) : 0xffffffffu;
  }
  for (int i = tid; i < 2 * kD; i += kSelectThreads) s_sum[i] = 0;
  if (tid < 2) s_range[2 * part + tid] = tid == 0 ? 0xffffffffu : 0u;
  // ---- the query: largest element, sums of whole numbers, seven bits
  const __nv_bfloat16* q = p.q + b * p.q_b + (int64_t)q0 * p.q_s + (int64_t)head * p.group * p.q_h;
  const int pieces = rows * p.group * kPieces;
  auto piece_of = [&](int i) -> uint4 {
    const int r = i / kPieces, s = fast_div(r, p.div_group), h = r - s * p.group;
    return *reinterpret_cast<const uint4*>(q + (int64_t)s * p.q_s + h * p.q_h + 8 * (i % kPieces));
  };
  uint32_t top = 0u;
#pragma unroll 4
  for (int i = tid; i < pieces; i += kSelectThreads) {
    const uint4 u = piece_of(i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = w[k] << 16 & 0x7fff0000u, hi = w[k] & 0x7fff0000u;
      top = max(top, max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_red[warp] = (int)top;
  __syncthreads();
  // the first bounds, on their way meanwhile: four lanes a block, which hold every fourth piece of 16 bytes of it
  constexpr int kParcels = kD / 32, kDeep = 2, kRound = kWarps * 8;           // pieces of a lane; rounds on their way; blocks of a round
  const int sub = lane >> 2, c = lane & 3;
  uint4 v[kDeep][kParcels];
  float scale[kDeep];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int j = j0 + k * kRound + sub;
      const uint32_t at = j < b1 ? s_key[j] : 0xffffffffu;
      scale[k] = -INFINITY;                        // (a page outside the pool; no index has it)
      if (at != 0xffffffffu) {
        const int64_t i = (int64_t)at * p.Hkv + head;
        const uint4* from = reinterpret_cast<const uint4*>(p.bounds + i * (2 * kD)) + c;
        // (the whole of a block at once from HBM: both in turn on a cold L2 0.8 us of 50)
#pragma unroll
        for (int r = 0; r < kParcels; ++r)
          asm volatile("ld.global.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[k][r].x), "=r"(v[k][r].y), "=r"(v[k][r].z), "=r"(v[k][r].w) : "l"(from + 4 * r));
        scale[k] = p.scale[i];
      } else {
#pragma unroll
        for (int r = 0; r < kParcels; ++r) v[k][r] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  fetch(b0 + warp * 8);
  top = __reduce_max_sync(0xffffffffu, (uint32_t)s_red[lane & (kWarps - 1)]);
  const int e = max((int)(top >> 23) - 127, -100);
  const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
  if (warp * 32 < pieces) {
    int pos[8] = {}, neg[8] = {};                  // (a thread stays with its eight channels)
#pragma unroll 2
    for (int i = tid; i < pieces; i += kSelectThreads) {
      float x[8];
      unpack8(piece_of(i), x);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int y = fabsf(x[k]) < INFINITY ? __float2int_rn(x[k] * up) : 0;
        pos[k] += max(y, 0);
        neg[k] += max(-y, 0);
      }
    }
    const int ch = tid % kPieces * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
      for (int o = kPieces; o < 32; o <<= 1) {
        pos[k] += __shfl_xor_sync(0xffffffffu, pos[k], o);
        neg[k] += __shfl_xor_sync(0xffffffffu, neg[k], o);
      }
      if (lane < kPieces) {
        atomicAdd(&s_sum[ch + k], pos[k]);
        atomicAdd(&s_sum[kD + ch + k], neg[k]);
      }
    }
  }
  __syncthreads();
  {
    static_assert(2 * kD <= kSelectThreads, "a thread a channel");
    int most = 0;                                  // (every warp looks at all sums)
#pragma unroll
    for (int i = 0; i < 2 * kD; i += 32) most = max(most, s_sum[i + lane]);
    most = __reduce_max_sync(0xffffffffu, most);
    const int shift = max(0, 32 - __clz(most) - 7), half = 1 << shift >> 1;
    if (tid < 2 * kD) {
      const int y = min((s_sum[tid] + half) >> shift, 127);
      s_q[tid] = (int8_t)(tid < kD ? y : -y);
    }
  }
  // (the first CTA of the cluster is there: its memory may be written to)
  if constexpr (kParts) cluster_sync();
  else __syncthreads();
  // ---- scores
  const int front = min(p.front, n), own = max(front, (max(first, 0) >> p.log_block) - (p.recent - 1));
  {
    uint4 mine[kParcels];
#pragma unroll
    for (int r = 0; r < kParcels; ++r) mine[r] = *reinterpret_cast<const uint4*>(s_q + 16 * (4 * r + c));
    uint32_t least = 0xffffffffu, most = 0u;
#pragma unroll 1
    for (int j0 = b0 + warp * 8; j0 < b1; j0 += kDeep * kRound) {
      uint32_t key[kDeep];
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        int dot = 0;
#pragma unroll
        for (int r = 0; r < kParcels; ++r) {
          dot = __dp4a((int)v[k][r].x, (int)mine[r].x, dot);
          dot = __dp4a((int)v[k][r].y, (int)mine[r].y, dot);
          dot = __dp4a((int)v[k][r].z, (int)mine[r].z, dot);
          dot = __dp4a((int)v[k][r].w, (int)mine[r].w, dot);
        }
        dot += __shfl_xor_sync(0xffffffffu, dot, 1);
        dot += __shfl_xor_sync(0xffffffffu, dot, 2);
        key[k] = score_key(scale[k] == -INFINITY ? -INFINITY : __fmul_rn((float)dot, scale[k]));
      }
      if (j0 + kDeep * kRound < b1) fetch(j0 + kDeep * kRound);
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        const int j = j0 + k * kRound + sub;
        if (c == 0 && j < b1) {
          if (j >= front && j < own) {
            least = min(least, key[k]);
            most = max(most, key[k]);
          } else {
            key[k] = kAlways;
          }
          if (kParts && part > 0) st_cluster_u32(smem_u32(s_key + j), 0, key[k]);
          else s_key[j] = key[k];
        }
      }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0 && least <= most) {
      atomicMin(&s_range[2 * part], least);
      atomicMax(&s_range[2 * part + 1], most);
    }
  }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0u;
  if constexpr (kParts) {
    if (part > 0 && tid < 2) st_cluster_u32(smem_u32(s_range + 2 * part + tid), 0, s_range[2 * part + tid]);
    cluster_sync();
    if (part > 0) return;
    for (int i = 0; i < p.parts; ++i) {
      lo = min(lo, s_range[2 * i]);
      hi = max(hi, s_range[2 * i + 1]);
    }
  } else {
    lo = s_range[0];
    hi = s_range[1];
  }
  // ---- what is chosen: keys from `from` on, and of those equal to `edge` the first `ties`.  A pass deals the keys of a range to 2048 bins: scores of one
  //      kind spread over them, and two passes do mostly (with the keys' bits, eight at a time, four, whose first counts all in a few bins).
  uint32_t from = kAlways, edge = 0u;
  int ties = 0, left = p.chosen - (front + n - own);
#pragma unroll 1
  while (left > 0) {
    const int shift = max(0, 32 - __clz((int)(hi - lo)) - 11);
    for (int i = tid; i < kBins; i += kSelectThreads) s_hist[i] = 0;
    __syncthreads();
    for (int i = front + tid; i < own; i += kSelectThreads) {
      const uint32_t key = s_key[i];
      if (key >= lo && key <= hi) atomicAdd(&s_hist[(key - lo) >> shift], 1);
    }
    __syncthreads();
    // bins from the largest on, four a thread
    const int4 h = *reinterpret_cast<const int4*>(s_hist + kBins - 4 - 4 * tid);
    static_assert(kBins == 4 * kSelectThreads, "four bins a thread");
    const int sum = h.x + h.y + h.z + h.w;
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) s_red[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += s_red[w];
    int before = upto - sum;
    if (before < left && upto >= left) {                             // (one thread)
      int bin = kBins - 1 - 4 * tid, here = h.w;
      if (before + here < left) { before += here; here = h.z; --bin; }
      if (before + here < left) { before += here; here = h.y; --bin; }
      if (before + here < left) { before += here; here = h.x; --bin; }
      s_bin[0] = bin;
      s_bin[1] = left - before;
      s_bin[2] = here;
    }
    __syncthreads();
    const uint32_t start = lo + ((uint32_t)s_bin[0] << shift);
    left = s_bin[1];
    if (s_bin[2] == left) {
      from = start;
      break;
    }
    if (shift == 0) {
      from = start + 1;
      edge = start;
      ties = left;
      break;
    }
    lo = start;
    hi = min(hi, start + ((1u << shift) - 1u));
  }
  // ---- the list, by number
  const int seg = ((n + kWarps - 1) / kWarps + 31) & ~31, i0 = warp * seg, i1 = min(n, i0 + seg);
  int above = 0, equal = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    above += s_key[i] >= from;
    equal += ties > 0 && s_key[i] == edge;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) {
    s_count[warp] = above;
    s_count[kWarps + warp] = equal;
  }
  __syncthreads();
  int a0 = 0, e0 = 0;
  for (int w = 0; w < warp; ++w) {
    a0 += s_count[w];
    e0 += s_count[kWarps + w];
  }
  for (int i = i0; i < i1; i += 32) {
    const uint32_t key = i + lane < i1 ? s_key[i + lane] : 0u;
    const bool is_above = i + lane < i1 && key >= from, is_equal = i + lane < i1 && ties > 0 && key == edge;
    const uint32_t am = __ballot_sync(0xffffffffu, is_above), em = __ballot_sync(0xffffffffu, is_equal), in_front = (1u << lane) - 1u;
    const int a = a0 + __popc(am & in_front), tie = e0 + __popc(em & in_front);
    if (is_above || (is_equal && tie < ties)) out[a + min(tie, ties)] = i + lane;
    a0 += __popc(am);
    e0 += __popc(em);
  }
}

}  // namespace fa4
