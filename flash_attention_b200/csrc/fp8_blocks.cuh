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

// A warp a block and kv head: kD / 16 lanes a row of 16-byte pieces.
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
#pragma unroll 4
  for (int r = row0; r < there; r += kRows) {
    const uint4 u = *reinterpret_cast<const uint4*>(src + r * p.k_tok);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
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
  FastDiv div_hkv, div_query_blocks, div_page, div_group;
  uint32_t* status;
  uint32_t epoch;
};

constexpr int kSelectThreads = 256;
constexpr int kSelectBlocks = 53248;           // of a sequence: their scores are 208 KB

// Order of scores as whole numbers: the larger the score the larger the key; NaN as +inf, -0 as 0.
__device__ __forceinline__ uint32_t score_key(float s) {
  s = s != s ? INFINITY : s + 0.f;
  const uint32_t u = __float_as_uint(s);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kAlways = 0xffffffffu;      // (no score has it)

// A CTA a unit (sequence, query block, kv head).
template <int kD>
__global__ void __launch_bounds__(kSelectThreads) fp8_select_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kWarps = kSelectThreads / 32, kPieces = kD / 8;
  extern __shared__ uint32_t s_key[];
  __shared__ int s_sum[2 * kD], s_hist[256], s_red[kWarps], s_count[2 * kWarps];
  __shared__ __align__(16) int8_t s_q[2 * kD];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x, rest = fast_div(unit, p.div_hkv), head = unit - rest * p.Hkv, b = fast_div(rest, p.div_query_blocks),
            q0 = (rest - b * p.query_blocks) * p.query_block;
  pdl_wait();
  int sk = p.used[b], sq = p.fresh != nullptr ? p.fresh[b] : p.Sq;
  sk = sk < 0 ? 0 : (sk < p.capacity ? sk : p.capacity);
  sq = sq < 0 ? 0 : (sq < p.Sq ? sq : p.Sq);
  const int rows = max(0, min(sq - q0, p.query_block)), first = sk - sq + q0, end = rows > 0 ? max(0, first + rows) : 0;
  const int bt = 1 << p.log_block, n = (end + bt - 1) >> p.log_block;
  int32_t* out = p.blocks + (int64_t)unit * p.chosen;
  if (n <= p.chosen) {
    for (int i = tid; i < p.chosen; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  // ---- the query: largest element, sums of whole numbers, seven bits
  const __nv_bfloat16* q = p.q + b * p.q_b + (int64_t)q0 * p.q_s + (int64_t)head * p.group * p.q_h;
  const int R = rows * p.group;
  auto row_piece = [&](int i, float (&x)[8]) {
    const int r = i / kPieces, s = fast_div(r, p.div_group), h = r - s * p.group;
    unpack8(*reinterpret_cast<const uint4*>(q + (int64_t)s * p.q_s + h * p.q_h + 8 * (i % kPieces)), x);
  };
  for (int i = tid; i < 2 * kD; i += kSelectThreads) s_sum[i] = 0;
  uint32_t top = 0u;
  for (int i = tid; i < R * kPieces; i += kSelectThreads) {
    float x[8];
    row_piece(i, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = __float_as_uint(x[k]) & 0x7fffffffu;
      top = max(top, m < 0x7f800000u ? m : 0u);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_red[warp] = (int)top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = max(top, (uint32_t)s_red[w]);
  const int e = max((int)(top >> 23) - 127, -100);
  const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
  {
    int pos[8] = {}, neg[8] = {};
    for (int i = tid; i < R * kPieces; i += kSelectThreads) {       // (a thread stays with its eight channels)
      float x[8];
      row_piece(i, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int v = fabsf(x[k]) < INFINITY ? __float2int_rn(x[k] * up) : 0;
        pos[k] += max(v, 0);
        neg[k] += max(-v, 0);
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
    int most = tid < 2 * kD ? s_sum[tid] : 0;
    static_assert(2 * kD <= kSelectThreads, "a thread a channel");
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) s_red[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = max(most, s_red[w]);
    const int shift = max(0, 32 - __clz(most) - 7), half = 1 << shift >> 1;
    if (tid < 2 * kD) {
      const int v = min((s_sum[tid] + half) >> shift, 127);
      s_q[tid] = (int8_t)(tid < kD ? v : -v);
    }
  }
  __syncthreads();
  // ---- scores
  {
    constexpr int kLanes = kD / 8, kPer = 32 / kLanes;           // lanes of a block's 2 D bytes
    const int sub = lane / kLanes, c = lane % kLanes;
    const uint4 mine = *reinterpret_cast<const uint4*>(s_q + 16 * c);
    const int own = max(0, (max(first, 0) >> p.log_block) - (p.recent - 1));
    const int log_per = p.log_block;
#pragma unroll 4
    for (int j0 = warp * kPer; j0 < n; j0 += kWarps * kPer) {
      const int j = j0 + sub;
      int dot = 0;
      float scale = 0.f;
      bool fine = j < n;
      if (fine) {
        const int key = j << log_per, pg = fast_div(key, p.div_page), off = key - pg * p.page_size;
        const int page = p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b;
        fine = page >= 0 && page < p.num_pages;
        if (fine) {
          const int64_t at = ((int64_t)page * (p.page_size >> p.log_block) + (off >> p.log_block)) * p.Hkv + head;
          const uint4 v = *reinterpret_cast<const uint4*>(p.bounds + at * (2 * kD) + 16 * c);
          scale = p.scale[at];
          dot = __dp4a((int)v.x, (int)mine.x, dot);
          dot = __dp4a((int)v.y, (int)mine.y, dot);
          dot = __dp4a((int)v.z, (int)mine.z, dot);
          dot = __dp4a((int)v.w, (int)mine.w, dot);
        } else if (c == 0) {
          report_bad_index(p.status, p.epoch, kPageSite);
        }
      }
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (c == 0 && j < n) s_key[j] = j < p.front || j >= own ? kAlways : score_key(fine ? __fmul_rn((float)dot, scale) : -INFINITY);
    }
  }
  // ---- the chosen'th largest key, eight bits at a time
  if (tid == 0) {
    s_prefix = 0u;
    s_left = p.chosen;
  }
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    s_hist[tid] = 0;
    static_assert(kSelectThreads == 256, "a thread a bin");
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int i = tid; i < n; i += kSelectThreads) {
      const uint32_t key = s_key[i];
      if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&s_hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {
      // bins from the largest on: lane l has 255 - 8 l and the seven below
      int own[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += own[k] = s_hist[255 - 8 * lane - k];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const int left = s_left;
      int before = upto - sum;
      if (before < left && upto >= left) {                         // (one lane)
        int k = 0;
        while (before + own[k] < left) before += own[k++];
        s_prefix = prefix << 8 | (uint32_t)(255 - 8 * lane - k);
        s_left = left - before;
      }
    }
    __syncthreads();
  }
  // ---- the list, by number: all above that key, and of those equal to it the first ones
  const uint32_t edge = s_prefix;
  const int ties = s_left, per = ((n + kWarps - 1) / kWarps + 31) & ~31, i0 = warp * per, i1 = min(n, i0 + per);
  int above = 0, equal = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    above += s_key[i] > edge;
    equal += s_key[i] == edge;
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
    const bool is_above = i + lane < i1 && key > edge, is_equal = i + lane < i1 && key == edge;
    const uint32_t am = __ballot_sync(0xffffffffu, is_above), em = __ballot_sync(0xffffffffu, is_equal), in_front = (1u << lane) - 1u;
    const int a = a0 + __popc(am & in_front), q_at = e0 + __popc(em & in_front);
    if (is_above || (is_equal && q_at < ties)) out[a + min(q_at, ties)] = i + lane;
    a0 += __popc(am);
    e0 += __popc(em);
  }
}

}  // namespace fa4
