// What the kernels of the attention over the 8-bit KV cache share: parameters, masks, the merge of splits.
#pragma once
#include "fp8_append.cuh"

namespace fa4 {

struct Fp8Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_b, q_s, q_h, o_b, o_s, o_h;   // elements
  const float *k_scale, *v_scale;
  const int32_t *used, *fresh, *table;
  const float* sink;
  int num_splits;                    // 0: dealt by the lengths (decode kernel); -1: whole units (chosen blocks)
  int meet;                          // chosen blocks: CTAs of a cluster, whose splits of a unit meet in shared memory; else 1
  float* o_partial;                  // rows of D fp32, normalised; log2 of their sums, the sink left out
  float* lse_partial;                //   many rows: (splits, B, Sq, Hq); decode: (slots, unit_rows)
  int2* pieces;                      // decode, dealt: (B, Hkv) first CTA and number of pieces of a unit
  int unit_rows;                     // Sq * group
  int bundle, bundles;               // kv heads side by side (a divisor of Hkv), and how many such
  int box;                           // keys of a tensor-map box: 128, or what pages and tiles of 128 share
  int B, Sq, Hq, Hkv, group, D, log_block, num_pages, page_size, pages_per_seq, capacity;
  int row_tiles, cta_rows;           // many rows: tiles of 128 or 256 rows of a kv head and sequence
  FastDiv div_page, div_group, div_hq, div_sq, div_groups;   // (groups of CTAs of the decode kernel)
  // scores in log2 units: (q . k8) * ks * sl2, or cap_out * tanh((q . k8) * ks * cap_in) with a soft cap
  float sl2, cap_in, cap_out;
  int win_left, win_right;           // -1: unlimited
  // Chosen blocks: (B, query blocks, Hkv, chosen) ascending.  A unit's sequence is then a query block of a sequence, its keys are those of
  // its list one behind the other.
  const int32_t* blocks;
  int chosen, query_block, query_blocks;
  int seqs;                          // B * query_blocks (dense: B)
  int cta_units, more_units;         // whole units: as many a CTA, and one more for the first `more_units`
  FastDiv div_query_blocks, div_query_block, div_hkv, div_splits;
  uint32_t* status;
  uint32_t epoch;
  uint64_t budget_ns;
};

// The keys [lo, hi) that query row s of a sequence with `sk` keys and `sq` rows sees.
__device__ __forceinline__ int2 seen_by(const Fp8Params& p, int sk, int sq, int s) {
  const int at = sk - sq + s;
  const int lo = p.win_left >= 0 && p.win_left < at ? at - p.win_left : 0;
  const int hi = p.win_right >= 0 && p.win_right < sq - 1 - s ? at + p.win_right + 1 : sk;     // (no sum passes 2^31)
  return make_int2(lo, hi > lo ? hi : lo);
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh in fp32 (tanh.approx is off by 2^-11, 1 % of a weight at a cap of 30): from 0.5 on 1 - 2 / (1 + e^2x), off by a few 2^-23; below, where that
// loses the bits that cancel, x times a polynomial in x^2 through the values of tanh x / x at the five Chebyshev nodes of [0, 0.25].
__device__ __forceinline__ float tanh_of(float x) {
  const float e = ex2_approx(x * (2.f * 1.4426950408889634f)), far = fmaf(-2.f, rcp_approx(1.f + e), 1.f), z = x * x;
  const float near = x * fmaf(fmaf(fmaf(fmaf(0.017131344f, z, -0.052984239f), z, 0.13324751f), z, -0.33333068f), z, 1.f);
  return fabsf(x) < 0.5f ? near : far;
}

// Valid keys and rows of a sequence.
struct SeqLens {
  int sk, sq;
};
__device__ __forceinline__ SeqLens lens_of(const Fp8Params& p, int b) {
  SeqLens n;
  n.sk = p.used[b];
  n.sk = n.sk < 0 ? 0 : (n.sk < p.capacity ? n.sk : p.capacity);
  n.sq = p.fresh != nullptr ? p.fresh[b] : p.Sq;
  n.sq = n.sq < 0 ? 0 : (n.sq < p.Sq ? n.sq : p.Sq);
  return n;
}

// ---- chosen blocks ----
// Query block `v` of a call: its sequence and first row.
struct QueryBlock {
  int b, q0;
};
template <bool kBlocks>
__device__ __forceinline__ QueryBlock query_block_of(const Fp8Params& p, int v) {
  if constexpr (!kBlocks) return {v, 0};
  const int b = fast_div(v, p.div_query_blocks);
  return {b, (v - b * p.query_blocks) * p.query_block};
}
// Valid keys and rows of a unit's sequence; with chosen blocks the position of its first row (which may be negative) and its rows.
template <bool kBlocks>
__device__ __forceinline__ SeqLens unit_lens(const Fp8Params& p, int v) {
  const QueryBlock at = query_block_of<kBlocks>(p, v);
  SeqLens n = lens_of(p, at.b);
  if constexpr (kBlocks) {
    n.sk = n.sk - n.sq + at.q0;
    n.sq = n.sq - at.q0;
    n.sq = n.sq < 0 ? 0 : (n.sq < p.query_block ? n.sq : p.query_block);
  }
  return n;
}
// A list of chosen blocks: it ends at the first entry that is not above the one in front of it.
__device__ __forceinline__ const int32_t* list_of(const Fp8Params& p, int v, int hk) { return p.blocks + ((int64_t)v * p.Hkv + hk) * p.chosen; }
// How many of its keys lie in front of position `end`, by a whole warp.
__device__ __forceinline__ int keys_in_front(const Fp8Params& p, const int32_t* list, int end) {
  const int lane = threadIdx.x & 31, block = end >> p.log_block;
  int keys = 0, last = -1;
  if (end <= 0) return 0;
#pragma unroll 1
  for (int i0 = 0; i0 < p.chosen; i0 += 32) {
    const int e = i0 + lane < p.chosen ? list[i0 + lane] : -1, up = __shfl_up_sync(0xffffffffu, e, 1);
    const uint32_t over = __ballot_sync(0xffffffffu, e <= (lane == 0 ? last : up)), there = over == 0u ? 0xffffffffu : (over & -over) - 1u;
    const uint32_t whole = __ballot_sync(0xffffffffu, e < block) & there, part = __ballot_sync(0xffffffffu, e == block) & there;
    keys += (__popc(whole) << p.log_block) + (part != 0u ? end & ((1 << p.log_block) - 1) : 0);
    if (whole != 0xffffffffu) break;
    last = __shfl_sync(0xffffffffu, e, 31);
  }
  return keys;
}

// A row's result from its sum `l` under the reference `m` (log2 units) and the sink of its head: the factor of the
// accumulated values, and the LSE in natural units.
struct RowEnd {
  float factor, lse;
};
__device__ __forceinline__ RowEnd finish_row(float m, float l, const float* sink, int h) {
  constexpr float kLn2 = 0.6931471805599453f;
  RowEnd e;
  float top = m, keep = 1.f;
  if (sink != nullptr) {
    const float x = sink[h] * 1.4426950408889634f;
    top = fmaxf(m, x);
    const float ref = top == -INFINITY ? 0.f : top;               // (a sink of -inf in a row that sees nothing: it adds 0)
    keep = ex2_approx(m - ref);
    l = fmaf(l, keep, ex2_approx(x - ref));                        // (of a row of NaN alone m is -inf and l NaN)
  }
  if (top == -INFINITY && l == 0.f) return {0.f, -INFINITY};    // (a row of NaN has l = NaN and goes on)
  e.factor = keep * rcp_approx(l);
  e.lse = (top + lg2_approx(l)) * kLn2;
  return e;
}

// Merge of a row's n partial results by one warp; sum_of(i), values_of(i): the log2 of the i-th one's sum, four of its values.
constexpr int kFp8CombineWarps = 4;
template <class SumOf, class ValuesOf>
__device__ __forceinline__ void merge_parts(const Fp8Params& p, int b, int s, int h, int lane, int n, SumOf sum_of, ValuesOf values_of) {
  const int col = 4 * lane;
  float m = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 8) {
    float l[8], top = m;
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      l[j] = -INFINITY;
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + j < n) {
        l[j] = sum_of(i0 + j);
        if (col < p.D) v[j] = values_of(i0 + j);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // (a part without a key wrote no values; they are asked for with the sums all the same)
      if (l[j] == -INFINITY) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      top = fmaxf(top, l[j]);
    }
    const float ref = top == -INFINITY ? 0.f : top, keep = ex2_approx(m - ref);
    sum *= keep;
    acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = ex2_approx(l[j] - ref);
      sum += w;
      const float w8 = w * 0x1p-8f;        // (up to 148 parts, whose values may be as large as bf16 has them)
      acc.x = fmaf(w8, v[j].x, acc.x); acc.y = fmaf(w8, v[j].y, acc.y);
      acc.z = fmaf(w8, v[j].z, acc.z); acc.w = fmaf(w8, v[j].w, acc.w);
    }
    m = top;
  }
  const RowEnd e = finish_row(m, sum, p.sink, h);
  const float up = e.factor * 0x1p8f;
  if (col < p.D)
    *reinterpret_cast<uint2*>(p.out + b * p.o_b + s * p.o_s + h * p.o_h + col) =
        make_uint2(pack_bf16x2(acc.x * up, acc.y * up), pack_bf16x2(acc.z * up, acc.w * up));
  if (lane == 0 && p.lse != nullptr) p.lse[((int64_t)b * p.Hq + h) * p.Sq + s] = e.lse;
}
// The same from memory; at(i): index of the i-th one's row.
template <class At>
__device__ __forceinline__ void merge_row(const Fp8Params& p, int b, int s, int h, int lane, int n, At at) {
  merge_parts(p, b, s, h, lane, n, [&](int i) { return p.lse_partial[at(i)]; },
              [&](int i) { return *reinterpret_cast<const float4*>(p.o_partial + at(i) * p.D + 4 * lane); });
}

// The splits of the kernel for many rows: a warp a row.
__global__ void __launch_bounds__(kFp8CombineWarps * 32) fp8_combine_kernel(const __grid_constant__ Fp8Params p) {
  const uint32_t r = blockIdx.x * kFp8CombineWarps + (threadIdx.x >> 5), rows = (uint32_t)p.B * p.Sq * p.Hq;
  pdl_wait();
  if (r >= rows) return;
  const int bs = fast_div((int)r, p.div_hq), h = (int)r - bs * p.Hq, b = fast_div(bs, p.div_sq), s = bs - b * p.Sq;
  if (p.fresh != nullptr && s >= p.fresh[b]) return;
  merge_row(p, b, s, h, threadIdx.x & 31, p.num_splits, [&](int i) { return (int64_t)i * rows + r; });
}

}  // namespace fa4
