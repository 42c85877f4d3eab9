// Keys and values of new tokens into the 8-bit KV cache, keys (and queries) rotated by their positions on the way.
//
//   pair (x1, x2) at position t:  y1 = x1 cos[t] - x2 sin[t],  y2 = x2 cos[t] + x1 sin[t]      (fp32, each step rounded)
//   scale of a block of tokens and head: the smallest 2^e with max |y| <= 448 * 2^e, no less than the scale that a
//   block in use has;   byte = e4m3_rne(y / scale)
//
// A power of two loses nothing to any other scale (an e4m3 value is a floating one: its error is relative down to 2^-6),
// and it lets a block grow: when a token raises the scale the bytes in the block are multiplied by 2^-k, which is
// exact but for values that fall below 2^-6 of the new scale.  So tokens that come one by one leave (but for those) the bytes
// of the block quantised at once.
//
// A unit is one block of one sequence, kv head and K or V, which one CTA (for a few tokens: one warp) owns: maxima need no atomics, old
// bytes are read and written by the same threads.  A thread has 16 elements of a row, as two 16-byte pieces that hold eight whole
// pairs.  With several rows it turns each twice, for the maximum and for the bytes, the second time from L1.
//
// What bounds it: 2 x 8192 tokens of 8 kv heads with 32 query heads, D = 128, blocks of 128: 87 us, 41 of them keys and values (101 MB, 2.5 TB/s), the rest q
// (268 MB, 5.8 TB/s).  Keys and values wait for loads (11 warps of an average instruction's latency, issue slots 42 % busy, 32 warps of an SM
// with 63 registers): a row is read twice, the angles of a key come from L1.  Not finite values are looked for by one multiply-add an element and
// treated on a path of their own; with that and the rows a thread has, keys and values went from 57 to 41.  More rows in flight (loops unrolled by four
// rather than two) 45, the loads of four query heads in front of their stores 45 with q's part unchanged: fewer warps.  A few tokens are a
// launch: 64 sequences of one token 2.9 us in a graph.
#pragma once
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace fa4 {

enum Fp8Site { kPositionSite = 120, kRotationSite = 122 };

struct AppendParams {
  const __nv_bfloat16 *k, *v, *q;
  __nv_bfloat16* q_out;              // (B, S, Hq, D) contiguous
  int64_t k_b, k_s, k_h, v_b, v_s, v_h, q_b, q_s, q_h;   // elements
  uint8_t *kc, *vc;
  int64_t kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head;   // bytes
  float *k_scale, *v_scale;
  const int32_t *seqlens, *fresh, *table;
  const void *cos, *sin;
  int rotary_dim, rotary_rows, rotary_bf16, interleaved;
  int B, S, Hq, Hkv, D, log_block, num_pages, page_size, pages_per_seq;
  int blocks;                        // units of a sequence and head: blocks that S tokens may touch
  int units;
  int kv_ctas;                       // CTAs of keys and values, in front of those of q
  int q_heads, q_head_groups;        // heads of a thread; groups of them
  FastDiv div_blocks, div_hkv2, div_page, div_groups, div_s;
  uint32_t* status;
  uint32_t epoch;
};

// Where the 16 elements of chunk c of a row lie: two runs of eight that are pairs of each other or (interleaved, or
// behind the rotated part) one run of 16.
struct Chunk {
  int a, b;
  bool turned;
};
__device__ __forceinline__ Chunk chunk_of(const AppendParams& p, int c) {
  const bool turned = 16 * c < p.rotary_dim;
  if (turned && !p.interleaved) return {8 * c, (p.rotary_dim >> 1) + 8 * c, true};
  return {16 * c, 16 * c + 8, turned};
}

__device__ __forceinline__ void unpack8(uint4 u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

struct Angles {
  float c[8], s[8];
};
// The angles of the eight pairs of chunk c at table row `row` (inside the table).
__device__ __forceinline__ Angles load_angles(const AppendParams& p, int row, int c) {
  Angles g;
  const int64_t at = (int64_t)row * (p.rotary_dim >> 1) + 8 * c;
  if (p.rotary_bf16) {
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.cos) + at), g.c);
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.sin) + at), g.s);
  } else {
    const float4* c4 = reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at);
    const float4* s4 = reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at);
    const float4 c0 = c4[0], c1 = c4[1], s0 = s4[0], s1 = s4[1];
    g.c[0] = c0.x; g.c[1] = c0.y; g.c[2] = c0.z; g.c[3] = c0.w; g.c[4] = c1.x; g.c[5] = c1.y; g.c[6] = c1.z; g.c[7] = c1.w;
    g.s[0] = s0.x; g.s[1] = s0.y; g.s[2] = s0.z; g.s[3] = s0.w; g.s[4] = s1.x; g.s[5] = s1.y; g.s[6] = s1.z; g.s[7] = s1.w;
  }
  return g;
}
__device__ __forceinline__ void turn(float& x1, float& x2, float c, float s) {
  const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  x2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
  x1 = y1;
}
// Elements 0-7 of x are run a, 8-15 run b.
__device__ __forceinline__ void turn16(float (&x)[16], const Angles& g, bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[2 * i], x[2 * i + 1], g.c[i], g.s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[i], x[8 + i], g.c[i], g.s[i]);
  }
}

// Four e4m3 bytes of x * inv (round to nearest even, saturating at 448; NaN stays NaN).
__device__ __forceinline__ uint32_t pack4_e4m3(float x0, float x1, float x2, float x3) {
  uint32_t r;
  asm("{\n"
      ".reg .b16 lo, hi;\n"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
      "mov.b32 %0, {lo, hi};\n"
      "}\n"
      : "=r"(r)
      : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
  return r;
}
__device__ __forceinline__ void unpack4_e4m3(uint32_t w, float* x) {
  uint32_t lo, hi;
  asm("{\n"
      ".reg .b16 l, h;\n"
      "mov.b32 {l, h}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n"
      "}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

// The smallest power of two, from 2^-120 on, by which `top` (finite, >= 0) is at most 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float top) {
  const uint32_t bits = __float_as_uint(top);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);   // (a denormal counts as below 2^-120)
  e = e < -120 ? -120 : (e > 120 ? 120 : e);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// x / scale with r = RN(1 / scale): the product and one residual step, the correctly rounded quotient (Markstein 1990) wherever
// it is an ordinary number; NaN where x is not finite (an infinity less itself).
__device__ __forceinline__ float quotient(float x, float scale, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-q, scale, x), r, q);
}

// Where a unit lies.
struct AppendUnit {
  const __nv_bfloat16* src;          // of the token at position `held`
  uint8_t* dst;                      // of position `start`
  float* scale;
  float before;                      // its scale, if it holds tokens already (`kept`)
  int held, start, t0, t1;           // tokens in front of the call; first position of the block; new ones in it
  bool is_v, kept, any;
};
__device__ __forceinline__ AppendUnit find_unit(const AppendParams& p, int unit, bool report) {
  AppendUnit u = {};
  // unit = ((b * Hkv + head) * 2 + is_v) * blocks + blk
  const int rest = fast_div(unit, p.div_blocks), blk = unit - rest * p.blocks;
  const int b = fast_div(rest, p.div_hkv2), hv = rest - b * 2 * p.Hkv, head = hv >> 1;
  u.is_v = (hv & 1) != 0;
  u.held = p.seqlens[b];
  int n = p.fresh != nullptr ? p.fresh[b] : p.S;
  n = n < 0 ? 0 : (n < p.S ? n : p.S);
  if (n == 0) return u;
  if (u.held < 0) {
    if (report) report_bad_index(p.status, p.epoch, kPositionSite);
    return u;
  }
  const int bt = 1 << p.log_block;
  // (positions stay below 2^31: those of the cache do, and the first one behind it ends the unit)
  const int64_t start = (int64_t)((u.held >> p.log_block) + blk) << p.log_block, end = (int64_t)u.held + n;
  if (start >= end) return u;
  if (start >= (int64_t)p.pages_per_seq * p.page_size) {
    if (report) report_bad_index(p.status, p.epoch, kPositionSite);
    return u;
  }
  u.start = (int)start;
  u.t0 = u.held > u.start ? u.held : u.start;
  u.t1 = end < start + bt ? (int)end : u.start + bt;
  const int pg = fast_div(u.start, p.div_page), off = u.start - pg * p.page_size;
  const int page = p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b;
  if (page < 0 || page >= p.num_pages) {
    if (report) report_bad_index(p.status, p.epoch, kPageSite);
    return u;
  }
  u.any = true;
  u.scale = (u.is_v ? p.v_scale : p.k_scale) + ((int64_t)page * (p.page_size >> p.log_block) + (off >> p.log_block)) * p.Hkv + head;
  u.dst = u.is_v ? p.vc + page * p.vc_page + off * p.vc_tok + head * p.vc_head : p.kc + page * p.kc_page + off * p.kc_tok + head * p.kc_head;
  u.src = u.is_v ? p.v + b * p.v_b + head * p.v_h : p.k + b * p.k_b + head * p.k_h;
  u.kept = u.held > u.start;
  u.before = u.kept ? *u.scale : 0.f;
  return u;
}

// kThreads threads of a unit (32: a warp, whose maxima stay in registers), a row each or (kMany) several.
template <int kThreads, bool kMany>
__device__ __forceinline__ void append_unit(const AppendParams& p, int unit, int tid, float* s_max) {
  const AppendUnit u = find_unit(p, unit, tid == 0);
  if (!u.any) return;
  const int log_chunks = p.D == 128 ? 3 : 2;                 // chunks of 16 in a row
  const int c = tid & ((1 << log_chunks) - 1), row0 = tid >> log_chunks, step = kThreads >> log_chunks;
  const Chunk ch = !u.is_v && p.cos != nullptr ? chunk_of(p, c) : Chunk{16 * c, 16 * c + 8, false};
  const int64_t src_tok = u.is_v ? p.v_s : p.k_s, dst_tok = u.is_v ? p.vc_tok : p.kc_tok;
  auto row_of = [&](int t, float (&x)[16]) {                 // the thread's piece of the row at position t, turned
    const __nv_bfloat16* row = u.src + (t - u.held) * src_tok;
    unpack8(*reinterpret_cast<const uint4*>(row + ch.a), x);
    unpack8(*reinterpret_cast<const uint4*>(row + ch.b), x + 8);
    if (ch.turned) turn16(x, load_angles(p, t < p.rotary_rows ? t : p.rotary_rows - 1, c), p.interleaved != 0);
  };
  // zero is NaN if an element is not finite
  float x[16], top = 0.f, zero = 0.f;
  auto take = [&](const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      top = fmaxf(top, fabsf(v[i]));
      zero = fmaf(v[i], 0.f, zero);
    }
  };
  if constexpr (kMany) {
#pragma unroll 2
    for (int t = u.t0 + row0; t < u.t1; t += step) {
      float y[16];
      row_of(t, y);
      take(y);
    }
  } else if (u.t0 + row0 < u.t1) {
    row_of(u.t0 + row0, x);
    take(x);
  }
  if (ch.turned && row0 == 0 && u.t1 > p.rotary_rows) report_bad_index(p.status, p.epoch, kRotationSite);
  const bool fine = zero == 0.f;
  if (!fine) {
    top = 0.f;
#pragma unroll 1
    for (int t = u.t0 + row0; t < u.t1; t += step) {
      if constexpr (kMany) row_of(t, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float m = fabsf(x[i]);
        top = fmaxf(top, m < INFINITY ? m : 0.f);
      }
      if constexpr (!kMany) break;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if constexpr (kThreads > 32) {
    if ((tid & 31) == 0) s_max[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, s_max[w]);
  }
  const float need = scale_for(top);
  const float scale = u.kept ? fmaxf(u.before, need) : need;
  if (u.kept && scale != u.before) {
    const float again = __fdiv_rn(u.before, scale);
#pragma unroll 1
    for (int t = row0; t < u.t0 - u.start; t += step) {
      uint4* held = reinterpret_cast<uint4*>(u.dst + t * dst_tok + 16 * c);
      uint4 v = *held;
      uint32_t* w = &v.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y[4];
        unpack4_e4m3(w[i], y);
        w[i] = pack4_e4m3(__fmul_rn(y[0], again), __fmul_rn(y[1], again), __fmul_rn(y[2], again), __fmul_rn(y[3], again));
      }
      *held = v;
    }
  }
  // (old scales need not be powers of two)
  const bool product = fine && (__float_as_uint(scale) & 0x7fffffu) == 0u;
  const float inv = __frcp_rn(scale);
  auto bytes_of = [&](int t, float (&v)[16]) {
    if (product) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __fmul_rn(v[i], inv);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = quotient(v[i], scale, inv);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack4_e4m3(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    uint8_t* to = u.dst + (t - u.start) * dst_tok;
    if (ch.b == ch.a + 8) {
      *reinterpret_cast<uint4*>(to + ch.a) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2*>(to + ch.a) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(to + ch.b) = make_uint2(w[2], w[3]);
    }
  };
  if constexpr (kMany) {
#pragma unroll 2
    for (int t = u.t0 + row0; t < u.t1; t += step) {
      float y[16];
      row_of(t, y);
      bytes_of(t, y);
    }
  } else if (u.t0 + row0 < u.t1) {
    bytes_of(u.t0 + row0, x);
  }
  if constexpr (kThreads == 32) __syncwarp();                  // (every lane has read it)
  if (tid == 0) *u.scale = scale;
}

// Rows of q: a thread turns one chunk of `q_heads` heads of a row, whose angles it loads once.
__device__ __forceinline__ void rotate_queries(const AppendParams& p, int64_t item) {
  const int log_chunks = p.D == 128 ? 3 : 2;
  const int c = (int)item & ((1 << log_chunks) - 1);
  const int64_t rest = item >> log_chunks;                     // (row, group)
  if (rest >= (int64_t)p.B * p.S * p.q_head_groups) return;
  const int row = fast_div((int)rest, p.div_groups), group = (int)rest - row * p.q_head_groups;
  const int b = fast_div(row, p.div_s), s = row - b * p.S;
  int64_t t = (int64_t)p.seqlens[b] + s;
  if (t < 0 || t >= p.rotary_rows) {
    // (rows of padding may lie behind the tables)
    if (p.fresh == nullptr || s < p.fresh[b]) report_bad_index(p.status, p.epoch, kRotationSite);
    t = t < 0 ? 0 : p.rotary_rows - 1;
  }
  const Chunk ch = chunk_of(p, c);
  Angles g;
  if (ch.turned) g = load_angles(p, (int)t, c);
  const int h0 = group * p.q_heads, h1 = h0 + p.q_heads < p.Hq ? h0 + p.q_heads : p.Hq;
  const __nv_bfloat16* src = p.q + b * p.q_b + s * p.q_s;
  __nv_bfloat16* dst = p.q_out + (int64_t)row * p.Hq * p.D;
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    uint4 a = *reinterpret_cast<const uint4*>(src + h * p.q_h + ch.a), e = *reinterpret_cast<const uint4*>(src + h * p.q_h + ch.b);
    if (ch.turned) {
      float x[16];
      unpack8(a, x);
      unpack8(e, x + 8);
      turn16(x, g, p.interleaved != 0);
      a = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
      e = make_uint4(pack_bf16x2(x[8], x[9]), pack_bf16x2(x[10], x[11]), pack_bf16x2(x[12], x[13]), pack_bf16x2(x[14], x[15]));
    }
    *reinterpret_cast<uint4*>(dst + h * p.D + ch.a) = a;
    *reinterpret_cast<uint4*>(dst + h * p.D + ch.b) = e;
  }
}

// kThreads = 32: a warp a unit, four units a CTA; else a CTA a unit.  The CTAs from kv_ctas on turn q.
template <int kThreads, bool kMany>
__global__ void __launch_bounds__(kThreads == 32 ? 128 : kThreads)
fp8_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kCta = kThreads == 32 ? 128 : kThreads;
  __shared__ float s_max[kCta / 32];
  pdl_wait();
  if ((int)blockIdx.x >= p.kv_ctas) {
    rotate_queries(p, (int64_t)(blockIdx.x - p.kv_ctas) * kCta + threadIdx.x);
  } else if constexpr (kThreads == 32) {
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (unit < p.units) append_unit<32, kMany>(p, unit, threadIdx.x & 31, s_max);
  } else {
    append_unit<kThreads, kMany>(p, blockIdx.x, threadIdx.x, s_max);
  }
}

}  // namespace fa4
