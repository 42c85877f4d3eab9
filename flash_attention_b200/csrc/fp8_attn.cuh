// Attention of bf16 queries over the 8-bit KV cache.
#pragma once
#include "fp8_append.cuh"

namespace fa4 {

struct Fp8Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_b, q_s, q_h, o_b, o_s, o_h;   // elements
  const uint8_t *kc, *vc;
  int64_t kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head;   // bytes
  const float *k_scale, *v_scale;
  const int32_t *used, *fresh, *table;
  const float* sink;
  int B, Sq, Hq, Hkv, group, D, log_block, num_pages, page_size, pages_per_seq, capacity;
  FastDiv div_page, div_group;
  float scale, softcap;              // softmax scale
  int win_left, win_right;           // -1: unlimited
  uint32_t* status;
  uint32_t epoch;
  uint64_t budget_ns;
};

// The keys [lo, hi) that query row s of a sequence with `sk` keys and `sq` rows sees.
__device__ __forceinline__ int2 seen_by(const Fp8Params& p, int sk, int sq, int s) {
  const int at = sk - sq + s;
  int lo = 0, hi = sk;
  if (p.win_left >= 0 && at - p.win_left > 0) lo = at - p.win_left;
  if (p.win_right >= 0 && (int64_t)at + p.win_right + 1 < sk) hi = at + p.win_right + 1;
  return make_int2(lo, hi > lo ? hi : lo);
}

// One query row a CTA of 128 threads, keys in steps of 128: a thread has a key, then an output element.
__global__ void __launch_bounds__(128) fp8_attn_rows_kernel(const __grid_constant__ Fp8Params p) {
  __shared__ float s_q[128], s_p[128], s_red[4];
  __shared__ int s_page[128];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int s = blockIdx.x / p.Hq, h = blockIdx.x - s * p.Hq, b = blockIdx.y, hk = h / p.group;
  pdl_wait();
  int sk = p.used[b], sq = p.fresh != nullptr ? p.fresh[b] : p.Sq;
  sk = sk < 0 ? 0 : (sk < p.capacity ? sk : p.capacity);
  if (s >= sq || s >= p.Sq) return;
  sq = sq < p.Sq ? sq : p.Sq;
  const int2 see = seen_by(p, sk, sq, s);
  if (tid < p.D) s_q[tid] = __bfloat162float(p.q[b * p.q_b + s * p.q_s + h * p.q_h + tid]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  if (p.sink != nullptr) {
    m = p.sink[h];
    l = 1.f;
  }
  for (int j0 = see.x; j0 < see.y; j0 += 128) {
    const int j = j0 + tid;
    float x = -INFINITY, vs = 0.f;
    int page = -1;
    if (j < see.y) {
      const int pg = fast_div(j, p.div_page), off = j - pg * p.page_size;
      page = p.table != nullptr ? p.table[(int64_t)b * p.pages_per_seq + pg] : b;
      float dot = 0.f;
      if (page >= 0 && page < p.num_pages) {
        const int64_t at = ((int64_t)page * (p.page_size >> p.log_block) + (off >> p.log_block)) * p.Hkv + hk;
        vs = p.v_scale[at];
        const uint8_t* kr = p.kc + page * p.kc_page + off * p.kc_tok + hk * p.kc_head;
        for (int d = 0; d < p.D; d += 4) {
          float y[4];
          unpack4_e4m3(*reinterpret_cast<const uint32_t*>(kr + d), y);
          dot += s_q[d] * y[0] + s_q[d + 1] * y[1] + s_q[d + 2] * y[2] + s_q[d + 3] * y[3];
        }
        dot *= p.k_scale[at];
      } else {
        report_bad_index(p.status, p.epoch, kPageSite);
        page = -1;
      }
      x = dot * p.scale;
      if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
    }
    float top = x;
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) s_red[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(m, fmaxf(s_red[0], s_red[1])), fmaxf(s_red[2], s_red[3]));
    const float ref = top == -INFINITY ? 0.f : top, keep = expf(m - ref);
    const float w = j < see.y ? expf(x - ref) : 0.f;
    m = top;
    s_p[tid] = w * vs;
    s_page[tid] = page;
    float sum = w;
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    __syncthreads();
    if (lane == 0) s_red[warp] = sum;
    __syncthreads();
    l = l * keep + s_red[0] + s_red[1] + s_red[2] + s_red[3];
    o *= keep;
    if (tid < p.D) {
      for (int i = 0; i < 128 && j0 + i < see.y; ++i) {
        if (s_page[i] < 0) continue;
        const int pg = fast_div(j0 + i, p.div_page), off = j0 + i - pg * p.page_size;
        float y[4];
        unpack4_e4m3(p.vc[s_page[i] * p.vc_page + off * p.vc_tok + hk * p.vc_head + tid], y);
        o += s_p[i] * y[0];
      }
    }
    __syncthreads();
  }
  if (tid < p.D) p.out[b * p.o_b + s * p.o_s + h * p.o_h + tid] = __float2bfloat16(l > 0.f || !(l == l) ? o / l : 0.f);
  if (tid == 0 && p.lse != nullptr) p.lse[((int64_t)b * p.Hq + h) * p.Sq + s] = m == -INFINITY ? -INFINITY : m + logf(l);
}

}  // namespace fa4
