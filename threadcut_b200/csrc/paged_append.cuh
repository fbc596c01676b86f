// A step's queries and keys normalised (optional) and rotated, keys and values written into the slots
// of a paged cache, in one launch: the chain of torch ops in front of tc_paged_write (transformers'
// Qwen3Attention q_norm, k_norm, apply_rotary_pos_emb, then the cache update of threadcut/kv.py:64-77).
//
// Per token and head, x being its d elements:
//   z = x * rsqrt(mean(x^2) + eps) * w                      (with a norm weight; else z = x)
//   out[i] = z[i] cos[i] - z[i + rot/2] sin[i]              i < rot/2
//   out[i] = z[i] cos[i] + z[i - rot/2] sin[i]              rot/2 <= i < rot
//   out[i] = z[i]                                           i >= rot (partial rotation)
// in fp32 from the loaded values on, rounded once to T at the store. (The torch chain, and with it
// tc_qk_norm_rope, rounds to T after each op; one rounding is nearer to the formula.)
#pragma once

#include <stdint.h>

namespace tc {

constexpr int kMaxAppendDim = 512;  // head size of the paged append (a warp holds a row in 2 KB of shared memory)

struct PagedAppendParams {
  const void* q;  // [hq][t][d] with element strides (q_sh, q_st), or null
  const void* k;  // [hkv][t][d]
  const void* v;
  void* q_out;    // [hq][t][d] with strides (qo_sh, qo_st); may be q itself
  void* kp;       // this layer's pools
  void* vp;
  const void* q_w;  // norm weights [d] of T, or null
  const void* k_w;
  const void* cos_t;  // [t][rot] of T or (table_f32) fp32, row strides cos_st / sin_st
  const void* sin_t;
  int hq, hkv, d, rot;
  int table_f32;
  int64_t t;
  int64_t q_sh, q_st, k_sh, k_st, v_sh, v_st, qo_sh, qo_st, cos_st, sin_st;
  int64_t page_rows, num_pages;
  int64_t s_page, s_h, s_row;
  const int32_t* slots;  // [t][2]: page, row
  float eps, inv_d;
};

// Any type, head size, strides and alignment: one warp per (token, head), the row staged in shared
// memory as fp32 so each lane can read its element's partner.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  __shared__ float rows[8][kMaxAppendDim];
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.hq + 2 * p.hkv;
  float* z = rows[warp];
  for (int64_t task = blockIdx.x * 8 + warp; task < p.t * heads; task += (int64_t)gridDim.x * 8) {
    const int64_t tok = task / heads;
    const int hh = (int)(task - tok * heads);
    const bool isq = hh < p.hq, isv = hh >= p.hq + p.hkv;
    const int h = isq ? hh : (isv ? hh - p.hq - p.hkv : hh - p.hq);
    const T* src = isq   ? static_cast<const T*>(p.q) + h * p.q_sh + tok * p.q_st
                   : isv ? static_cast<const T*>(p.v) + h * p.v_sh + tok * p.v_st
                         : static_cast<const T*>(p.k) + h * p.k_sh + tok * p.k_st;
    T* dst;
    if (isq) {
      dst = static_cast<T*>(p.q_out) + h * p.qo_sh + tok * p.qo_st;
    } else {
      const int64_t page = p.slots[2 * tok], row = p.slots[2 * tok + 1];
      if (page < 0 || page >= p.num_pages || row < 0 || row >= p.page_rows) continue;
      dst = static_cast<T*>(isv ? p.vp : p.kp) + page * p.s_page + h * p.s_h + row * p.s_row;
    }
    if (isv) {
      for (int i = lane; i < p.d; i += 32) dst[i] = src[i];
      continue;
    }
    const T* w = static_cast<const T*>(isq ? p.q_w : p.k_w);
    float ss = 0.f;
    for (int i = lane; i < p.d; i += 32) {
      const float x = to_f32(src[i]);
      z[i] = x;
      ss += x * x;
    }
    if (w != nullptr) {
      const float r = rsqrtf(warp_sum(ss) * p.inv_d + p.eps);
      for (int i = lane; i < p.d; i += 32) z[i] = z[i] * r * to_f32(w[i]);
    }
    __syncwarp();
    const int half = p.rot / 2;
    for (int i = lane; i < p.d; i += 32) {
      float o = z[i];
      if (i < p.rot) {
        const float c = p.table_f32 ? static_cast<const float*>(p.cos_t)[tok * p.cos_st + i]
                                    : to_f32(static_cast<const T*>(p.cos_t)[tok * p.cos_st + i]);
        const float s = p.table_f32 ? static_cast<const float*>(p.sin_t)[tok * p.sin_st + i]
                                    : to_f32(static_cast<const T*>(p.sin_t)[tok * p.sin_st + i]);
        o = z[i] * c + (i < half ? -z[i + half] : z[i - half]) * s;
      }
      dst[i] = from_f32<T>(o);
    }
    __syncwarp();
  }
}

}  // namespace tc
