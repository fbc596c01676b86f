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
  int pairs;  // paged_append_vec_kernel: threads per row, d / (2 * elements in 16 bytes)
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

// Rows of 16-byte chunks (p.pairs, a power of two <= 32, thread pairs of chunks a row): a thread holds a
// chunk and its rotation partner, so a row is p.pairs threads and a warp 32 / p.pairs heads of ONE token,
// whose cos and sin it keeps in registers for kRows rows each. Bytes are the bound; kRows rows are loaded
// before the first is used to keep enough of them in flight.
template <typename T, typename TT, int kRows>
__global__ void __launch_bounds__(256) paged_append_vec_kernel(const __grid_constant__ PagedAppendParams p) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kTabVec = 16 / sizeof(TT);
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int heads = p.hq + 2 * p.hkv;
  const int per_warp = 32 / p.pairs * kRows;  // heads a warp takes
  const int groups = (heads + per_warp - 1) / per_warp;
  const int64_t task = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t tok = task / groups;
  if (tok >= p.t) return;
  const int head0 = (int)(task - tok * groups) * per_warp + lane / p.pairs;
  const int c = lane & (p.pairs - 1);
  const int turned = p.rot / (2 * VEC);  // pairs that rotate; the others pass through side by side
  const bool turns = c < turned;
  const int ia = (turns ? c : 2 * c) * VEC, ib = turns ? ia + p.rot / 2 : ia + VEC;

  const int64_t page = p.slots[2 * tok], row = p.slots[2 * tok + 1];
  const bool slot = page >= 0 && page < p.num_pages && row >= 0 && row < p.page_rows;
  Chunk<T, VEC> a[kRows], b[kRows];
  T* dst[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int hh = head0 + u * (32 / p.pairs);
    const T* src = nullptr;
    dst[u] = nullptr;
    if (hh < p.hq) {
      src = static_cast<const T*>(p.q) + hh * p.q_sh + tok * p.q_st;
      dst[u] = static_cast<T*>(p.q_out) + hh * p.qo_sh + tok * p.qo_st;
    } else if (hh < heads && slot) {
      const bool isv = hh >= p.hq + p.hkv;
      const int h = hh - p.hq - (isv ? p.hkv : 0);
      src = isv ? static_cast<const T*>(p.v) + h * p.v_sh + tok * p.v_st
                : static_cast<const T*>(p.k) + h * p.k_sh + tok * p.k_st;
      dst[u] = static_cast<T*>(isv ? p.vp : p.kp) + page * p.s_page + h * p.s_h + row * p.s_row;
    }
    if (src != nullptr) {
      a[u] = ld_chunk<T, VEC>(src + ia);
      b[u] = ld_chunk<T, VEC>(src + ib);
    } else {
      a[u] = b[u] = Chunk<T, VEC>{};
    }
  }
  float ca[VEC], cb[VEC], sa[VEC], sb[VEC];
  if (turns && head0 < p.hq + p.hkv) {
    const TT* ct = static_cast<const TT*>(p.cos_t) + tok * p.cos_st;
    const TT* st = static_cast<const TT*>(p.sin_t) + tok * p.sin_st;
#pragma unroll
    for (int x = 0; x < VEC; x += kTabVec) {
      const Chunk<TT, kTabVec> t0 = ld_chunk<TT, kTabVec>(ct + ia + x), t1 = ld_chunk<TT, kTabVec>(ct + ib + x);
      const Chunk<TT, kTabVec> t2 = ld_chunk<TT, kTabVec>(st + ia + x), t3 = ld_chunk<TT, kTabVec>(st + ib + x);
#pragma unroll
      for (int e = 0; e < kTabVec && x + e < VEC; ++e) {
        ca[x + e] = to_f32(t0.v[e]);
        cb[x + e] = to_f32(t1.v[e]);
        sa[x + e] = to_f32(t2.v[e]);
        sb[x + e] = to_f32(t3.v[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ca[e] = cb[e] = 1.f;
      sa[e] = sb[e] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int hh = head0 + u * (32 / p.pairs);
    const bool isq = hh < p.hq, isv = hh >= p.hq + p.hkv;
    const T* w = static_cast<const T*>(isq ? p.q_w : p.k_w);
    float xa[VEC], xb[VEC], ss = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      xa[e] = to_f32(a[u].v[e]);
      xb[e] = to_f32(b[u].v[e]);
      ss += xa[e] * xa[e] + xb[e] * xb[e];
    }
    for (int o = p.pairs >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (dst[u] == nullptr) continue;
    if (!isv) {
      if (w != nullptr) {
        const float r = rsqrtf(ss * p.inv_d + p.eps);
        const Chunk<T, VEC> wa = ld_chunk<T, VEC>(w + ia), wb = ld_chunk<T, VEC>(w + ib);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          xa[e] = xa[e] * r * to_f32(wa.v[e]);
          xb[e] = xb[e] * r * to_f32(wb.v[e]);
        }
      }
      if (turns) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float oa = xa[e] * ca[e] - xb[e] * sa[e];
          xb[e] = xb[e] * cb[e] + xa[e] * sb[e];
          xa[e] = oa;
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        a[u].v[e] = from_f32<T>(xa[e]);
        b[u].v[e] = from_f32<T>(xb[e]);
      }
    }
    st_chunk<T, VEC>(dst[u] + ia, a[u]);
    st_chunk<T, VEC>(dst[u] + ib, b[u]);
  }
}

}  // namespace tc
