// A step's queries and keys normalised (optional) and rotated, keys and values written into the slots
// of a paged cache, in one launch: the chain of torch ops in front of tc_paged_write (transformers'
// Qwen3Attention q_norm, k_norm, apply_rotary_pos_emb, then the cache update of threadcut/kv.py:64-77).
//
// Per token and head, x being its d elements:
//   z = x * rsqrt(mean(x^2) + eps) * w                      (with a norm weight; else z = x)
//   out[i] = z[i] cos[i] - z[i + rot/2] sin[i]              i < rot/2
//   out[i] = z[i] cos[i] + z[i - rot/2] sin[i]              rot/2 <= i < rot
//   out[i] = z[i]                                           i >= rot (partial rotation; x[i] itself, to the bit,
//                                                           without a weight)
// in fp32 from the loaded values on, rounded once to T at the store. (The torch chain, and with it
// tc_qk_norm_rope, rounds to T after each op; one rounding is nearer to the formula.)
#pragma once

#include <stdint.h>

namespace tc {

constexpr int kMaxAppendDim = 512;  // head size of the paged append (a warp holds a row in 2 KB of shared memory)

constexpr int kAppendThreads = 128;
constexpr int kAppendRows = 2;  // rows a thread of paged_append_vec_kernel takes

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
      dst[i] = i >= p.rot && w == nullptr ? src[i] : from_f32<T>(o);
    }
    __syncwarp();
  }
}

// A 16-byte chunk as fp32 pairs and back.
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Chunk<T, VEC>& c, float2 (&x)[VEC / 2]) {
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) x[e] = make_float2(to_f32(c.v[2 * e]), to_f32(c.v[2 * e + 1]));
}
template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> narrow(const float2 (&x)[VEC / 2]) {
  Chunk<T, VEC> c;
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w = Mma<T>::pack(x[e].x, x[e].y);
      memcpy(&c.v[2 * e], &w, 4);
    } else {
      c.v[2 * e] = x[e].x;
      c.v[2 * e + 1] = x[e].y;
    }
  }
  return c;
}

// Rows of 16-byte chunks: a thread holds a chunk and its rotation partner, so a row is p.pairs threads (a
// power of two <= 32) and a warp takes 32 / p.pairs heads of ONE token at a time, kRows times: kRows query
// rows a thread, or kRows / 2 keys and the values of the same heads. With the weight w folded into the
// token's cos and sin once,
//   out_a = (r x_a) (w_a cos_a) - (r x_b) (w_b sin_a),   out_b = (r x_b) (w_b cos_b) + (r x_a) (w_a sin_b),
// a row costs three packed operations an output pair beside its conversions.
// Bound by bytes for long chunks, by latency for short ones: resident warps count in both. 16,384 tokens of
// 48 bf16 heads of 128 (411 MB): 2 rows a thread and 7 CTAs an SM (72 registers) 76.7 us, 5.4 TB/s. Before the split
// below: 78.6, with 6 CTAs 81.8, 8 CTAs (spills) 83.7, 4 rows 86.9, 8 rows 102; with the formula's own order of
// operations, unpacked, 106.
// kPartial: rot < d, some threads hold chunks that pass through. Full rotations have a kernel without their branch
// (32 bytes of spills a thread instead of 56): the prompt above takes 76.7 us, with one kernel for both 80.4.
template <typename T, typename TT, bool kPartial>
__global__ void __launch_bounds__(kAppendThreads, 7)
    paged_append_vec_kernel(const __grid_constant__ PagedAppendParams p) {
  constexpr int kRows = kAppendRows;
  static_assert(kRows % 2 == 0, "half of a key/value warp's rows are keys");
  constexpr int VEC = 16 / sizeof(T), P2 = VEC / 2;
  constexpr int kTabVec = 16 / sizeof(TT);
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int step = 32 / p.pairs;  // heads side by side in the warp
  const int q_groups = (p.hq + step * kRows - 1) / (step * kRows);
  const int kv_groups = (p.hkv + step * kRows / 2 - 1) / (step * kRows / 2);
  const int groups = q_groups + kv_groups;
  const uint32_t task = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const uint32_t tok = task / groups;
  if (tok >= p.t) return;
  const int grp = (int)(task - tok * groups);
  const bool isq = grp < q_groups;
  const int c = lane & (p.pairs - 1);
  const int turned = p.rot / (2 * VEC);  // pairs that rotate; the others pass through side by side
  const bool turns = !kPartial || c < turned;
  const int ia = (turns ? c : 2 * c) * VEC, ib = turns ? ia + p.rot / 2 : ia + VEC;

  // ---- the rows: this thread's row u is head h0 + u * step (keys: u < kRows / 2, then their values)
  Chunk<T, VEC> a[kRows], b[kRows];
  T* dst[kRows];
  if (isq) {
    const int h0 = grp * step * kRows + lane / p.pairs;
    const T* src = static_cast<const T*>(p.q) + tok * p.q_st + h0 * p.q_sh;
    T* out = static_cast<T*>(p.q_out) + tok * p.qo_st + h0 * p.qo_sh;
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const bool use = h0 + u * step < p.hq;
      dst[u] = use ? out + u * step * p.qo_sh : nullptr;
      if (use) {
        a[u] = ld_chunk<T, VEC>(src + u * step * p.q_sh + ia);
        b[u] = ld_chunk<T, VEC>(src + u * step * p.q_sh + ib);
      } else {
        a[u] = b[u] = Chunk<T, VEC>{};
      }
    }
  } else {
    const int h0 = (grp - q_groups) * step * (kRows / 2) + lane / p.pairs;
    const int2 slot = *reinterpret_cast<const int2*>(p.slots + 2 * (int64_t)tok);
    const bool in = slot.x >= 0 && slot.x < p.num_pages && slot.y >= 0 && slot.y < p.page_rows;
    const int64_t at = in ? slot.x * p.s_page + slot.y * p.s_row : 0;
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const bool isv = u >= kRows / 2;
      const int h = h0 + (isv ? u - kRows / 2 : u) * step;
      const bool use = in && h < p.hkv;
      dst[u] = use ? static_cast<T*>(isv ? p.vp : p.kp) + at + h * p.s_h : nullptr;
      if (use) {
        const T* src = isv ? static_cast<const T*>(p.v) + tok * p.v_st + h * p.v_sh
                           : static_cast<const T*>(p.k) + tok * p.k_st + h * p.k_sh;
        a[u] = ld_chunk<T, VEC>(src + ia);
        b[u] = ld_chunk<T, VEC>(src + ib);
      } else {
        a[u] = b[u] = Chunk<T, VEC>{};
      }
    }
  }

  // ---- the token's factors
  float2 fac[P2], fas[P2], fbc[P2], fbs[P2];  // of z_a and z_b in out_a, of z_b and z_a in out_b
  const T* w = static_cast<const T*>(isq ? p.q_w : p.k_w);
  if (turns) {
    const TT* ct = static_cast<const TT*>(p.cos_t) + tok * p.cos_st;
    const TT* st = static_cast<const TT*>(p.sin_t) + tok * p.sin_st;
#pragma unroll
    for (int x = 0; x < VEC; x += kTabVec) {
      float2 t0[kTabVec / 2], t1[kTabVec / 2], t2[kTabVec / 2], t3[kTabVec / 2];
      widen<TT, kTabVec>(ld_chunk<TT, kTabVec>(ct + ia + x), t0);
      widen<TT, kTabVec>(ld_chunk<TT, kTabVec>(st + ia + x), t1);
      widen<TT, kTabVec>(ld_chunk<TT, kTabVec>(ct + ib + x), t2);
      widen<TT, kTabVec>(ld_chunk<TT, kTabVec>(st + ib + x), t3);
#pragma unroll
      for (int e = 0; e < kTabVec / 2; ++e) {
        fac[x / 2 + e] = t0[e];
        fas[x / 2 + e] = make_float2(-t1[e].x, -t1[e].y);
        fbc[x / 2 + e] = t2[e];
        fbs[x / 2 + e] = t3[e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < P2; ++e) {
      fac[e] = fbc[e] = make_float2(1.f, 1.f);
      fas[e] = fbs[e] = make_float2(0.f, 0.f);
    }
  }
  if (w != nullptr) {
    float2 wa[P2], wb[P2];
    widen<T, VEC>(ld_chunk<T, VEC>(w + ia), wa);
    widen<T, VEC>(ld_chunk<T, VEC>(w + ib), wb);
#pragma unroll
    for (int e = 0; e < P2; ++e) {
      fac[e] = fmul2(fac[e], wa[e]);
      fas[e] = fmul2(fas[e], wb[e]);
      fbc[e] = fmul2(fbc[e], wb[e]);
      fbs[e] = fmul2(fbs[e], wa[e]);
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    // Elements that pass through are not multiplied with their chunk's neighbour (0 * inf is NaN); without a
    // weight they stay as they were loaded.
    if ((isq || u < kRows / 2) && (turns || w != nullptr)) {
      float2 xa[P2], xb[P2];
      widen<T, VEC>(a[u], xa);
      widen<T, VEC>(b[u], xb);
      if (w != nullptr) {
        float2 s2 = fmul2(xa[0], xa[0]);
#pragma unroll
        for (int e = 1; e < P2; ++e) s2 = ffma2(xa[e], xa[e], s2);
#pragma unroll
        for (int e = 0; e < P2; ++e) s2 = ffma2(xb[e], xb[e], s2);
        float ss = s2.x + s2.y;
        for (int o = p.pairs >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(ss * p.inv_d + p.eps);
        const float2 r2 = make_float2(r, r);
#pragma unroll
        for (int e = 0; e < P2; ++e) {
          xa[e] = fmul2(xa[e], r2);
          xb[e] = fmul2(xb[e], r2);
        }
      }
      if (turns) {
#pragma unroll
        for (int e = 0; e < P2; ++e) {
          const float2 oa = ffma2(xa[e], fac[e], fmul2(xb[e], fas[e]));
          xb[e] = ffma2(xb[e], fbc[e], fmul2(xa[e], fbs[e]));
          xa[e] = oa;
        }
      } else {
#pragma unroll
        for (int e = 0; e < P2; ++e) {
          xa[e] = fmul2(xa[e], fac[e]);
          xb[e] = fmul2(xb[e], fbc[e]);
        }
      }
      a[u] = narrow<T, VEC>(xa);
      b[u] = narrow<T, VEC>(xb);
    }
    if (dst[u] != nullptr) {
      st_chunk<T, VEC>(dst[u] + ia, a[u]);
      st_chunk<T, VEC>(dst[u] + ib, b[u]);
    }
  }
}

}  // namespace tc
