// Rows of a KV cache held in 4 bits: writing (with the step's q/k norm and rotation), reading back, and
// rotating keys where they lie.
//
// A row of D elements is D/2 bytes of codes (element e in byte e/2, the even one in the low half) and
// D/32 pairs (S, z) of the 16-bit type T, one for each group of 32 neighbours. Code c of 0..15 stands for
//   T(S (1 + c/16) + z),     S = T((hi - lo) / 0.9375),  z = T(lo - S)
// with lo and hi the group's extremes: 16 levels from lo to hi, S being 16 steps. In this form the codes are
// the top four mantissa bits of numbers in [1, 2), so that a shift and one logic instruction turn two codes
// into 16-bit floats, and one packed fma turns those into two values: no conversion, no subtraction, one
// rounding. What the offset form costs: z's rounding, at most 2^-9 |z| (bf16), where |z| is about 23 steps for
// data around zero: 0.05 of a step, beside the 0.5 of the code itself.
// Each element takes its nearest level, ties to the even code (quantise8). A group with a NaN or an infinity,
// or whose S or z overflows T (fp16: magnitudes above 20,000), reads back as NaN throughout.
#pragma once

#include <stdint.h>

#include "rope_splice.cuh"  // kMaxLayers, kMaxRopeDim

namespace tc {

constexpr int kI4Group = 32;      // elements that share a scale
constexpr int kI4TileRows = 32;   // rows of a tile-table entry

// Bytes of a row.
__host__ __device__ constexpr int i4_row_bytes(int d) { return d / 2 + d / 8; }

template <typename T>
struct I4;
template <>
struct I4<__nv_bfloat16> {
  static constexpr uint32_t kOne = 0x3F803F80u, kMask = 0x00780078u;  // 1.0 twice; mantissa bits 6..3
  static constexpr int kBit = 3;
  __device__ __forceinline__ static uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
};
template <>
struct I4<__half> {
  static constexpr uint32_t kOne = 0x3C003C00u, kMask = 0x03C003C0u;  // mantissa bits 9..6
  static constexpr int kBit = 6;
  __device__ __forceinline__ static uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
};

// (w & kMask) | kSet as one instruction: written with operators it becomes two.
template <uint32_t kMask, uint32_t kSet>
__device__ __forceinline__ uint32_t mask_set(uint32_t w) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(w), "n"(kMask), "n"(kSet));
  return d;
}

// 1 + c/16 for codes J (low half) and J + 4 (high half) of a word.
template <typename T, int J>
__device__ __forceinline__ uint32_t i4_mant(uint32_t w) {
  constexpr int up = I4<T>::kBit - 4 * J;
  const uint32_t s = up >= 0 ? w << (up >= 0 ? up : 0) : w >> (up >= 0 ? 0 : -up);
  return mask_set<I4<T>::kMask, I4<T>::kOne>(s);
}
__device__ __forceinline__ uint32_t i4_low2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t i4_high2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// The values of a word's 8 codes under its group's (S, z), in order, two a register.
template <typename T>
__device__ __forceinline__ void i4_values(uint32_t w, uint32_t param, uint32_t (&v)[4]) {
  const uint32_t s = i4_low2(param, param), z = i4_high2(param, param);
  const uint32_t p0 = I4<T>::fma2(i4_mant<T, 0>(w), s, z), p1 = I4<T>::fma2(i4_mant<T, 1>(w), s, z);
  const uint32_t p2 = I4<T>::fma2(i4_mant<T, 2>(w), s, z), p3 = I4<T>::fma2(i4_mant<T, 3>(w), s, z);
  v[0] = i4_low2(p0, p1);
  v[1] = i4_low2(p2, p3);
  v[2] = i4_high2(p0, p1);
  v[3] = i4_high2(p2, p3);
}

// The same numbers 1 + c/16, by whichever pipe is free: codes 0 and 1 of a half need no shift, as an fma (on the
// otherwise idle fma pipe) moves them into place: 128 + c and 1024 + c are what a logic instruction makes of code 0; code 1
// (bits 7..4) is c 2^-129 as a bf16 as it stands (subnormal up to 7, linear on through the first binade), and
// 1024 + 16 c as an f16.
template <typename T, int J>
__device__ __forceinline__ uint32_t i4_ones(uint32_t w) {
  constexpr bool bf = I4<T>::kBit == 3;
  if constexpr (J == 0) {
    const uint32_t x = mask_set<0x000f000fu, bf ? 0x43004300u : 0x64006400u>(w);
    return bf ? I4<T>::fma2(x, 0x3d803d80u, 0xc0e0c0e0u)   // x / 16 - 7
              : I4<T>::fma2(x, 0x2c002c00u, 0xd3e0d3e0u);  // x / 16 - 63
  } else if constexpr (J == 1) {
    return bf ? I4<T>::fma2(w & 0x00f000f0u, 0x7e007e00u, 0x3f803f80u)                    // x 2^125 + 1
              : I4<T>::fma2(mask_set<0x00f000f0u, 0x64006400u>(w), 0x1c001c00u, 0xc200c200u);  // x / 256 - 3
  } else {
    return i4_mant<T, J>(w);
  }
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <typename X>
__device__ __forceinline__ void load8(const X* p, float (&x)[8]) {
  constexpr int V = 16 / sizeof(X);
#pragma unroll
  for (int a = 0; a < 8; a += V) {
    const uint4 u = *reinterpret_cast<const uint4*>(p + a);
    X h[V];
    memcpy(h, &u, 16);
#pragma unroll
    for (int e = 0; e < V; ++e) x[a + e] = to_f32(h[e]);
  }
}

// Codes of this lane's 8 elements (values of T) of a group that four neighbouring lanes (aligned to 4) hold, and
// the group's (S, z). Every lane of the warp calls it.
// The nearest level is found through the reciprocal of a step, and decided by the exact distance from it: many
// elements of coarse 16-bit data lie on a border between two levels, where the reciprocal's error would show.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& param) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = min_nan(lo, x[e]);
    hi = max_nan(hi, x[e]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const T st = from_f32<T>(__fdiv_rn(__fsub_rn(hi, lo), 0.9375f));
  float s = to_f32(st);
  const T zt = from_f32<T>(__fsub_rn(lo, s));
  float z = to_f32(zt);
  uint16_t sb, zb;
  memcpy(&sb, &st, 2);
  memcpy(&zb, &zt, 2);
  if (fabsf(z) == INFINITY) sb = 0x7fffu;  // NaN: a finite S would leave infinities that look like data
  param = (uint32_t)sb | ((uint32_t)zb << 16);
  // (bf16) where the reciprocal or x - z would overflow: the same levels, a power of two larger or smaller
  const float by = s < 1e-30f ? 18446744073709551616.f : s > 1e30f ? 1.f / 18446744073709551616.f : 1.f;
  s *= by;
  z *= by;
  const float r = s > 0.f ? __fdividef(16.f, s) : 0.f;
  const float step = 0.0625f * s, half = 0.03125f * s;
  constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: adding it leaves a whole number in the low bits
  uint32_t word = 0;
#pragma unroll
  for (int e = 7; e >= 0; --e) {
    const float t = fmaf(x[e], by, -z);  // by 1: x - z
    const float y = fmaf(t, r, kWhole);
    float k = y - kWhole;  // 16 + code, or its neighbour near a border
    const float off = fmaf(-k, step, t);
    const bool odd = __float_as_uint(y) & 1u;
    if (odd ? off >= half : off > half) k += 1.f;
    if (odd ? off <= -half : off < -half) k -= 1.f;
    k = fminf(fmaxf(k, 16.f), 31.f);
    word = (word << 4) | (__float_as_uint(k + kWhole) & 15u);
  }
  return word;
}

// ------------------------------------------------------------------------------------------------ writing
struct Int4AppendParams {
  const void* q;  // [hq][t][d] with element strides (q_sh, q_st), or null
  const void* k;  // [hkv][t][d]
  const void* v;
  void* q_out;
  uint8_t* kp;  // this layer's pools, strides in bytes
  uint8_t* vp;
  const void* q_w;  // norm weights [d] of T, or null
  const void* k_w;
  const void* cos_t;  // [t][rot] of T or fp32, row strides cos_st / sin_st; rot = 0: no rotation
  const void* sin_t;
  int hq, hkv, rot;
  int64_t t;
  int64_t q_sh, q_st, k_sh, k_st, v_sh, v_st, qo_sh, qo_st, cos_st, sin_st;
  int64_t page_rows, num_pages;
  int64_t s_page, s_h, s_row;
  const int32_t* slots;  // [t][2]: page, row
  float eps, inv_d;
};

// A lane holds 8 neighbouring elements of a row, so a row is D/8 lanes, a group four of them, and a warp 256/D
// heads of one token, all of them queries, keys or values. The elements that an element is rotated with are
// loaded a second time (they are in L1: another lane of the row holds them). Arithmetic of the rotation as
// elementary fp32 operations give it (no contraction), then one rounding to T, whose result is quantised (keys)
// or stored (queries).
// kVec: rows, tables and weights on 16-byte boundaries, rot a multiple of 16.
template <typename T, typename TT, int D, bool kVec>
__global__ void __launch_bounds__(256) int4_append_kernel(const __grid_constant__ Int4AppendParams p) {
  constexpr int L = D / 8;
  constexpr int RW = 32 / L;
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, c = lane % L, i0 = 8 * c;
  const int q_groups = (p.hq + RW - 1) / RW, kv_groups = (p.hkv + RW - 1) / RW;
  const int groups = q_groups + 2 * kv_groups;
  const int64_t step = (int64_t)gridDim.x * 8;
  for (int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); task < p.t * groups; task += step) {
    const int64_t tok = task / groups;
    int grp = (int)(task - tok * groups);
    const bool isq = grp < q_groups, isv = grp >= q_groups + kv_groups;
    grp -= isq ? 0 : isv ? q_groups + kv_groups : q_groups;
    const int h = grp * RW + lane / L;
    bool use = h < (isq ? p.hq : p.hkv);
    const T* src = isq   ? static_cast<const T*>(p.q) + h * p.q_sh + tok * p.q_st
                   : isv ? static_cast<const T*>(p.v) + h * p.v_sh + tok * p.v_st
                         : static_cast<const T*>(p.k) + h * p.k_sh + tok * p.k_st;
    uint8_t* row = nullptr;
    if (!isq) {
      const int64_t page = p.slots[2 * tok], r = p.slots[2 * tok + 1];
      use = use && page >= 0 && page < p.num_pages && r >= 0 && r < p.page_rows;
      row = (isv ? p.vp : p.kp) + page * p.s_page + h * p.s_h + r * p.s_row;
    }
    float x[8], o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (use) {
      if constexpr (kVec) {
        load8(src + i0, x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_f32(src[i0 + e]);
      }
    }
    if (isv) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = x[e];
    } else {
      const T* w = static_cast<const T*>(isq ? p.q_w : p.k_w);
      const int half = p.rot / 2;
      float y[8], cs[8], sn[8], r = 1.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = sn[e] = 0.f;
        cs[e] = 1.f;
      }
      const TT* ct = static_cast<const TT*>(p.cos_t) + tok * p.cos_st;
      const TT* st = static_cast<const TT*>(p.sin_t) + tok * p.sin_st;
      // the partner of element i: i + half in the first half, i - half in the second
      if constexpr (kVec) {
        if (use && i0 < p.rot) {
          load8(src + (i0 < half ? i0 + half : i0 - half), y);
          load8(ct + i0, cs);
          load8(st + i0, sn);
        }
      } else {
        if (use) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = i0 + e;
            if (i < p.rot) {
              y[e] = to_f32(src[i < half ? i + half : i - half]);
              cs[e] = to_f32(ct[i]);
              sn[e] = to_f32(st[i]);
            }
          }
        }
      }
      if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
        for (int a = 1; a < L; a <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, a);
        r = rsqrtf(ss * p.inv_d + p.eps);
        float wx[8], wy[8];
        if constexpr (kVec) {
          load8(w + i0, wx);
          load8(w + (i0 >= p.rot ? i0 : i0 < half ? i0 + half : i0 - half), wy);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = i0 + e;
            wx[e] = to_f32(w[i]);
            wy[e] = to_f32(w[i >= p.rot ? i : i < half ? i + half : i - half]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = x[e] * r * wx[e];
          y[e] = y[e] * r * wy[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = i0 + e;
        const float turned = __fadd_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(i < half ? -y[e] : y[e], sn[e]));
        o[e] = to_f32(from_f32<T>(i < p.rot ? turned : x[e]));
      }
    }
    if (isq) {
      if (use) {
        T* out = static_cast<T*>(p.q_out) + h * p.qo_sh + tok * p.qo_st + i0;
        if constexpr (kVec) {
          *reinterpret_cast<uint4*>(out) = make_uint4(Mma<T>::pack(o[0], o[1]), Mma<T>::pack(o[2], o[3]),
                                                      Mma<T>::pack(o[4], o[5]), Mma<T>::pack(o[6], o[7]));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) out[e] = from_f32<T>(o[e]);
        }
      }
      continue;
    }
    uint32_t param;
    const uint32_t word = quantise8<T>(o, param);
    if (use) {
      *reinterpret_cast<uint32_t*>(row + 4 * c) = word;
      if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(row + D / 2 + c) = param;
    }
  }
}

// ------------------------------------------------------------------------------------------------ reading back
struct Int4GatherParams {
  const uint8_t* kp;  // pools, strides in bytes
  const uint8_t* vp;
  void* k_out;  // [hkv][n][d] of T, element strides out_sh, out_sn
  void* v_out;
  int hkv;
  int64_t n;
  int64_t out_sh, out_sn;
  int64_t page_rows, num_pages;
  int64_t s_page, s_h, s_row;
  const int32_t* tiles;  // [n_tiles][4]: page, first row, rows, position of the first row
  int64_t n_tiles;
};

// A warp per (tile, head): a lane turns one word of a key row and of the value row beside it into 16 bytes
// each, a row being D/8 lanes.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_gather_kernel(const __grid_constant__ Int4GatherParams p) {
  constexpr int L = D / 8;
  constexpr int RW = 32 / L;  // rows a warp takes at a time
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, c = lane % L;
  const int64_t tasks = p.n_tiles * p.hkv;
  for (int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += (int64_t)gridDim.x * 8) {
    const int64_t tile = task / p.hkv;
    const int h = (int)(task - tile * p.hkv);
    const int4 te = *reinterpret_cast<const int4*>(p.tiles + 4 * tile);
    if (te.x < 0 || te.x >= p.num_pages) continue;
    const int rows = te.z < kI4TileRows ? te.z : kI4TileRows;
    const int64_t base = te.x * p.s_page + h * p.s_h;
#pragma unroll 4
    for (int r = lane / L; r < rows; r += RW) {
      const int64_t pr = (int64_t)te.y + r, pos = (int64_t)te.w + r;
      if (pr < 0 || pr >= p.page_rows || pos < 0 || pos >= p.n) continue;
      const uint8_t* kr = p.kp + base + pr * p.s_row;
      const uint8_t* vr = p.vp + base + pr * p.s_row;
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(kr + 4 * c);
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(vr + 4 * c);
      const uint32_t kq = *reinterpret_cast<const uint32_t*>(kr + D / 2 + 4 * (c / 4));
      const uint32_t vq = *reinterpret_cast<const uint32_t*>(vr + D / 2 + 4 * (c / 4));
      uint32_t k4[4], v4[4];
      i4_values<T>(kw, kq, k4);
      i4_values<T>(vw, vq, v4);
      const int64_t o = h * p.out_sh + pos * p.out_sn + 8 * c;
      *reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + o) = make_uint4(k4[0], k4[1], k4[2], k4[3]);
      *reinterpret_cast<uint4*>(static_cast<T*>(p.v_out) + o) = make_uint4(v4[0], v4[1], v4[2], v4[3]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ rotating keys
struct Int4RotateParams {
  uint8_t* kp[kMaxLayers];  // key pool of each layer, strides in bytes
  int layers, hkv;
  int64_t page_rows, num_pages;
  int64_t s_page, s_h, s_row;
  const int32_t* tiles;  // [n_tiles][tile_cols]: page, first row, rows, ...
  int tile_cols;
  int64_t n_tiles;
  float cs[kMaxRopeDim];  // cos of the D/2 angles, then sin
};

// Keys re-rotated in place by one angle a frequency (the splice of threadcut/kv.py:28-41 over 4-bit rows): a row's
// values, rotated in fp32 as the 16-bit splice rotates them, rounded to T and quantised again. A warp per
// (layer, tile, head); a row is D/8 lanes, the partner's values come from the lane half a row away.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_rotate_kernel(const __grid_constant__ Int4RotateParams p) {
  constexpr int L = D / 8;
  constexpr int RW = 32 / L;
  const int lane = threadIdx.x & 31, c = lane % L;
  const bool first = c < L / 2;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = 8 * (c % (L / 2)) + e;
    cs[e] = p.cs[i];
    sn[e] = first ? -p.cs[D / 2 + i] : p.cs[D / 2 + i];
  }
  pdl_launch();
  pdl_wait();
  const int64_t per_layer = p.n_tiles * p.hkv;
  const int64_t tasks = p.layers * per_layer;
  for (int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += (int64_t)gridDim.x * 8) {
    const int layer = (int)(task / per_layer);
    const int64_t th = task - layer * per_layer;
    const int64_t tile = th / p.hkv;
    const int h = (int)(th - tile * p.hkv);
    const int32_t* te = p.tiles + p.tile_cols * tile;
    const int64_t page = te[0], r0 = te[1];
    const int rows = te[2] < kI4TileRows ? te[2] : kI4TileRows;
    if (page < 0 || page >= p.num_pages) continue;
    uint8_t* base = p.kp[layer] + page * p.s_page + h * p.s_h;
#pragma unroll 2
    for (int rb = 0; rb < rows; rb += RW) {  // the whole warp: the lanes exchange values
      const int64_t pr = r0 + rb + lane / L;
      const bool use = rb + lane / L < rows && pr >= 0 && pr < p.page_rows;
      uint8_t* row = base + pr * p.s_row;
      uint32_t v[4] = {0u, 0u, 0u, 0u}, u[4];
      if (use)
        i4_values<T>(*reinterpret_cast<const uint32_t*>(row + 4 * c),
                     *reinterpret_cast<const uint32_t*>(row + D / 2 + 4 * (c / 4)), v);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = __shfl_xor_sync(0xffffffffu, v[i], L / 2);
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = e & 1 ? Mma<T>::hi(v[e / 2]) : Mma<T>::lo(v[e / 2]);
        const float y = e & 1 ? Mma<T>::hi(u[e / 2]) : Mma<T>::lo(u[e / 2]);
        o[e] = to_f32(from_f32<T>(__fadd_rn(__fmul_rn(x, cs[e]), __fmul_rn(y, sn[e]))));
      }
      uint32_t param;
      const uint32_t word = quantise8<T>(o, param);
      // every lane of the row has read it: the exchange above waited for them
      if (use) {
        *reinterpret_cast<uint32_t*>(row + 4 * c) = word;
        if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(row + D / 2 + c) = param;
      }
    }
  }
}

}  // namespace tc
