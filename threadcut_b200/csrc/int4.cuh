// Rows of a KV cache held in 4 bits: writing (with the step's q/k norm and rotation), reading back, and
// rotating keys where they lie.
//
// A row of D elements is D/2 bytes of codes (element e in byte e/2, the even one in the low half) and
// D/32 pairs (S, z) of the 16-bit type T, one for each group of 32 neighbours. Code c of 0..15 stands for
//   T(S (1 + c/16) + z),     S = T((hi - lo) / 0.9375),  z = T(lo - S)
// with lo and hi the group's extremes: 16 levels from lo to hi, S being 16 steps. In this form the codes are
// the top four mantissa bits of numbers in [1, 2), so that a shift and one logic instruction turn two codes
// into 16-bit floats, and one packed fma turns those into two values: no conversion, no subtraction, one
// rounding. What the offset form costs: z's rounding, at most 2^-8 |z| (bf16), where |z| is about 23 steps for
// data around zero: 0.09 of a step, beside the 0.5 of the code itself.
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
  __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {  // NaN if either is
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  __device__ __forceinline__ static uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
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
  __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  __device__ __forceinline__ static uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
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

// Two products, each rounded: an fma with -0, which is not merged with a sum that follows it, as packed products are. (nz is -0
// from memory: as a constant it would make them products again.)
__device__ __forceinline__ float2 product2(float2 a, float2 b, float2 nz) { return ffma2(a, b, nz); }

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

// x / 0.9375, correctly rounded: a product with the rounded reciprocal, corrected by its exact remainder (Markstein 1990).
__device__ __forceinline__ float by_15_16(float x) {
  constexpr float kUnit = 16.f / 15.f;
  const float q = x * kUnit;
  return fmaf(fmaf(-q, 0.9375f, x), kUnit, q);
}

// 16/S (NaN for an S of 0 or too small), and where among the levels zero lies, -16 z/S - 16.
__device__ __forceinline__ void i4_line(float s, float z, float& r, float& c) {
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0.0625f * s));
  r = fmaf(r, fmaf(-0.0625f * s, r, 1.f), r);
  c = fmaf(-z, r, -16.f);
}
constexpr float kI4Whole = 12582912.f;  // 1.5 * 2^23: adding it leaves a whole number in the low bits
constexpr float kI4Snap = 192.f;        // 1.5 * 2^7: adding it leaves multiples of 2^-16
constexpr float kI4Far = 64.f;          // offsets from which on zero is far outside the levels
// The half next to c, + kI4Snap.
__device__ __forceinline__ float i4_tie(float c) {
  return __fsub_rn(__fadd_rn(c + 0.5f, kI4Whole), kI4Whole) + (kI4Snap - 0.5f);
}

// quantise8 for a warp with groups that its usual way is not for; w0 to w3: this lane's elements (pairs of T).
// Where S is in order and nothing came out on a border near zero, the usual way again, but from x - z for groups far from zero, and
// with a clamp; x - z is exact there.
// Else any group, whatever S and z are (not finite: some codes): a level by an approximate reciprocal, off by one at most and only
// beside a border, then the sign of x - z - S h against the borders h around it: d = x - z rounded, its error exactly (Knuth's
// two-sum), and d - S h by one fma, which is 0 or larger than that error, as it is a multiple of d's last bit. A bf16 S that x - z would
// overflow with is taken a fourth of (exact in fp32).
// A function of its own, as it is rare and takes registers and instruction cache where it is inlined: with a costlier test for
// it than there is now, 49,152 keys of 8 heads of 128 were rotated in 42 us so, 43 with this loop inlined, 49 unrolled. The same keys
// far from zero for their spread (8 times) take 60 us, 117 with the comparisons for all such groups.
template <typename T>
__device__ __noinline__ uint32_t quantise8_rare(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, float s, float z) {
  float r, c;
  i4_line(s, z, r, c);
  const bool far = !(fabsf(c) < kI4Far), flat = s == 0.f;
  const float from = far ? z : 0.f, c0 = far ? -16.f : c, tie = far ? 0.f : i4_tie(c);
  bool usual = flat || fabsf(c) < INFINITY;
  uint32_t codes = 0u;
  {
    const uint32_t w[4] = {w0, w1, w2, w3};
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      const float x = (e & 1 ? Mma<T>::hi(w[e / 2]) : Mma<T>::lo(w[e / 2])) - from;
      const float t = __fadd_rn(fminf(fmaxf(fmaf(x, r, c0), 0.f), 15.f), kI4Snap);
      usual = usual && (flat || t != tie);
      codes = codes * 16u + __float_as_uint(__fadd_rn(t, kI4Whole - kI4Snap));
    }
  }
  if (__all_sync(0xffffffffu, usual)) return flat ? 0u : codes - 0x4b400000u * 0x11111111u;
  float by = 1.f, up = 1.f;
  if constexpr (I4<T>::kBit == 3) {
    by = s > 1e30f ? 0.25f : 1.f;
    up = s > 1e30f ? 1.f / 18446744073709551616.f : s < 1e-30f ? 18446744073709551616.f : 1.f;  // 2^64: for the reciprocal
    s *= by;
    z *= by;
  }
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s * up));
  r = s > 0.f ? 16.f * r : 0.f;
  codes = 0u;
#pragma unroll 1
  for (int e = 0; e < 32; e += 4) {
    const float x = Mma<T>::lo(w0) * by;
    w0 = __funnelshift_r(w0, w1, 16);
    w1 = __funnelshift_r(w1, w2, 16);
    w2 = __funnelshift_r(w2, w3, 16);
    w3 >>= 16;
    const float d = __fsub_rn(x, z), back = __fsub_rn(d, x);
    const float err = __fsub_rn(__fsub_rn(x, __fsub_rn(d, back)), __fadd_rn(z, back));
    c = fminf(fmaxf(rintf(fmaf(d * up, r, -16.f)), 0.f), 15.f);  // NaN gives 0
    float below = fmaf(-s, (c + 15.5f) * 0.0625f, d), above = fmaf(-s, (c + 16.5f) * 0.0625f, d);
    below = below == 0.f ? err : below;
    above = above == 0.f ? err : above;
    int code = (int)c;
    const bool odd = code & 1;  // on a border, the even level
    code += (above > 0.f || (above == 0.f && odd)) - (below < 0.f || (below == 0.f && odd));
    codes |= (uint32_t)(code < 0 ? 0 : code > 15 ? 15 : code) << e;
  }
  return codes;
}

// Codes of this lane's 8 elements (w: pairs of T) of a group that four neighbouring lanes (aligned to 4) hold, and the
// group's (S, z). Every lane of the warp calls it.
// The extremes as packed maxima and minima. A code is x (16/S) + (-16 z/S - 16) rounded. Many elements of coarse 16-bit data
// lie exactly on a border between two levels, and the even one is theirs. That sum is off by at most 4.3e-6: 32 * 2^-24 from
// 16/S (one Newton step behind the approximate reciprocal), 2^-19 from the offset's rounding while it is below 64, 2^-21 from
// its own. So it is first rounded to a multiple of 2^-16, which a border is (half of one is 7.6e-6), then to a whole number, both
// by adding constants, two elements an instruction; the codes are collected as the floats' bits, whose exponents add up to a
// constant. No clamp: below that offset z's and S's roundings move an end by 0.37 of a level at most (z's, 16 * 2^-8 |z|/S in
// bf16 with |z| < 5 S, by 0.31; S's by 0.06).
// An element beside a border but less than 2^-16 of a level from it may come out as on it. With p significant bits (8 or 11),
// z and the borders S (33 + 2 j) / 32 + z are multiples of 2^-(p+5) S, so that such an element's last bit must be finer:
// |x| < 2^(p-20) S, and the border lies as near to zero. That is one border at most, and the offset, which is zero's own place
// among the levels, is within 2^(p-16) of its number. Groups with such an offset look whether anything came out on that border.
// Warps where something did, and those with an offset of 64 or more (values many times their spread, with coarse last bits
// therefore), an S too small for the reciprocal, or a NaN, take quantise8_rare. Every way gives the nearest level, so that a row's
// bytes are the same in any company.
// 49,152 keys of 8 heads of 128 are rotated in 37 us in bf16 and 39 in fp16; 37 and 37 without that test, 47 and 51 with the
// elements near such a border compared with it and both ways inlined.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&w)[4], uint32_t& param) {
  constexpr bool bf = I4<T>::kBit == 3;
  const uint32_t hi2 = I4<T>::max2(I4<T>::max2(w[0], w[1]), I4<T>::max2(w[2], w[3]));
  const uint32_t lo2 = I4<T>::min2(I4<T>::min2(w[0], w[1]), I4<T>::min2(w[2], w[3])) ^ 0x80008000u;
  uint32_t m = I4<T>::max2(i4_low2(hi2, lo2), i4_high2(hi2, lo2));  // (largest, largest negative)
  m = I4<T>::max2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = I4<T>::max2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const float hi = Mma<T>::lo(m), lo = -Mma<T>::hi(m);
  const uint32_t st = Mma<T>::pack(by_15_16(__fsub_rn(hi, lo)), 0.f);
  const float s = Mma<T>::lo(st);
  param = Mma<T>::pack(s, __fsub_rn(lo, s));
  const float z = Mma<T>::hi(param);
  float r, c;
  i4_line(s, z, r, c);
  float2 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t[i] = fadd2(ffma2(make_float2(Mma<T>::lo(w[i]), Mma<T>::hi(w[i])), make_float2(r, r), make_float2(c, c)),
                 make_float2(kI4Snap, kI4Snap));
  const bool flat = s == 0.f;  // one value throughout, as of lanes without a head or row of their own
  bool sure = flat || fabsf(c) < kI4Far;  // (false for NaN too)
  // whether c, to a multiple of 2^(p-18), is within 2^(p-16) of a half: its fraction from 1/2 - 2^(p-16) on, as bits
  constexpr float kFine = bf ? 12288.f : 49152.f;       // 1.5 * 2^13 or 2^15: adding it leaves multiples of 2^-10 or 2^-8
  constexpr float kFrom = bf ? 0.49609375f : 0.46875f;  // 1/2 - 2^-8 or - 2^-5
  constexpr uint32_t kUnit = bf ? 1024 : 256, kWide = bf ? 8 : 16;
  if ((__float_as_uint(c + (kFine - kFrom)) & (kUnit - 1)) <= kWide) {
    const float tie = i4_tie(c);
#pragma unroll
    for (int i = 0; i < 4; ++i) sure = sure && t[i].x != tie && t[i].y != tie;
  }
  if (__all_sync(0xffffffffu, sure)) {
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      const float2 n = fadd2(t[i], make_float2(kI4Whole - kI4Snap, kI4Whole - kI4Snap));
      codes = (codes * 16u + __float_as_uint(n.y)) * 16u + __float_as_uint(n.x);
    }
    return flat ? 0u : codes - 0x4b400000u * 0x11111111u;  // the bits of kI4Whole, as often as they came in
  }
  if (fabsf(z) == INFINITY) param |= 0x7fffu;  // S NaN: a finite S would leave infinities that look like data
  return quantise8_rare<T>(w[0], w[1], w[2], w[3], s, z);
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
  float minus_zero;  // -0
  int table_f32;
};

template <typename T>
__device__ __forceinline__ float table_at(const void* t, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(t)[i] : to_f32(static_cast<const T*>(t)[i]);
}

// Rotation of 8 elements (fp32, first element i0) with the 8 they are paired with, by elementary fp32 operations (no
// contraction), rounded to T; elements from rot on pass through.
template <typename T>
__device__ __forceinline__ void rotate8(const float (&x)[8], const float (&y)[8], const float (&cs)[8], const float (&sn)[8],
                                        int i0, int rot, uint32_t (&w)[4]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float o[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = i0 + e + u;
      const float a = __fmul_rn(x[e + u], cs[e + u]), b = __fmul_rn(y[e + u], sn[e + u]);
      o[u] = i >= rot ? x[e + u] : i < rot / 2 ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
    w[e / 2] = Mma<T>::pack(o[0], o[1]);
  }
}

// Any strides, alignment and rot: a lane holds 8 neighbouring elements of a row, loaded one by one, so a row is D/8 lanes and a
// group four of them; a warp takes 256/D heads of one token, all of them queries, keys or values.
template <typename T, int D>
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
    const int rot = isv ? 0 : p.rot;
    const T* w = static_cast<const T*>(isq ? p.q_w : isv ? nullptr : p.k_w);
    float x[8], y[8], cs[8], sn[8], ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = i0 + e;
      const bool turns = use && i < rot;
      x[e] = use ? to_f32(src[i]) : 0.f;
      y[e] = turns ? to_f32(src[i < rot / 2 ? i + rot / 2 : i - rot / 2]) : 0.f;
      cs[e] = turns ? table_at<T>(p.cos_t, p.table_f32, tok * p.cos_st + i) : 0.f;
      sn[e] = turns ? table_at<T>(p.sin_t, p.table_f32, tok * p.sin_st + i) : 0.f;
      ss += x[e] * x[e];
    }
    if (w != nullptr) {
#pragma unroll
      for (int a = 1; a < L; a <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, a);
      const float r = rsqrtf(ss * p.inv_d + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = i0 + e;
        x[e] = x[e] * r * to_f32(w[i]);
        if (i < rot) y[e] = y[e] * r * to_f32(w[i < rot / 2 ? i + rot / 2 : i - rot / 2]);
      }
    }
    uint32_t o[4];
    rotate8<T>(x, y, cs, sn, i0, rot, o);
    if (isq) {
      if (use) {
        T v[8];
        memcpy(v, o, 16);
        T* out = static_cast<T*>(p.q_out) + h * p.qo_sh + tok * p.qo_st + i0;
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = v[e];
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

// Rows, tables and weights on 16-byte boundaries, rot a multiple of 16: the same with 16-byte accesses. A warp stays with its
// heads (256/D times U of them, queries, keys or values) and goes through tokens; a lane has the same 8 elements of U heads,
// for which it converts a token's cos and sin once. The elements that it rotates them with are loaded a second time (they are
// in L1: another lane of the row holds them). A 16,384-token prompt of 32 query and 8 KV heads of 128: 69 us (5.3 TB/s); half as
// many heads a lane 87, one CTA an SM less 83, the next token's rows loaded ahead 82, both elements of a pair in one lane 86:
// each has fewer bytes in flight or fewer warps.
// kKind: 0 queries, 1 keys, 2 values. kNorm: with a norm weight.
template <typename T, int D, int U, int kKind, bool kNorm>
__device__ __forceinline__ void append_tokens(const Int4AppendParams& p, int grp, uint32_t tok0, uint32_t step) {
  constexpr int L = D / 8;
  constexpr int RW = 32 / L;
  const int lane = threadIdx.x & 31, c = lane % L, i0 = 8 * c;
  const int h0 = grp * RW * U + lane / L, heads = kKind == 0 ? p.hq : p.hkv;
  const int64_t sh = kKind == 0 ? p.q_sh : kKind == 1 ? p.k_sh : p.v_sh;
  const int64_t st = kKind == 0 ? p.q_st : kKind == 1 ? p.k_st : p.v_st;
  const T* src0 = static_cast<const T*>(kKind == 0 ? p.q : kKind == 1 ? p.k : p.v) + h0 * sh + i0;
  const bool turns = kKind < 2 && i0 < p.rot;
  const bool first = i0 < p.rot / 2;
  const int other = turns ? (first ? p.rot / 2 : -(p.rot / 2)) : 0;  // where its elements' partners are
  const T* w = static_cast<const T*>(kKind == 0 ? p.q_w : p.k_w);
  const float2 nz = make_float2(p.minus_zero, p.minus_zero);
  for (uint32_t tok = tok0; tok < p.t; tok += step) {
    const T* src = src0 + tok * st;
    uint4 a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
      if (h0 + u * RW < heads) {
        a[u] = *reinterpret_cast<const uint4*>(src + u * RW * sh);
        if (turns) b[u] = *reinterpret_cast<const uint4*>(src + u * RW * sh + other);
      }
    }
    uint8_t* row = nullptr;
    if constexpr (kKind > 0) {
      const int2 slot = *reinterpret_cast<const int2*>(p.slots + 2 * (int64_t)tok);
      if (slot.x >= 0 && slot.x < p.num_pages && slot.y >= 0 && slot.y < p.page_rows)
        row = (kKind == 1 ? p.kp : p.vp) + slot.x * p.s_page + slot.y * p.s_row + h0 * p.s_h;
    }
    float2 cs[4], sn[4];
    if constexpr (kKind < 2) {
      if (turns) {
        float x[8], y[8];
        if (p.table_f32) {
          load8(static_cast<const float*>(p.cos_t) + tok * p.cos_st + i0, x);
          load8(static_cast<const float*>(p.sin_t) + tok * p.sin_st + i0, y);
        } else {
          load8(static_cast<const T*>(p.cos_t) + tok * p.cos_st + i0, x);
          load8(static_cast<const T*>(p.sin_t) + tok * p.sin_st + i0, y);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cs[e] = make_float2(x[2 * e], x[2 * e + 1]);
          sn[e] = first ? make_float2(-y[2 * e], -y[2 * e + 1]) : make_float2(y[2 * e], y[2 * e + 1]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t o[4] = {a[u].x, a[u].y, a[u].z, a[u].w};
      if constexpr (kKind < 2) {
        const uint32_t q[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
        float2 x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = make_float2(Mma<T>::lo(o[e]), Mma<T>::hi(o[e]));
          y[e] = make_float2(Mma<T>::lo(q[e]), Mma<T>::hi(q[e]));
        }
        if constexpr (kNorm) {
          float2 s2 = fmul2(x[0], x[0]);
#pragma unroll
          for (int e = 1; e < 4; ++e) s2 = ffma2(x[e], x[e], s2);
          float ss = s2.x + s2.y;
#pragma unroll
          for (int i = 1; i < L; i <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, i);
          const float r = rsqrtf(ss * p.inv_d + p.eps);
          float wx[8], wy[8];
          load8(w + i0, wx);
          load8(w + i0 + other, wy);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = fmul2(fmul2(x[e], make_float2(r, r)), make_float2(wx[2 * e], wx[2 * e + 1]));
            y[e] = fmul2(fmul2(y[e], make_float2(r, r)), make_float2(wy[2 * e], wy[2 * e + 1]));
            if (!turns) o[e] = Mma<T>::pack(x[e].x, x[e].y);
          }
        }
        if (turns) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 r = fadd2(product2(x[e], cs[e], nz), product2(y[e], sn[e], nz));
            o[e] = Mma<T>::pack(r.x, r.y);
          }
        }
      }
      if constexpr (kKind == 0) {
        if (h0 + u * RW < heads)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + tok * p.qo_st + (h0 + u * RW) * p.qo_sh + i0) =
              make_uint4(o[0], o[1], o[2], o[3]);
      } else {
        uint32_t param;
        const uint32_t word = quantise8<T>(o, param);
        if (row != nullptr && h0 + u * RW < heads) {
          uint8_t* at = row + u * RW * p.s_h;
          *reinterpret_cast<uint32_t*>(at + 4 * c) = word;
          if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(at + D / 2 + c) = param;
        }
      }
    }
  }
}

// Keys and values take about twice the instructions of queries, so a warp has half as many of them.
__host__ __device__ constexpr int i4_kv_heads(int u) { return u > 1 ? u / 2 : 1; }
// Resident CTAs an SM: what spills nothing.
__host__ __device__ constexpr int i4_append_ctas(int u, bool norm) { return u > 1 && norm ? 2 : 3; }

template <typename T, int D, int U, bool kNorm>
__global__ void __launch_bounds__(256, i4_append_ctas(U, kNorm)) int4_append_vec_kernel(const __grid_constant__ Int4AppendParams p) {
  constexpr int KU = i4_kv_heads(U);
  constexpr int QW = 256 / D * U, KW = 256 / D * KU;
  pdl_launch();
  pdl_wait();
  const int q_groups = (p.hq + QW - 1) / QW, kv_groups = (p.hkv + KW - 1) / KW;
  const uint32_t groups = q_groups + 2 * kv_groups;
  const uint32_t warp = blockIdx.x * 8 + (threadIdx.x >> 5), step = gridDim.x * 8 / groups;  // warps of a group
  const uint32_t tok0 = warp / groups;
  if (tok0 >= step) return;
  const int grp = (int)(warp - tok0 * groups);
  if (grp < q_groups) {
    if (kNorm && p.q_w != nullptr)
      append_tokens<T, D, U, 0, true>(p, grp, tok0, step);
    else
      append_tokens<T, D, U, 0, false>(p, grp, tok0, step);
  } else if (grp < q_groups + kv_groups) {
    if (kNorm && p.k_w != nullptr)
      append_tokens<T, D, KU, 1, true>(p, grp - q_groups, tok0, step);
    else
      append_tokens<T, D, KU, 1, false>(p, grp - q_groups, tok0, step);
  } else {
    append_tokens<T, D, KU, 2, false>(p, grp - q_groups - kv_groups, tok0, step);
  }
}

// Keys and values alone, as they are, many of them: the same with the next token's rows loaded before this one's are quantised,
// as it is bound by the bytes in flight otherwise: 49,152 tokens of 8 heads of 128 in 51 us (5.1 TB/s; fp16 55), 74 without.
constexpr int kI4WriteHeads = 4;  // heads of a lane, times 256/D of a warp

template <typename T, int D>
__global__ void __launch_bounds__(256, 3) int4_write_kernel(const __grid_constant__ Int4AppendParams p) {
  constexpr int L = D / 8;
  constexpr int RW = 32 / L;
  constexpr int U = kI4WriteHeads;
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, c = lane % L;
  const uint32_t half = (p.hkv + RW * U - 1) / (RW * U);
  const uint32_t warp = blockIdx.x * 8 + (threadIdx.x >> 5), step = gridDim.x * 8 / (2 * half);
  if (warp / (2 * half) >= step) return;
  const int grp = (int)(warp % (2 * half));
  const bool isv = grp >= (int)half;
  const int h0 = (isv ? grp - (int)half : grp) * RW * U + lane / L;
  const int64_t sh = isv ? p.v_sh : p.k_sh, st = isv ? p.v_st : p.k_st;
  const T* src = static_cast<const T*>(isv ? p.v : p.k) + h0 * sh + 8 * c;
  uint8_t* pool = (isv ? p.vp : p.kp) + h0 * p.s_h;
  uint4 next[U];
  int2 slot;
  uint32_t tok = warp / (2 * half);
  const auto load = [&] {
    slot = *reinterpret_cast<const int2*>(p.slots + 2 * (int64_t)tok);
#pragma unroll
    for (int u = 0; u < U; ++u)
      next[u] = h0 + u * RW < p.hkv ? *reinterpret_cast<const uint4*>(src + tok * st + u * RW * sh) : make_uint4(0u, 0u, 0u, 0u);
  };
  if (tok < p.t) load();
  while (tok < p.t) {
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
    const bool use = slot.x >= 0 && slot.x < p.num_pages && slot.y >= 0 && slot.y < p.page_rows;
    uint8_t* row = pool + slot.x * p.s_page + slot.y * p.s_row;
    tok += step;
    if (tok < p.t) load();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t w[4] = {now[u].x, now[u].y, now[u].z, now[u].w};
      uint32_t param;
      const uint32_t word = quantise8<T>(w, param);
      if (use && h0 + u * RW < p.hkv) {
        uint8_t* at = row + u * RW * p.s_h;
        *reinterpret_cast<uint32_t*>(at + 4 * c) = word;
        if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(at + D / 2 + c) = param;
      }
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

// A warp per (tile, head): a lane turns one word of a key row and of the value row beside it into 16 bytes each, a row
// being D/8 lanes. kI4Ahead rows' words are loaded before any is turned: 16,384 tokens of 8 heads of 128 in 14.8 us (5.9 TB/s,
// bound by memory), 29 with one row at a time.
constexpr int kI4Ahead = 4;

template <typename T, int D>
__global__ void __launch_bounds__(256, 4) int4_gather_kernel(const __grid_constant__ Int4GatherParams p) {
  constexpr int L = D / 8;
  constexpr int RW = 32 / L;  // rows a warp takes at a time
  constexpr int A = kI4Ahead;
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
    const int64_t base = te.x * p.s_page + h * p.s_h + te.y * p.s_row;
    const int64_t out = h * p.out_sh + te.w * p.out_sn + 8 * c;
#pragma unroll 1
    for (int r0 = lane / L; r0 < rows; r0 += A * RW) {
      uint32_t kw[A], vw[A], kq[A], vq[A];
      bool use[A];
#pragma unroll
      for (int u = 0; u < A; ++u) {
        const int r = r0 + u * RW;
        const int64_t pr = (int64_t)te.y + r, pos = (int64_t)te.w + r;
        use[u] = r < rows && pr >= 0 && pr < p.page_rows && pos >= 0 && pos < p.n;
        if (use[u]) {
          const uint8_t* kr = p.kp + base + r * p.s_row;
          const uint8_t* vr = p.vp + base + r * p.s_row;
          kw[u] = *reinterpret_cast<const uint32_t*>(kr + 4 * c);
          vw[u] = *reinterpret_cast<const uint32_t*>(vr + 4 * c);
          kq[u] = *reinterpret_cast<const uint32_t*>(kr + D / 2 + 4 * (c / 4));
          vq[u] = *reinterpret_cast<const uint32_t*>(vr + D / 2 + 4 * (c / 4));
        }
      }
#pragma unroll
      for (int u = 0; u < A; ++u) {
        if (use[u]) {
          const int64_t o = out + (r0 + u * RW) * p.out_sn;
          uint32_t x[4];
          i4_values<T>(kw[u], kq[u], x);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + o) = make_uint4(x[0], x[1], x[2], x[3]);
          i4_values<T>(vw[u], vq[u], x);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.v_out) + o) = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
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
  float minus_zero;       // -0
};

// Keys re-rotated in place by one angle a frequency (the splice of threadcut/kv.py:28-41 over 4-bit rows): a row's
// values, rotated in fp32 as the 16-bit splice rotates them, rounded to T and quantised again. A warp per
// (layer, tile, head); a row is D/16 lanes, each with 8 elements of its first half and the 8 that they are paired with. kI4Ahead
// rows' words are loaded before any is turned. Bound by instructions (18 an element, half of them on the half-rate pipe: 72 %
// of the issue slots used, 59 % of that pipe; its bytes alone would take 10 us): 49,152 keys of 8 heads of 128 in 37 us, 47 with a lane's partners fetched by
// shuffles and converted twice.
template <typename T, int D>
__global__ void __launch_bounds__(256, 3) int4_rotate_kernel(const __grid_constant__ Int4RotateParams p) {
  constexpr int L = D / 16;
  constexpr int RW = 32 / L;
  constexpr int A = kI4Ahead;
  const int lane = threadIdx.x & 31, c = lane % L;
  float2 cs[4], sn[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    cs[e] = make_float2(p.cs[8 * c + 2 * e], p.cs[8 * c + 2 * e + 1]);
    sn[e] = make_float2(p.cs[D / 2 + 8 * c + 2 * e], p.cs[D / 2 + 8 * c + 2 * e + 1]);
  }
  const float2 nz = make_float2(p.minus_zero, p.minus_zero);
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
    const int64_t page = te[0], first_row = te[1];
    const int rows = te[2] < kI4TileRows ? te[2] : kI4TileRows;
    if (page < 0 || page >= p.num_pages) continue;
    uint8_t* base = p.kp[layer] + page * p.s_page + h * p.s_h + first_row * p.s_row;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += A * RW) {  // the whole warp: quantise8 exchanges extremes
      uint32_t wx[A], wy[A], qx[A], qy[A];
      bool use[A];
#pragma unroll
      for (int u = 0; u < A; ++u) {
        const int r = r0 + u * RW + lane / L;
        const int64_t pr = first_row + r;
        use[u] = r < rows && pr >= 0 && pr < p.page_rows;
        wx[u] = wy[u] = qx[u] = qy[u] = 0u;
        if (use[u]) {
          const uint32_t* row = reinterpret_cast<const uint32_t*>(base + r * p.s_row);
          wx[u] = row[c];
          wy[u] = row[D / 16 + c];
          qx[u] = row[D / 8 + c / 4];
          qy[u] = row[D / 8 + D / 64 + c / 4];
        }
      }
#pragma unroll
      for (int u = 0; u < A; ++u) {
        if (r0 + u * RW >= rows) break;  // (the same for every lane)
        uint32_t vx[4], vy[4];
        i4_values<T>(wx[u], qx[u], vx);
        i4_values<T>(wy[u], qy[u], vy);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = make_float2(Mma<T>::lo(vx[e]), Mma<T>::hi(vx[e])), y = make_float2(Mma<T>::lo(vy[e]), Mma<T>::hi(vy[e]));
          const float2 a = fadd2(product2(x, cs[e], nz), product2(y, make_float2(-sn[e].x, -sn[e].y), nz));
          const float2 b = fadd2(product2(y, cs[e], nz), product2(x, sn[e], nz));
          vx[e] = Mma<T>::pack(a.x, a.y);
          vy[e] = Mma<T>::pack(b.x, b.y);
        }
        const uint32_t ox = quantise8<T>(vx, qx[u]), oy = quantise8<T>(vy, qy[u]);
        // every lane of a group has read its (S, z): the exchange above waited for them
        if (use[u]) {
          uint32_t* row = reinterpret_cast<uint32_t*>(base + (r0 + u * RW + lane / L) * p.s_row);
          row[c] = ox;
          row[D / 16 + c] = oy;
          if ((c & 3) == 0) {
            row[D / 8 + c / 4] = qx[u];
            row[D / 8 + D / 64 + c / 4] = qy[u];
          }
        }
      }
    }
  }
}

}  // namespace tc
