// Split-KV decode attention over a cache held in 4 bits (rows as in int4.cuh): softmax(scale q K^T) V of the g
// query heads of each KV head over the values that the rows stand for, which are exactly what the products take.
//
// Split, merge and partials are those of the 16-bit decode kernel (finish_cta). Inside a CTA each warp works
// alone, on tiles of 32 rows that it copies into its own two shared-memory stages with cp.async: nothing waits
// for another warp before the end. Per tile
//   S^T[32 tok x 8 heads] = K q^T   K's fragments straight from the codes: lane (r, c) takes word c of a
//                                   group's four, 8 neighbouring elements, as the columns of two products, so
//                                   that every product lies within one group and q is permuted once instead
//   online softmax                  as in the 16-bit kernel
//   O^T[D x 8 heads] += V^T P^T     the words of two tokens are paired by byte permutes, lane r's rows of the
//                                   products being its own D/8 neighbouring elements, all of one group
// with P in two 16-bit parts, as there.
#pragma once

#include "decode_attn.cuh"
#include "int4.cuh"

namespace tc {

constexpr int kI4Warps = 8;
constexpr int kI4Stages = 2;

struct Int4DecodeParams : DecodeParams {
  // k, v: uint8 bases; sk_*, sv_* in bytes. Paged: k, v are pools [num_pages][hkv][page_rows], sk_b the page
  // stride, and tile t is rows [te[1], te[1] + te[2]) of page te[0], te = tiles + tile_cols t.
  int paged;  // (a sequence without tiles needs no table)
  int tile_cols;
  int64_t page_rows, num_pages;
};

template <int D>
struct I4Geom {
  static constexpr int kRow = i4_row_bytes(D);
  // Shared-memory row stride: the 32 words that a warp reads of 8 rows lie in different banks.
  static constexpr int kStride = D == 64 ? 48 : D == 128 ? 80 : 176;
  static constexpr int kCopy = D == 64 ? 8 : 16;  // bytes of a copy
  static constexpr int kCopies = kRow / kCopy;    // of a row
  static constexpr int kStage = 2 * kTile * kStride;
  static constexpr int kWarpBytes = kI4Stages * kStage;
  static constexpr int kSmem = kI4Warps * kWarpBytes;
};

// Asynchronous copy of kBytes; without `in`, zeros (src is not read).
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool in) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes),
                 "r"(in ? kBytes : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                   : "r"(addr + 4 * i));
  }
}

// T in {bf16, f16}, D in {64, 128, 256}, NG tiles of 8 query heads (g <= 8 NG).
template <typename T, int D, int NG>
__global__ void __launch_bounds__(32 * kI4Warps, D * NG <= 128 ? 2 : 1)
    int4_decode_kernel(const __grid_constant__ Int4DecodeParams p) {
  using G = I4Geom<D>;
  constexpr int HP = 8 * NG;
  constexpr int NGR = D / kI4Group;  // groups of a row
  constexpr int WPT = D / 64;        // words of a value row that a lane takes
  static_assert(Region<D, HP>::kFloats * 4 <= G::kWarpBytes, "a warp's state must fit in its stages");
  static_assert(merge_scratch_bytes(32 * kI4Warps) <= G::kSmem, "merge scratch must fit in the stages");
  extern __shared__ __align__(16) uint8_t i4_smem[];
  __shared__ int s_mi;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  pdl_launch();
  pdl_wait();
  const int64_t n = seq_length<true>(p, b);  // clamped into [0, p.n]
  const bool paged = p.paged;
  const int64_t seq_tiles = paged ? p.n_tiles : (n + kTile - 1) / kTile;
  const int nsplit = seq_tiles > 0 ? (int)((seq_tiles + p.tiles_per_split - 1) / p.tiles_per_split) : 1;
  if (split >= nsplit) return;
  int64_t tt0, tt1;
  split_range(seq_tiles, split, nsplit, tt0, tt1);
  const int ntiles = (int)(tt1 - tt0);
  if (threadIdx.x == 0)
    s_mi = nsplit > 1 && !last_arrival_merge(nsplit, blockDim.x) ? merger_index(p, b, h, nsplit, p.g * (D / 4)) : -1;

  uint8_t* ring = i4_smem + warp * G::kWarpBytes;
  const uint32_t ring_s = smem_u32(ring);
  const uint8_t* kb = static_cast<const uint8_t*>(p.k) + h * p.sk_h;
  const uint8_t* vb = static_cast<const uint8_t*>(p.v) + h * p.sv_h;

  // Valid rows of tile j, and where they begin.
  auto locate = [&](int j, const uint8_t*& ks, const uint8_t*& vs) -> int {
    const int64_t t = tt0 + j;
    int64_t outer = b, row = t * kTile, rows = n - row;
    if (paged) {
      const int32_t* te = p.tiles + p.tile_cols * t;
      outer = te[0];
      row = te[1];
      rows = te[2];
      if (outer < 0 || outer >= p.num_pages || row < 0 || row >= p.page_rows) rows = 0;
      if (rows > p.page_rows - row) rows = p.page_rows - row;
    }
    if (rows <= 0) {
      ks = kb;
      vs = vb;
      return 0;
    }
    ks = kb + outer * p.sk_b + row * p.sk_n;
    vs = vb + outer * p.sv_b + row * p.sv_n;
    return rows < kTile ? (int)rows : kTile;
  };
  // Starts the copies of tile j into stage s; rows behind the valid ones become zeros (code 0, S = z = 0).
  auto fetch = [&](int j, int s) -> int {
    const uint8_t *ks, *vs;
    const int valid = locate(j, ks, vs);
    const uint32_t dst = ring_s + s * G::kStage;
#pragma unroll
    for (int u = 0; u < G::kCopies; ++u) {
      const int x = lane + 32 * u;
      const int row = x / G::kCopies, ch = x - row * G::kCopies;
      const bool in = row < valid;
      const uint32_t d = dst + row * G::kStride + ch * G::kCopy;
      copy_async<G::kCopy>(d, in ? ks + row * p.sk_n + ch * G::kCopy : kb, in);
      copy_async<G::kCopy>(d + kTile * G::kStride, in ? vs + row * p.sv_n + ch * G::kCopy : vb, in);
    }
    return valid;
  };

  int valid_next = 0;
  if (warp < ntiles) valid_next = fetch(warp, 0);
  copy_commit();

  // q^T fragments: product 2 grp + m takes of each group's word c the codes (2m, 2m + 4) and (2m + 1, 2m + 5)
  uint32_t bq[NG][2 * NGR][2];
  {
    const T* qb = static_cast<const T*>(p.q) + b * p.sq_b + h * p.sq_h;
    const T zero = from_f32<T>(0.f);
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
      const int i = nt * 8 + r;
      const bool ok = i < p.g;
      const T* qr = qb + (ok ? i : 0) * p.sq_g;
#pragma unroll
      for (int ks = 0; ks < 2 * NGR; ++ks) {
        const int e = (ks >> 1) * kI4Group + 8 * c + 2 * (ks & 1);
        bq[nt][ks][0] = pack_raw<T>(ok ? qr[e] : zero, ok ? qr[e + 4] : zero);
        bq[nt][ks][1] = pack_raw<T>(ok ? qr[e + 1] : zero, ok ? qr[e + 5] : zero);
      }
    }
  }
  float m_run[NG][2], l_run[NG][2];
  float oacc[4 * WPT][NG][4];
#pragma unroll
  for (int nt = 0; nt < NG; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m_run[nt][e] = -INFINITY;
      l_run[nt][e] = 0.f;
    }
#pragma unroll
  for (int i = 0; i < 4 * WPT; ++i)
#pragma unroll
    for (int nt = 0; nt < NG; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) oacc[i][nt][e] = 0.f;

  int s = 0;
  for (int j = warp; j < ntiles; j += kI4Warps, s ^= 1) {
    const int valid = valid_next;
    if (j + kI4Warps < ntiles) valid_next = fetch(j + kI4Warps, s ^ 1);
    copy_commit();
    copy_wait<1>();
    __syncwarp();
    const uint32_t kst = ring_s + s * G::kStage, vst = kst + kTile * G::kStride;

    float sacc[2][NG][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NG; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sacc[mt][nt][e] = 0.f;
      const uint32_t k0 = kst + (mt * 16 + r) * G::kStride, k1 = k0 + 8 * G::kStride;
      uint32_t p0[NGR], p1[NGR];
      lds_words(k0 + D / 2, p0);
      lds_words(k1 + D / 2, p1);
#pragma unroll
      for (int gr = 0; gr < NGR; ++gr) {
        uint32_t w0[1], w1[1], a[4];
        lds_words(k0 + 16 * gr + 4 * c, w0);
        lds_words(k1 + 16 * gr + 4 * c, w1);
        const uint32_t s0 = i4_low2(p0[gr], p0[gr]), z0 = i4_high2(p0[gr], p0[gr]);
        const uint32_t s1 = i4_low2(p1[gr], p1[gr]), z1 = i4_high2(p1[gr], p1[gr]);
        a[0] = I4<T>::fma2(i4_mant<T, 0>(w0[0]), s0, z0);
        a[1] = I4<T>::fma2(i4_mant<T, 0>(w1[0]), s1, z1);
        a[2] = I4<T>::fma2(i4_mant<T, 1>(w0[0]), s0, z0);
        a[3] = I4<T>::fma2(i4_mant<T, 1>(w1[0]), s1, z1);
#pragma unroll
        for (int nt = 0; nt < NG; ++nt) Mma<T>::run(sacc[mt][nt], a, bq[nt][2 * gr][0], bq[nt][2 * gr][1]);
        a[0] = I4<T>::fma2(i4_mant<T, 2>(w0[0]), s0, z0);
        a[1] = I4<T>::fma2(i4_mant<T, 2>(w1[0]), s1, z1);
        a[2] = I4<T>::fma2(i4_mant<T, 3>(w0[0]), s0, z0);
        a[3] = I4<T>::fma2(i4_mant<T, 3>(w1[0]), s1, z1);
#pragma unroll
        for (int nt = 0; nt < NG; ++nt) Mma<T>::run(sacc[mt][nt], a, bq[nt][2 * gr + 1][0], bq[nt][2 * gr + 1][1]);
      }
    }

    // online softmax; this lane holds tokens {r, r+8, r+16, r+24} x heads {2c, 2c+1}
    float alpha[NG][2];
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x0 = sacc[0][nt][e] * p.c, x1 = sacc[0][nt][2 + e] * p.c;
        float x2 = sacc[1][nt][e] * p.c, x3 = sacc[1][nt][2 + e] * p.c;
        if (r >= valid) x0 = -INFINITY;
        if (r + 8 >= valid) x1 = -INFINITY;
        if (r + 16 >= valid) x2 = -INFINITY;
        if (r + 24 >= valid) x3 = -INFINITY;
        float mx = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mnew = fmaxf(m_run[nt][e], mx);
        const float mref = max_ref(mnew);
        alpha[nt][e] = fast_exp2(m_run[nt][e] - mref);
        m_run[nt][e] = mnew;
        const float e0 = fast_exp2(x0 - mref), e1 = fast_exp2(x1 - mref);
        const float e2 = fast_exp2(x2 - mref), e3 = fast_exp2(x3 - mref);
        l_run[nt][e] = l_run[nt][e] * alpha[nt][e] + ((e0 + e1) + (e2 + e3));
        sacc[0][nt][e] = e0;
        sacc[0][nt][2 + e] = e1;
        sacc[1][nt][e] = e2;
        sacc[1][nt][2 + e] = e3;
      }
    }
#pragma unroll
    for (int i = 0; i < 4 * WPT; ++i)
#pragma unroll
      for (int nt = 0; nt < NG; ++nt) {
        oacc[i][nt][0] *= alpha[nt][0];
        oacc[i][nt][1] *= alpha[nt][1];
        oacc[i][nt][2] *= alpha[nt][0];
        oacc[i][nt][3] *= alpha[nt][1];
      }

#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      // P^T fragments of 16 tokens, in two 16-bit parts
      uint32_t hi[NG][2], lo[NG][2];
#pragma unroll
      for (int nt = 0; nt < NG; ++nt) {
        const float* sp = sacc[kk][nt];
        const uint32_t x0 = Mma<T>::pack(sp[0], sp[1]), x1 = Mma<T>::pack(sp[2], sp[3]);
        const uint32_t y0 = Mma<T>::pack(sp[0] - Mma<T>::lo(x0), sp[1] - Mma<T>::hi(x0));
        const uint32_t y1 = Mma<T>::pack(sp[2] - Mma<T>::lo(x1), sp[3] - Mma<T>::hi(x1));
        hi[nt][0] = movm_t(x0);
        hi[nt][1] = movm_t(x1);
        lo[nt][0] = movm_t(y0);
        lo[nt][1] = movm_t(y1);
      }
      // this lane's tokens 2c, 2c+1, 2c+8, 2c+9 of the 16: its D/8 elements and their group's (S, z)
      uint32_t w[4][WPT], q[4][1];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t row = vst + (kk * 16 + 2 * c + (t & 1) + 8 * (t >> 1)) * G::kStride;
        lds_words(row + 4 * WPT * r, w[t]);
        lds_words(row + D / 2 + 4 * (WPT * r / 4), q[t]);
      }
      const uint32_t s01 = i4_low2(q[0][0], q[1][0]), z01 = i4_high2(q[0][0], q[1][0]);
      const uint32_t s23 = i4_low2(q[2][0], q[3][0]), z23 = i4_high2(q[2][0], q[3][0]);
#pragma unroll
      for (int x = 0; x < WPT; ++x) {
        const uint32_t l01 = i4_low2(w[0][x], w[1][x]), h01 = i4_high2(w[0][x], w[1][x]);
        const uint32_t l23 = i4_low2(w[2][x], w[3][x]), h23 = i4_high2(w[2][x], w[3][x]);
        auto product = [&](int i, uint32_t m0, uint32_t m1, uint32_t m2, uint32_t m3) {
          const uint32_t a[4] = {I4<T>::fma2(m0, s01, z01), I4<T>::fma2(m1, s01, z01), I4<T>::fma2(m2, s23, z23),
                                 I4<T>::fma2(m3, s23, z23)};
#pragma unroll
          for (int nt = 0; nt < NG; ++nt) {
            Mma<T>::run(oacc[i][nt], a, hi[nt][0], hi[nt][1]);
            Mma<T>::run(oacc[i][nt], a, lo[nt][0], lo[nt][1]);
          }
        };
        product(4 * x, i4_mant<T, 0>(l01), i4_mant<T, 0>(h01), i4_mant<T, 0>(l23), i4_mant<T, 0>(h23));
        product(4 * x + 1, i4_mant<T, 1>(l01), i4_mant<T, 1>(h01), i4_mant<T, 1>(l23), i4_mant<T, 1>(h23));
        product(4 * x + 2, i4_mant<T, 2>(l01), i4_mant<T, 2>(h01), i4_mant<T, 2>(l23), i4_mant<T, 2>(h23));
        product(4 * x + 3, i4_mant<T, 3>(l01), i4_mant<T, 3>(h01), i4_mant<T, 3>(l23), i4_mant<T, 3>(h23));
      }
    }
    __syncwarp();  // the stage may be filled again
  }
  copy_wait<0>();
  __syncwarp();

  // this warp's state -> its own (now idle) stages
  using R = Region<D, HP>;
  float* reg = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int nt = 0; nt < NG; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[nt][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int head = nt * 8 + 2 * c + e;
      if (r == 0) {
        R::m(reg)[head] = m_run[nt][e];
        R::l(reg)[head] = l;
      }
#pragma unroll
      for (int x = 0; x < WPT; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* acc = R::acc(reg, head) + 8 * WPT * r + 8 * x + i;
          acc[0] = oacc[4 * x + i][nt][e];
          acc[4] = oacc[4 * x + i][nt][2 + e];
        }
    }
  __syncthreads();
  finish_cta<T, D, HP>(p, i4_smem, G::kWarpBytes, kI4Warps, b, h, split, nsplit, s_mi);
}

}  // namespace tc
