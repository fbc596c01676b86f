// Split-KV decode attention over a cache held in 4 bits (rows as in int4.cuh): softmax(scale q K^T) V of the g
// query heads of each KV head over the values that the rows stand for, which are exactly what the products take.
//
// Partials and their merge are those of the 16-bit decode kernel (finish_cta). Inside a CTA each warp works alone, on
// tiles of 32 rows that it brings into its own two shared-memory stages: nothing waits for another warp before the end.
// Per tile
//   S^T[32 tok x heads] = K q^T     K's fragments straight from the codes: lane (r, c) takes word c of a group's four, 8
//                                   neighbouring elements, as the columns of two products, so that every product lies
//                                   within one group and q is permuted once instead
//   online softmax                  as in the 16-bit kernel, the sums so far rescaled only where a maximum grew
//   O^T[D x heads] += V^T P^T       the words of two tokens are paired by byte permutes, lane r's rows of the products being
//                                   its own D/8 neighbouring elements, all of one group
// P enters in two 16-bit parts; for up to 4 query heads a KV head (NH = 1) these are neighbouring columns of one product.
//
// A tile of d = 128 takes about 800 instructions, most of them on the half-rate ALU pipe (masks, shifts, permutes). Over a launch 61
// to 65 % of the issue slots are used, 54 to 57 % of that pipe and 20 % of the tensor pipe: nothing is full. An instruction waits 1.1
// cycles for the one ahead of it, 1.0 to 1.1 for that pipe and 1.2 to 1.3 for another warp's turn: the 16 warps that an SM's registers
// hold do not cover a tile's chain of product, softmax and product with each other. 8 KV heads of 128 with 4 query heads
// each: 98,304 rows 34 us (3.7 TB/s; start, merge and launch about 10 of it), 64 ragged sequences with 560,000 rows in all
// 174 us (4.1 TB/s), 1,536 rows 8.1 us. Below some 12,000 rows of one sequence the 16-bit
// kernel, whose first tiles may be loaded ahead, is as fast on its own rows.
#pragma once

#include "decode_attn.cuh"
#include "int4.cuh"

namespace tc {

constexpr int kI4Stages = 2;

struct Int4DecodeParams : DecodeParams {
  // k, v: uint8 bases; sk_*, sv_* in bytes. Paged: k, v are pools [num_pages][hkv][page_rows], sk_b the page
  // stride, and tile t is rows [te[1], te[1] + te[2]) of page te[0], te = tiles + tile_cols t.
  int paged;  // (a sequence without tiles needs no table)
  int tile_cols;
  int q_vec;  // q in 16-byte chunks
  int64_t page_rows, num_pages;
};

// kBulk: a tile's rows are neighbours in memory (of one page, or of a sequence), 16-byte aligned, and come as one bulk
// copy; else a lane copies units of 16 bytes (d = 64: 8) row by row.
template <int D, bool kBulk, int kWarps>
struct I4Geom {
  static constexpr int kRow = i4_row_bytes(D);
  // Shared-memory row stride. Where it is free, the 32 words that a warp reads of 8 rows lie in different banks; 160 of a
  // bulk copy at d = 256 has two to a bank.
  static constexpr int kStride = kBulk ? kRow : D == 64 ? 48 : D == 128 ? 80 : 176;
  static constexpr int kCopy = D == 64 ? 8 : 16;  // bytes of a copy
  static constexpr int kCopies = kRow / kCopy;    // of a row
  static constexpr int kStage = 2 * kTile * kStride;
  static constexpr int kWarpBytes = kI4Stages * kStage;
  static constexpr int kSmem = kWarps * kWarpBytes;
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

// Warps an SM holds, by what a lane holds (O^T's sums and q's fragments): 16 within 128 registers, where that spills nothing.
__host__ __device__ constexpr int i4_warps(int d, int nh) { return d * nh <= 256 && d <= 128 ? 16 : 8; }

// T in {bf16, f16}, D in {64, 128, 256}, NH tiles of 4 query heads (g <= 4 NH), kWarps of a CTA.
template <typename T, int D, int NH, bool kBulk, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, i4_warps(D, NH) / kWarps)
    int4_decode_kernel(const __grid_constant__ Int4DecodeParams p) {
  using G = I4Geom<D, kBulk, kWarps>;
  constexpr int NT = NH == 1 ? 1 : NH / 2;  // tiles of 8 columns
  constexpr int HP = 8 * NT;
  constexpr int NGR = D / kI4Group;  // groups of a row
  constexpr int WPT = D / 64;        // words of a value row that a lane takes
  using R = Region<D, HP>;
  static_assert(R::kFloats * 4 <= G::kWarpBytes, "a warp's state must fit in its stages");
  static_assert(merge_scratch_bytes(32 * kWarps) <= G::kSmem, "merge scratch must fit in the stages");
  extern __shared__ __align__(16) uint8_t i4_smem[];
  __shared__ uint64_t s_full[kBulk ? kWarps * kI4Stages : 1];
  __shared__ float s_weight[kWarps][HP];
  __shared__ int s_mi;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  uint64_t* full = s_full + (kBulk ? warp * kI4Stages : 0);
  if constexpr (kBulk) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kI4Stages; ++i) mbar_init(&full[i], 1);
      fence_mbar_init();
    }
    __syncwarp();
  }
  pdl_launch();
  pdl_wait();
  const int n = (int)seq_length<true>(p, b);  // clamped into [0, p.n], below 2^30
  const bool paged = p.paged;
  const int seq_tiles = paged ? (int)p.n_tiles : (n + kTile - 1) / kTile;
  const int nsplit = seq_tiles > 0 ? (seq_tiles + p.tiles_per_split - 1) / p.tiles_per_split : 1;
  if (split >= nsplit) return;
  // as even as whole tiles allow
  const int share = seq_tiles / nsplit, more = seq_tiles - share * nsplit;
  const int tt0 = split * share + (split < more ? split : more);
  const int ntiles = share + (split < more);

  uint8_t* ring = i4_smem + warp * G::kWarpBytes;
  const uint32_t ring_s = smem_u32(ring);
  const uint64_t pol = policy_evict_first();

  // Where tile j lies: (page or sequence, first row, rows), read a tile ahead of its use.
  auto entry = [&](int j) -> int3 {
    const int t = tt0 + j;
    if (paged) {
      const int32_t* te = p.tiles + p.tile_cols * (int64_t)t;
      return make_int3(te[0], te[1], te[2]);
    }
    return make_int3(b, t * kTile, n - t * kTile);
  };
  // Valid rows of a tile.
  auto rows_of = [&](int3 te) -> int {
    int valid = te.z;
    if (paged) {
      if (te.x < 0 || te.x >= p.num_pages || te.y < 0 || te.y >= p.page_rows) valid = 0;
      if (valid > p.page_rows - te.y) valid = (int)(p.page_rows - te.y);
    }
    return valid < 0 ? 0 : valid > kTile ? kTile : valid;
  };
  // Starts the copies of a tile's valid rows into stage s. What lies behind them: zeros (cp.async), or whatever was
  // there (bulk).
  auto fetch = [&](int3 te, int valid, int s) {
    if constexpr (kBulk) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[s], 2 * valid * G::kRow);
        if (valid > 0) {
          bulk_g2s(ring + s * G::kStage, static_cast<const uint8_t*>(p.k) + h * p.sk_h + te.x * p.sk_b + te.y * p.sk_n,
                   valid * G::kRow, &full[s], pol);
          bulk_g2s(ring + s * G::kStage + kTile * G::kStride,
                   static_cast<const uint8_t*>(p.v) + h * p.sv_h + te.x * p.sv_b + te.y * p.sv_n, valid * G::kRow, &full[s],
                   pol);
        }
      }
    } else {
      const uint8_t* kb = static_cast<const uint8_t*>(p.k) + h * p.sk_h;
      const uint8_t* vb = static_cast<const uint8_t*>(p.v) + h * p.sv_h;
      const uint8_t* ks = kb + te.x * p.sk_b + te.y * p.sk_n;
      const uint8_t* vs = vb + te.x * p.sv_b + te.y * p.sv_n;
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
    }
  };

  int valid_next = 0;
  int3 ahead = make_int3(0, 0, 0);
  if (warp < ntiles) {
    const int3 te = entry(warp);
    valid_next = rows_of(te);
    fetch(te, valid_next, 0);
  }
  if constexpr (!kBulk) copy_commit();
  if (warp + kWarps < ntiles) ahead = entry(warp + kWarps);
  if (threadIdx.x == 0)
    s_mi = nsplit > 1 && !last_arrival_merge(nsplit, blockDim.x) ? merger_index(p, b, h, nsplit, p.g * (D / 4)) : -1;

  // q^T fragments: product 2 gr + m takes of each group's word c the codes (2m, 2m + 4) and (2m + 1, 2m + 5). Column 2i of
  // tile nt is query head 8 nt + i, column 2i + 1 head 8 nt + 4 + i (NH = 1: nothing, P's second part goes there)
  uint32_t bq[NT][2 * NGR][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int i = 8 * nt + (r >> 1) + 4 * (r & 1);
    const bool ok = i < p.g && (NH > 1 || !(r & 1));
    const T* qr = static_cast<const T*>(p.q) + b * p.sq_b + h * p.sq_h + (ok ? i : 0) * p.sq_g + 8 * c;
#pragma unroll
    for (int gr = 0; gr < NGR; ++gr) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (ok) {
        if (p.q_vec) {
          x = *reinterpret_cast<const uint4*>(qr + gr * kI4Group);
        } else {
          T e[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) e[u] = qr[gr * kI4Group + u];
          memcpy(&x, e, 16);
        }
      }
      bq[nt][2 * gr][0] = i4_low2(x.x, x.z);
      bq[nt][2 * gr][1] = i4_high2(x.x, x.z);
      bq[nt][2 * gr + 1][0] = i4_low2(x.y, x.w);
      bq[nt][2 * gr + 1][1] = i4_high2(x.y, x.w);
    }
  }
  float m_run[NH], l_run[NH];
  float oacc[4 * WPT][NT][4];
#pragma unroll
  for (int t = 0; t < NH; ++t) {
    m_run[t] = -INFINITY;
    l_run[t] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4 * WPT; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) oacc[i][nt][e] = 0.f;

  int s = 0, phase = 0;
  for (int j = warp; j < ntiles; j += kWarps) {
    const int valid = valid_next;
    if (j + kWarps < ntiles) {
      valid_next = rows_of(ahead);
      fetch(ahead, valid_next, s ^ 1);
    }
    if (j + 2 * kWarps < ntiles) ahead = entry(j + 2 * kWarps);
    const uint32_t kst = ring_s + s * G::kStage, vst = kst + kTile * G::kStride;
    if constexpr (kBulk) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], phase, TC_DEVERR_PIPE_TIMEOUT))) {
        // given up by the whole warp, and only once its copies had another chance to end
        mbar_wait(&full[s], phase, TC_DEVERR_PIPE_TIMEOUT);
        if (j + kWarps < ntiles) mbar_wait(&full[s ^ 1], phase ^ s, TC_DEVERR_PIPE_TIMEOUT);
        break;
      }
      if (valid < kTile) {
        // values of rows that the tile does not have: S = z = 0, so that a weight of 0 never meets a NaN
        if (lane >= valid) {
          uint4* param = reinterpret_cast<uint4*>(ring + s * G::kStage + (kTile + lane) * G::kStride + D / 2);
#pragma unroll
          for (int i = 0; i < D / 128; ++i) param[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
      }
    } else {
      copy_commit();
      copy_wait<1>();
      __syncwarp();
    }

    // scores of tokens r, r + 8, r + 16, r + 24 (index 2 mt + half), of head 4 t + c
    float sc[4][NH];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint32_t k0 = kst + (mt * 16 + r) * G::kStride, k1 = k0 + 8 * G::kStride;
      uint32_t p0[NGR], p1[NGR];
      lds_words(k0 + D / 2, p0);
      lds_words(k1 + D / 2, p1);
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NGR; ++gr) {
        uint32_t w0[1], w1[1];
        lds_words(k0 + 16 * gr + 4 * c, w0);
        lds_words(k1 + 16 * gr + 4 * c, w1);
        const uint32_t s0 = i4_low2(p0[gr], p0[gr]), z0 = i4_high2(p0[gr], p0[gr]);
        const uint32_t s1 = i4_low2(p1[gr], p1[gr]), z1 = i4_high2(p1[gr], p1[gr]);
        const uint32_t a[4] = {I4<T>::fma2(i4_ones<T, 0>(w0[0]), s0, z0), I4<T>::fma2(i4_ones<T, 0>(w1[0]), s1, z1),
                               I4<T>::fma2(i4_ones<T, 1>(w0[0]), s0, z0), I4<T>::fma2(i4_ones<T, 1>(w1[0]), s1, z1)};
        const uint32_t a2[4] = {I4<T>::fma2(i4_ones<T, 2>(w0[0]), s0, z0), I4<T>::fma2(i4_ones<T, 2>(w1[0]), s1, z1),
                                I4<T>::fma2(i4_ones<T, 3>(w0[0]), s0, z0), I4<T>::fma2(i4_ones<T, 3>(w1[0]), s1, z1)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          Mma<T>::run(acc[nt], a, bq[nt][2 * gr][0], bq[nt][2 * gr][1]);
          Mma<T>::run(acc[nt], a2, bq[nt][2 * gr + 1][0], bq[nt][2 * gr + 1][1]);
        }
      }
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        sc[2 * mt][t] = acc[t / 2][t & 1] * p.c;
        sc[2 * mt + 1][t] = acc[t / 2][2 + (t & 1)] * p.c;
      }
    }

    // online softmax
    if (valid < kTile) {
#pragma unroll
      for (int t = 0; t < NH; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + 8 * i >= valid) sc[i][t] = -INFINITY;
    }
    float mref[NH], alpha[NH];
    bool grew = false;
#pragma unroll
    for (int t = 0; t < NH; ++t) {
      float mx = fmaxf(fmaxf(sc[0][t], sc[1][t]), fmaxf(sc[2][t], sc[3][t]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float mnew = fmaxf(m_run[t], mx);
      grew = grew || mnew > m_run[t];
      mref[t] = max_ref(mnew);
      alpha[t] = fast_exp2(m_run[t] - mref[t]);
      m_run[t] = mnew;
    }
    if (__any_sync(0xffffffffu, grew)) {
      // columns 2c, 2c + 1 of O^T: the two parts of head c (NH = 1), else heads c and c + 4 of a tile
#pragma unroll
      for (int t = 0; t < NH; ++t) l_run[t] *= alpha[t];
#pragma unroll
      for (int i = 0; i < 4 * WPT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float a0 = alpha[NH == 1 ? 0 : 2 * nt], a1 = alpha[NH == 1 ? 0 : 2 * nt + 1];
          oacc[i][nt][0] *= a0;
          oacc[i][nt][1] *= a1;
          oacc[i][nt][2] *= a0;
          oacc[i][nt][3] *= a1;
        }
    }
#pragma unroll
    for (int t = 0; t < NH; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i][t] = fast_exp2(sc[i][t] - mref[t]);
      l_run[t] += (sc[0][t] + sc[1][t]) + (sc[2][t] + sc[3][t]);
    }

#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      // P^T fragments of 16 tokens
      uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float* x = sc[2 * kk + e];
          if constexpr (NH == 1) {
            hi[nt][e] = movm_t(Mma<T>::pack(x[0], x[0] - Mma<T>::lo(Mma<T>::pack(x[0], 0.f))));
          } else {
            const uint32_t y = Mma<T>::pack(x[2 * nt], x[2 * nt + 1]);
            hi[nt][e] = movm_t(y);
            lo[nt][e] = movm_t(Mma<T>::pack(x[2 * nt] - Mma<T>::lo(y), x[2 * nt + 1] - Mma<T>::hi(y)));
          }
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
          for (int nt = 0; nt < NT; ++nt) {
            Mma<T>::run(oacc[i][nt], a, hi[nt][0], hi[nt][1]);
            if constexpr (NH > 1) Mma<T>::run(oacc[i][nt], a, lo[nt][0], lo[nt][1]);
          }
        };
        product(4 * x, i4_ones<T, 0>(l01), i4_ones<T, 0>(h01), i4_ones<T, 0>(l23), i4_ones<T, 0>(h23));
        product(4 * x + 1, i4_ones<T, 1>(l01), i4_ones<T, 1>(h01), i4_ones<T, 1>(l23), i4_ones<T, 1>(h23));
        product(4 * x + 2, i4_ones<T, 2>(l01), i4_ones<T, 2>(h01), i4_ones<T, 2>(l23), i4_ones<T, 2>(h23));
        product(4 * x + 3, i4_ones<T, 3>(l01), i4_ones<T, 3>(h01), i4_ones<T, 3>(l23), i4_ones<T, 3>(h23));
      }
    }
    if (kBulk && valid < kTile) fence_proxy_async_smem();  // the zeros above precede the next copy into the stage
    __syncwarp();  // the stage may be filled again
    s ^= 1;
    phase ^= s == 0;
  }
  if constexpr (!kBulk) copy_wait<0>();
  __syncwarp();

  // this warp's state -> its own (now idle) stages
  float* reg = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int t = 0; t < NH; ++t) {
    float l = l_run[t];
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    l += __shfl_xor_sync(0xffffffffu, l, 16);
    const int head = 4 * t + c;
    if (r == 0) {
      R::m(reg)[head] = m_run[t];
      R::l(reg)[head] = l;
    }
    const int nt = NH == 1 ? 0 : t / 2, e = NH == 1 ? 0 : t & 1;
#pragma unroll
    for (int x = 0; x < WPT; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* o = oacc[4 * x + i][nt];
        float* acc = R::acc(reg, head) + 8 * WPT * r + 8 * x + i;
        acc[0] = NH == 1 ? o[0] + o[1] : o[e];
        acc[4] = NH == 1 ? o[2] + o[3] : o[2 + e];
      }
  }
  __syncthreads();
  // the warps' states as one, in the first warp's place: a head's maximum, weights and sum by the lanes of one warp, then an
  // output a thread
  auto region = [&](int w) { return reinterpret_cast<float*>(i4_smem + w * G::kWarpBytes); };
  for (int i = warp; i < p.g; i += kWarps) {
    const float m = lane < kWarps ? R::m(region(lane))[i] : -INFINITY;
    const float M = warp_max(m);
    const float w = fast_exp2(m - max_ref(M));
    const float L = warp_sum(lane < kWarps ? w * R::l(region(lane))[i] : 0.f);
    if (lane < kWarps) s_weight[lane][i] = w;
    __syncwarp();
    if (lane == 0) {
      R::m(reg = region(0))[i] = M;
      R::l(reg)[i] = L;
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < p.g * D; idx += 32 * kWarps) {
    const int i = idx / D, d = idx - i * D;
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) o += R::acc(region(w), i)[d] * s_weight[w][i];
    R::acc(region(0), i)[d] = o;
  }
  __syncthreads();
  finish_cta<T, D, HP>(p, i4_smem, G::kWarpBytes, 1, b, h, split, nsplit, s_mi);
}

}  // namespace tc
