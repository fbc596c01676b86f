// A few tokens times a weight matrix held in 4 bits: out[m][row] = sum_k x[m][k] w[row][k], the weights being
// S (1 + code/16) + z with an (S, z) of T for each `group` neighbours along k (32, 64 or 128).
//
// Layout (made once, by the caller): tiles of 16 rows x 64 columns, 512 bytes; lane 4r + c of a warp owns 16 bytes
// of a tile, the words of (row r, columns 8c..8c+7), (row r + 8, the same), (row r, columns 32 + 8c..), (row r + 8,
// the same); in a word, code j is column 2j and code j + 4 column 2j + 1. (S, z) as [row tile][group][r][row r | row r + 8].
// Rows and columns behind the matrix have codes and (S, z) of 0.
//
// Products on the tensor cores, the weights as the 16-row operand straight from registers, the tokens as its 8
// columns: with one token seven of them idle, which costs nothing, as the bytes of the weights are the bound.
// 1 + code/16 goes into the product as it is; S and z are applied to the sums in fp32:
//   sum_k x (S (1 + code/16) + z) = S P + z X,     P = sum_k x (1 + code/16),  X = sum_k x over the group's columns.
// A warp takes every 8th tile of a row of tiles; the 8 warps' sums are added in shared memory in warp order.
#pragma once

#include "int4_attn.cuh"

namespace tc {

constexpr int kGvWarps = 8;
constexpr int kGvStages = 8;     // tiles in flight a warp
constexpr int kGvPartBytes = 16 * 1024;  // one of the two buffers of sums

struct Int4GemvParams {
  const void* x;  // [m][k], row stride sx (swiglu: [m][2k], gate | up)
  const uint8_t* codes;
  const void* params;
  void* out;  // [m][n], row stride so
  int64_t n;
  int k, m;
  int64_t sx, so;
  int swiglu;
  int vec;       // x in 16-byte chunks
  int x_stride;  // elements between the tokens' rows in shared memory
  int flush;     // row tiles whose sums a buffer holds
};

__host__ __device__ __forceinline__ int gv_blocks(int k) { return (k + 63) / 64; }

// Elements of a token's row in shared memory: whole tiles, and 16 bytes more, so that the 8 tokens' chunks that a
// warp reads together lie in different banks.
__host__ __device__ __forceinline__ int gv_x_stride(int k) { return 64 * gv_blocks(k) + 8; }

// Sums X kept for each group: the tokens, in pairs as a lane reads them.
__host__ __device__ __forceinline__ int gv_sums(int m) { return (m + 1) & ~1; }

template <int G>
__host__ __device__ constexpr int gv_stage_bytes() {
  return 512 + (G == 32 ? 128 : 64);
}

template <typename T, int NT, int G>
__global__ void __launch_bounds__(32 * kGvWarps) int4_gemv_kernel(const __grid_constant__ Int4GemvParams p) {
  constexpr int kParamBytes = G == 32 ? 128 : 64;
  constexpr int kStage = gv_stage_bytes<G>();
  constexpr int kXw = G == 32 ? 32 : 64;  // columns of a sum X
  constexpr int XS = 64 / kXw;            // sums a tile
  extern __shared__ __align__(16) uint8_t gv_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int KT = gv_blocks(p.k);
  const int groups = (p.k + G - 1) / G;
  uint8_t* ring = gv_smem + warp * (kGvStages * kStage);
  float* part = reinterpret_cast<float*>(gv_smem + kGvWarps * kGvStages * kStage);
  float* xsum = part + 2 * (kGvPartBytes / 4);  // [KT * XS][xw]
  const int xw = gv_sums(p.m);
  T* xs = reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(xsum) + (KT * XS * xw * 4 + 15) / 16 * 16);

  const int64_t row_tiles = (p.n + 15) / 16;
  const int64_t rt0 = row_tiles * blockIdx.x / gridDim.x, rt1 = row_tiles * (blockIdx.x + 1) / gridDim.x;
  const int nk = warp < KT ? (KT - warp + kGvWarps - 1) / kGvWarps : 0;  // this warp's tiles of a row
  const uint8_t* params = static_cast<const uint8_t*>(p.params);
  const uint32_t ring_s = smem_u32(ring);

  // The weights do not depend on the previous kernel: the first tiles are fetched before waiting for it.
  int64_t f_rt = rt0;
  int f_kt = warp, f_s = 0;
  auto fetch = [&]() {
    if (f_rt < rt1 && nk > 0) {
      const uint32_t dst = ring_s + f_s * kStage;
      copy_async<16>(dst + 16 * lane, p.codes + (f_rt * KT + f_kt) * 512 + 16 * lane, true);
      const int g0 = G == 32 ? 2 * f_kt : f_kt * 64 / G;
      if (lane < kParamBytes / 16) {
        // (G = 32: the last tile's second half may lie behind the last group)
        const bool in = G != 32 || g0 + lane / 4 < groups;
        copy_async<16>(dst + 512 + 16 * lane, params + (f_rt * groups + g0) * 64 + (in ? 16 * lane : 0), in);
      }
      f_kt += kGvWarps;
      if (f_kt >= KT) {
        f_kt = warp;
        ++f_rt;
      }
      f_s = f_s + 1 == kGvStages ? 0 : f_s + 1;
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kGvStages - 1; ++i) fetch();

  pdl_launch();
  pdl_wait();
  {
    // tokens into shared memory, 8 elements a thread, with their groups' sums
    const int chunks = 8 * KT;
    const T zero = from_f32<T>(0.f);
    const int total = p.m * chunks;
    for (int base = 0; base < total; base += 32 * kGvWarps) {  // every thread: neighbours add up their sums
      const int idx = base + threadIdx.x;
      const bool use = idx < total;
      const int m = use ? idx / chunks : 0, k0 = use ? 8 * (idx - m * chunks) : 0;
      const T* xr = static_cast<const T*>(p.x) + m * p.sx;
      T v[8], u[8];
      if (use && p.vec && k0 + 8 <= p.k) {
        const uint4 a = *reinterpret_cast<const uint4*>(xr + k0);
        memcpy(v, &a, 16);
        if (p.swiglu) {
          const uint4 b = *reinterpret_cast<const uint4*>(xr + p.k + k0);
          memcpy(u, &b, 16);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = use && k0 + e < p.k ? xr[k0 + e] : zero;
          u[e] = use && p.swiglu && k0 + e < p.k ? xr[p.k + k0 + e] : zero;
        }
      }
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (p.swiglu) {
          // the arithmetic of the 16-bit projection's staging
          const float g = to_f32(v[e]);
          v[e] = from_f32<T>(to_f32(from_f32<T>(g / (1.0f + expf(-g)))) * to_f32(u[e]));
        }
        sum += to_f32(v[e]);
      }
      if (use) {
        uint4 a;
        memcpy(&a, v, 16);
        *reinterpret_cast<uint4*>(xs + (int64_t)m * p.x_stride + k0) = a;
      }
#pragma unroll
      for (int o = 1; o < kXw / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (use && (k0 & (kXw - 1)) == 0) xsum[(k0 / kXw) * xw + m] = sum;
    }
    if (p.m < xw)  // the pair's other column
      for (int idx = threadIdx.x; idx < KT * XS; idx += 32 * kGvWarps) xsum[idx * xw + p.m] = 0.f;
  }
  __syncthreads();

  int s = 0, buf = 0;
  for (int64_t f0 = rt0; f0 < rt1; f0 += p.flush, buf ^= 1) {
    const int nf = rt1 - f0 < p.flush ? (int)(rt1 - f0) : p.flush;
    float* pb = part + buf * (kGvPartBytes / 4);  // [nf][warps][m][16]
    for (int f = 0; f < nf; ++f) {
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
      for (int i = 0, kt = warp; i < nk; ++i, kt += kGvWarps) {
        fetch();
        copy_wait<kGvStages - 1>();
        __syncwarp();  // the (S, z) came through other lanes
        const uint32_t st = ring_s + s * kStage;
        uint32_t w[4], q[XS][2];
        lds_words(st + 16 * lane, w);
#pragma unroll
        for (int x = 0; x < XS; ++x) lds_words(st + 512 + 64 * x + 8 * r, q[x]);
        uint32_t a[4][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          a[2 * x][0] = i4_mant<T, 0>(w[2 * x]);
          a[2 * x][1] = i4_mant<T, 0>(w[2 * x + 1]);
          a[2 * x][2] = i4_mant<T, 1>(w[2 * x]);
          a[2 * x][3] = i4_mant<T, 1>(w[2 * x + 1]);
          a[2 * x + 1][0] = i4_mant<T, 2>(w[2 * x]);
          a[2 * x + 1][1] = i4_mant<T, 2>(w[2 * x + 1]);
          a[2 * x + 1][2] = i4_mant<T, 3>(w[2 * x]);
          a[2 * x + 1][3] = i4_mant<T, 3>(w[2 * x + 1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int m = nt * 8 + r;
          uint32_t b0[4] = {0u, 0u, 0u, 0u}, b1[4] = {0u, 0u, 0u, 0u};
          if (m < p.m) {
            const uint32_t xa = smem_u32(xs + (int64_t)m * p.x_stride + 64 * kt + 8 * c);
            lds_words(xa, b0);
            lds_words(xa + 64, b1);
          }
          float d[XS][4];
#pragma unroll
          for (int x = 0; x < XS; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[x][e] = 0.f;
          Mma<T>::run(d[0], a[0], b0[0], b0[1]);
          Mma<T>::run(d[0], a[1], b0[2], b0[3]);
          Mma<T>::run(d[XS - 1], a[2], b1[0], b1[1]);
          Mma<T>::run(d[XS - 1], a[3], b1[2], b1[3]);
#pragma unroll
          for (int x = 0; x < XS; ++x) {
            float2 X = make_float2(0.f, 0.f);
            if (nt * 8 + 2 * c < xw) X = *reinterpret_cast<const float2*>(xsum + (kt * XS + x) * xw + nt * 8 + 2 * c);
            const float s0 = Mma<T>::lo(q[x][0]), z0 = Mma<T>::hi(q[x][0]);
            const float s1 = Mma<T>::lo(q[x][1]), z1 = Mma<T>::hi(q[x][1]);
            acc[nt][0] = fmaf(z0, X.x, fmaf(s0, d[x][0], acc[nt][0]));
            acc[nt][1] = fmaf(z0, X.y, fmaf(s0, d[x][1], acc[nt][1]));
            acc[nt][2] = fmaf(z1, X.x, fmaf(s1, d[x][2], acc[nt][2]));
            acc[nt][3] = fmaf(z1, X.y, fmaf(s1, d[x][3], acc[nt][3]));
          }
        }
        __syncwarp();  // the stage may be filled again
        s = s + 1 == kGvStages ? 0 : s + 1;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int m = nt * 8 + 2 * c + e;
          if (m < p.m) {
            float* o = pb + ((f * kGvWarps + warp) * p.m + m) * 16 + r;
            o[0] = acc[nt][e];
            o[8] = acc[nt][2 + e];
          }
        }
    }
    __syncthreads();  // (the other buffer's readers are a barrier ahead of its next writers)
    const int outs = nf * p.m * 16;
    for (int idx = threadIdx.x; idx < outs; idx += 32 * kGvWarps) {
      const int rr = idx & 15, fm = idx >> 4;
      const int f = fm / p.m, m = fm - f * p.m;
      const int64_t row = (f0 + f) * 16 + rr;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kGvWarps; ++w) sum += pb[((f * kGvWarps + w) * p.m + m) * 16 + rr];
      if (row < p.n) static_cast<T*>(p.out)[m * p.so + row] = from_f32<T>(sum);
    }
  }
  copy_wait<0>();
}

}  // namespace tc
