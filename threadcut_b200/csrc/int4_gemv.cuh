// A few tokens times a weight matrix held in 4 bits: out[m][row] = sum_k x[m][k] w[row][k], the weights being
// S (1 + code/16) + z with an (S, z) of T for each `group` neighbours along k (32, 64 or 128).
//
// Layout (made once, by the caller): tiles of 16 rows x 64 columns, 512 bytes; lane 4r + c of a warp owns 16 bytes
// of a tile, the words of (row r, columns 8c..8c+7), (row r + 8, the same), (row r, columns 32 + 8c..), (row r + 8,
// the same); in a word, code j is column 2j and code j + 4 column 2j + 1. (S, z) as [row tile][group][r][row r | row r + 8].
// Rows and columns behind the matrix have codes and (S, z) of 0.
//
// Products on the tensor cores, a tile's weights being the 16-row operand straight from shared memory and the tokens its 8
// columns. S and z are applied to the sums in fp32:
//   sum_k x (S (1 + code/16) + z) = S P + (S + z) X,   P = sum_k x code/16,  X = sum_k x, over the group's columns in a tile.
// One or two tokens: P as an integer product of the codes, bytes after two masks and a shift (12 instructions for a lane's 32
// codes), with the digits of x, which are otherwise idle columns: x of each 64 columns, scaled by a power of two and rounded
// to a whole number below 2^20 (off by at most 2^-20 of the largest of the 64), is 65536 h + 256 m + l. More tokens: 1 + code/16 and x as they are, 16-bit operands (24 and
// 8; S P + z X then), 8 tokens a product.
//
// A CTA an SM takes neighbouring row tiles, in one or more streams of warps. A stream's warps share out the columns in
// neighbouring runs, each bringing in its run of a row tile, and of the next ones, by bulk copies of a few tiles; their sums are
// added in shared memory in warp order.
//
// Groups of 64, bf16: 2,560 x 4,096 with one token 3.7 us and 19,456 x 2,560 7.5 (start and end of a launch), 151,936 x 2,560
// 35 (6.2 TB/s, bound by memory), with 7 tokens 51 (4.1 TB/s: 98 instructions a tile, 64 % of the issue slots used; an instruction
// waits 1.3 cycles for the one ahead of it, 1.2 for another warp's turn and 0.8 for the ALU pipe). Tokens beside a small ring, and the
// turns of those that do not fit, cost more: 8, 16 and 32 tokens 55, 91 and 235.
#pragma once

#include "int4_attn.cuh"

namespace tc {

constexpr int kGvWarps = 16;
constexpr int kGvMaxStages = 2;          // of a warp's ring (a third gains nothing)
constexpr int kGvPreWait = 1;            // stages filled before the previous kernel has ended
constexpr int kGvPartBytes = 16 * 1024;  // one of the two buffers of sums, at least a row tile's of each stream
constexpr int kGvMaxChunk = 8;           // tiles of a stage (151,936 x 2,560, one token: 34.4 us; 5 35.8, 3 43.0, 10 36.1)
constexpr int kGvDigits = 3;

struct Int4GemvParams {
  const void* x;  // [m][k], row stride sx (swiglu: [m][2k], gate | up)
  const uint8_t* codes;
  const void* params;
  void* out;  // [m][n], row stride so
  int64_t n;
  int k, m;
  int64_t sx, so;
  int swiglu;
  int vec;         // x in 16-byte chunks
  int streams;     // a power of two, 8 at most
  int slice_bits;  // kGvWarps / streams warps share a row tile's columns: 2^slice_bits
  int share, more; // row tiles of a CTA: share, and one more for the first `more` CTAs
  int flush;       // row tiles whose sums a buffer holds
  int part_bytes;  // of a buffer
  int chunk;       // tiles a stage holds
  int stages;
};

__host__ __device__ __forceinline__ int gv_blocks(int k) { return (k + 63) / 64; }

// Bytes of a token's row in shared memory. 16-bit tokens: 16 bytes beside whole tiles, so that the 8 tokens' chunks that a warp
// reads together lie in different banks. Digits: a row for each, an odd number of 64-byte blocks.
__host__ __device__ __forceinline__ int gv_x_bytes(int k, bool digits) {
  return digits ? 64 * (gv_blocks(k) | 1) : 128 * gv_blocks(k) + 16;
}
// Tokens that sums are kept for: in pairs, as a lane reads them.
__host__ __device__ __forceinline__ int gv_sums(int m) { return (m + 1) & ~1; }

// Bytes a tile takes in a stage, its (S, z) included.
__host__ __device__ constexpr int gv_tile_bytes(int g) { return 512 + (g == 32 ? 128 : 64); }
// Sums X: [block of 64 columns][1 or 2 groups][token]; with digits [..][lane c of an operand's four] with a factor beside each.
__host__ __device__ __forceinline__ int gv_sum_bytes(int k, int m, int g, bool digits) {
  return (gv_blocks(k) * (g == 32 ? 2 : 1) * (digits ? 32 : 4 * gv_sums(m)) + 15) / 16 * 16;
}

// Products into d, from 0 (kFirst) or from what is there.
template <bool kFirst>
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kFirst)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float2 lds_float2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
// Codes of two words (rows r and r + 8) as bytes: codes 0, 2, 4, 6, then 1, 3, 5, 7.
__device__ __forceinline__ void i4_bytes(uint32_t w0, uint32_t w1, uint32_t (&a)[4]) {
  a[0] = w0 & 0x0f0f0f0fu;
  a[1] = w1 & 0x0f0f0f0fu;
  a[2] = (w0 >> 4) & 0x0f0f0f0fu;
  a[3] = (w1 >> 4) & 0x0f0f0f0fu;
}
// The digits (l, m, h) of 4 whole numbers below 2^20, as 4 signed bytes each. V: the numbers + 0x8080, whose bytes are the digits
// above 128 less than themselves.
__device__ __forceinline__ void digits4(int v0, int v1, int v2, int v3, uint32_t (&d)[kGvDigits]) {
  d[0] = __byte_perm(__byte_perm(v0, v1, 0x0040), __byte_perm(v2, v3, 0x0040), 0x5410) ^ 0x80808080u;
  d[1] = __byte_perm(__byte_perm(v0, v1, 0x0051), __byte_perm(v2, v3, 0x0051), 0x5410) ^ 0x80808080u;
  d[2] = __byte_perm(__byte_perm(v0, v1, 0x0062), __byte_perm(v2, v3, 0x0062), 0x5410);
}
// The power of two that brings a largest magnitude (0, or 2^-86 at least) into [2^19, 2^20), and its inverse; NaN as the inverse where
// it is not finite, so that it shows.
__device__ __forceinline__ void digit_scale(float most, float& up, float& down) {
  int e = 146 - (int)(__float_as_uint(most) >> 23);
  e = e > 100 ? 100 : e;
  up = __uint_as_float((uint32_t)(127 + e) << 23);
  down = most < INFINITY ? __uint_as_float((uint32_t)(127 - e) << 23) : __uint_as_float(0x7fffffffu);
}

// NT tiles of 8 tokens, or (kInt) up to 2 tokens as digits.
template <typename T, int NT, int G, bool kInt>
__global__ void __launch_bounds__(32 * kGvWarps, 1) int4_gemv_kernel(const __grid_constant__ Int4GemvParams p) {
  constexpr int kXw = G == 32 ? 32 : 64;  // columns of a sum X
  constexpr int XS = 64 / kXw;            // sums a tile
  extern __shared__ __align__(16) uint8_t gv_smem[];
  __shared__ uint64_t s_full[kGvWarps][kGvMaxStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int slices = 1 << p.slice_bits;
  const int stream = warp >> p.slice_bits, slice = warp & (slices - 1);
  const int KT = gv_blocks(p.k);
  const int groups = (p.k + G - 1) / G;
  const int stage_bytes = p.chunk * gv_tile_bytes(G);
  uint8_t* ring = gv_smem + warp * (p.stages * stage_bytes);
  float* part = reinterpret_cast<float*>(gv_smem + kGvWarps * p.stages * stage_bytes);
  float* xsum = part + 2 * (p.part_bytes / 4);
  const int xw = gv_sums(p.m);
  uint8_t* xs = reinterpret_cast<uint8_t*>(xsum) + gv_sum_bytes(p.k, p.m, G, kInt);
  const int x_bytes = gv_x_bytes(p.k, kInt);
  uint64_t* full = s_full[warp];
  if (lane == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncwarp();

  const int cta = blockIdx.x;
  const int rt0 = cta * p.share + (cta < p.more ? cta : p.more), rt1 = rt0 + p.share + (cta < p.more);
  // this warp's run of columns, in tiles
  const int per = KT >> p.slice_bits, over = KT - (per << p.slice_bits);
  const int kt0 = slice * per + (slice < over ? slice : over), nk = per + (slice < over);

  // Lane 0 fetches: its runs of the stream's row tiles, chunk by chunk.
  int f_rt = rt0 + stream, f_kt = kt0, f_s = 0;
  const uint64_t pol = policy_evict_first();
  auto fetch = [&]() {
    if (lane == 0 && f_rt < rt1 && nk > 0) {
      const int left = kt0 + nk - f_kt, nt = left < p.chunk ? left : p.chunk;
      const int g0 = f_kt * 64 / G;
      int g1 = ((f_kt + nt) * 64 + G - 1) / G;
      g1 = g1 < groups ? g1 : groups;
      uint8_t* dst = ring + f_s * stage_bytes;
      mbar_arrive_expect_tx(&full[f_s], nt * 512 + (g1 - g0) * 64);
      bulk_g2s(dst, p.codes + ((int64_t)f_rt * KT + f_kt) * 512, nt * 512, &full[f_s], pol);
      bulk_g2s(dst + p.chunk * 512, static_cast<const uint8_t*>(p.params) + ((int64_t)f_rt * groups + g0) * 64,
               (g1 - g0) * 64, &full[f_s], pol);
      f_kt += nt;
      if (f_kt == kt0 + nk) {
        f_kt = kt0;
        f_rt += p.streams;
      }
      f_s = f_s + 1 == p.stages ? 0 : f_s + 1;
    }
  };
  // Weights are constant: the first tiles are fetched before waiting for the previous kernel. (19,456 x 2,560 7.5 us, 8.2 with
  // nothing fetched before the wait, 8.4 with an L2 prefetch in its place; 151,936 x 2,560 of 7 tokens 53.9, 54.5, 60.3.)
  for (int i = 0; i < kGvPreWait; ++i) fetch();
  pdl_launch();
  pdl_wait();
  for (int i = kGvPreWait; i < p.stages; ++i) fetch();
  {
    // tokens into shared memory, 8 elements a thread, with their groups' sums
    const int chunks = 8 * KT, total = p.m * chunks;
    const T zero = from_f32<T>(0.f);
    for (int base = 32 * warp; base < total; base += 32 * kGvWarps) {  // whole warps: neighbours work out their sums together
      const int idx = base + lane;
      const bool use = idx < total;
      const int m = !use || p.m == 1 ? 0 : idx / chunks, k0 = use ? 8 * (idx - m * chunks) : 0;
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
      float f[8], sum = 0.f;
      if (p.swiglu) {
        // the arithmetic of the 16-bit projection's staging
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float g = to_f32(v[e]);
          v[e] = from_f32<T>(to_f32(from_f32<T>(g / (1.0f + expf(-g)))) * to_f32(u[e]));
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = to_f32(v[e]);
        sum += f[e];
      }
#pragma unroll
      for (int o = 1; o < kXw / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const bool writes = use && (k0 & (kXw - 1)) == 0;
      if constexpr (kInt) {
        float most = fabsf(f[0]);
#pragma unroll
        for (int e = 1; e < 8; ++e) most = fmaxf(most, fabsf(f[e]));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // below the powers of two that fp32 has on both sides: as many times 2^64 (the same for the 8 lanes of a block)
        const bool tiny = most < 0x1p-64f;
        if (tiny) {
          most *= 0x1p64f;
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= 0x1p64f;
        }
        float up, down;
        digit_scale(sum * 0.f == 0.f ? most : INFINITY, up, down);
        if (tiny) down *= 0x1p-64f;
        constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: adding it leaves a whole number in the low bits
        int q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = __float_as_int(fmaf(f[e], up, kWhole)) + (0x8080 - 0x4b400000);
        uint32_t even[kGvDigits], odd[kGvDigits];
        // bytes in the order of a word's codes 0, 2, 4, 6 (columns 0, 4, 1, 5) and 1, 3, 5, 7 (columns 2, 6, 3, 7)
        digits4(q[0], q[4], q[1], q[5], even);
        digits4(q[2], q[6], q[3], q[7], odd);
        if (use) {
          const int chunk = k0 / 8;
          uint8_t* to = xs + m * kGvDigits * x_bytes + (chunk / 8) * 64 + (chunk & 3) * 16 + ((chunk >> 2) & 1) * 8;
#pragma unroll
          for (int i = 0; i < kGvDigits; ++i)
            *reinterpret_cast<uint2*>(to + i * x_bytes) = make_uint2(even[kGvDigits - 1 - i], odd[kGvDigits - 1 - i]);
        }
        if (writes) {
          // lane c's sums of a token are 256 h + m (c even), and l; the products are with codes, 16 times code/16. Powers of two: where
          // they are subnormal, a tiny token's low digits, which would make them inexact, are 0
          float2* to = reinterpret_cast<float2*>(xsum) + (k0 / kXw) * 4 + 2 * m;
          to[0] = make_float2(sum, 16.f * down);
          to[1] = make_float2(0.f, 0.0625f * down);
        }
      } else {
        if (use) {
          uint4 a;
          memcpy(&a, v, 16);
          *reinterpret_cast<uint4*>(xs + m * x_bytes + 2 * k0) = a;
        }
        if (writes) xsum[(k0 / kXw) * xw + m] = sum;
      }
    }
    if (p.m < xw) {  // the pair's other token
      for (int idx = threadIdx.x; idx < KT * XS; idx += 32 * kGvWarps) {
        if constexpr (kInt)
          reinterpret_cast<float4*>(xsum)[idx * 2 + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
        else
          xsum[idx * xw + p.m] = 0.f;
      }
    }
  }
  __syncthreads();

  // This lane's operand is column r of the tokens: token nt 8 + r, or (kInt) digit r & 3 of token r / 4, the fourth column being
  // the last digit again. Columns that no token has repeat another's: nothing reads their sums.
  uint32_t xa0[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int token = kInt ? r / 4 : nt * 8 + r, last = p.m - 1;
    const int digit = (r & 3) < kGvDigits ? r & 3 : kGvDigits - 1;
    xa0[nt] = smem_u32(xs) + ((token < last ? token : last) * (kInt ? kGvDigits : 1) + (kInt ? digit : 0)) * x_bytes + 16 * c;
  }
  // and its sums are those of columns 2c and 2c + 1
  uint32_t sum0[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int token = nt * 8 + 2 * c;
    sum0[nt] = smem_u32(xsum) + (kInt ? 8 * c : 4 * (token < xw ? token : 0));
  }
  const uint32_t sum_step = kInt ? 32 : 4 * xw;
  const int high = c & 1 ? 0 : 256;  // (kInt) what column 2c counts: an odd lane's columns are both the last digit
  int s = 0, phase = 0, buf = 0;
  bool alive = true;
  for (int f0 = rt0; f0 < rt1; f0 += p.flush, buf ^= 1) {
    const int nf = rt1 - f0 < p.flush ? rt1 - f0 : p.flush;  // (flush is a multiple of streams)
    float* pb = part + buf * (p.part_bytes / 4);             // [nf][slices][m][16]
    for (int f = stream; f < nf; f += p.streams) {
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
      for (int kt = kt0; kt < kt0 + nk;) {
        if (alive && !__all_sync(0xffffffffu, mbar_wait(&full[s], phase, TC_DEVERR_PIPE_TIMEOUT))) {
          // given up by the whole warp for the rest of the launch, and only once its copies had another chance to end
          for (int i = 0; i < p.stages; ++i)
            mbar_wait(&full[s + i < p.stages ? s + i : s + i - p.stages], phase ^ (s + i >= p.stages), TC_DEVERR_PIPE_TIMEOUT);
          alive = false;
        }
        if (!alive) break;
        const uint32_t st = smem_u32(ring) + s * stage_bytes;
        const int end = kt + p.chunk < kt0 + nk ? kt + p.chunk : kt0 + nk;
        uint32_t code = st + 16 * lane, param = st + p.chunk * 512 + 8 * r, xk = kt * (kInt ? 64 : 128), xx = kt * XS * sum_step;
#pragma unroll 2
        for (; kt < end; ++kt, code += 512, xk += kInt ? 64 : 128, xx += XS * sum_step) {
          uint32_t w[4], q[XS][2];
          lds_words(code, w);
#pragma unroll
          for (int x = 0; x < XS; ++x) lds_words(param + 64 * x, q[x]);
          param += G == 32 ? 128 : G == 64 ? 64 : (kt & 1) * 64;  // (G = 128: two tiles a group)
          if (G == 32 && 2 * kt + 1 >= groups) q[XS - 1][0] = q[XS - 1][1] = 0u;  // (no such group: nothing was copied)
          if constexpr (kInt) {
            uint32_t b[4], a[4];
            lds_words(xa0[0] + xk, b);
            int d[XS][4];
            i4_bytes(w[0], w[1], a);
            mma_u8s8<true>(d[0], a, b[0], b[1]);
            i4_bytes(w[2], w[3], a);
            mma_u8s8<XS == 2>(d[XS - 1], a, b[2], b[3]);
#pragma unroll
            for (int x = 0; x < XS; ++x) {
              const float2 X = lds_float2(sum0[0] + xx + x * 32);
              // (at most 64 * 15 * (256 * 16 + 128) < 2^24)
              const float P0 = X.y * (float)(high * d[x][0] + d[x][1]), P1 = X.y * (float)(high * d[x][2] + d[x][3]);
              const float s0 = Mma<T>::lo(q[x][0]), s1 = Mma<T>::lo(q[x][1]);
              acc[0][0] = fmaf(s0 + Mma<T>::hi(q[x][0]), X.x, fmaf(s0, P0, acc[0][0]));
              acc[0][2] = fmaf(s1 + Mma<T>::hi(q[x][1]), X.x, fmaf(s1, P1, acc[0][2]));
            }
          } else {
            uint32_t a[4][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              a[2 * x][0] = i4_ones<T, 0>(w[2 * x]);
              a[2 * x][1] = i4_ones<T, 0>(w[2 * x + 1]);
              a[2 * x][2] = i4_ones<T, 1>(w[2 * x]);
              a[2 * x][3] = i4_ones<T, 1>(w[2 * x + 1]);
              a[2 * x + 1][0] = i4_ones<T, 2>(w[2 * x]);
              a[2 * x + 1][1] = i4_ones<T, 2>(w[2 * x + 1]);
              a[2 * x + 1][2] = i4_ones<T, 3>(w[2 * x]);
              a[2 * x + 1][3] = i4_ones<T, 3>(w[2 * x + 1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t b0[4], b1[4];
              lds_words(xa0[nt] + xk, b0);
              lds_words(xa0[nt] + xk + 64, b1);
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
                const float2 X = lds_float2(sum0[nt] + xx + x * sum_step);
                const float s0 = Mma<T>::lo(q[x][0]), z0 = Mma<T>::hi(q[x][0]);
                const float s1 = Mma<T>::lo(q[x][1]), z1 = Mma<T>::hi(q[x][1]);
                acc[nt][0] = fmaf(z0, X.x, fmaf(s0, d[x][0], acc[nt][0]));
                acc[nt][1] = fmaf(z0, X.y, fmaf(s0, d[x][1], acc[nt][1]));
                acc[nt][2] = fmaf(z1, X.x, fmaf(s1, d[x][2], acc[nt][2]));
                acc[nt][3] = fmaf(z1, X.y, fmaf(s1, d[x][3], acc[nt][3]));
              }
            }
          }
        }
        __syncwarp();  // the stage may be filled again
        fetch();
        if (++s == p.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      float* o = pb + (f * slices + slice) * p.m * 16 + r;
      if constexpr (kInt) {
        const float a0 = acc[0][0] + __shfl_xor_sync(0xffffffffu, acc[0][0], 1);
        const float a1 = acc[0][2] + __shfl_xor_sync(0xffffffffu, acc[0][2], 1);
        if ((c & 1) == 0 && c / 2 < p.m) {
          o[c / 2 * 16] = a0;
          o[c / 2 * 16 + 8] = a1;
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int m = nt * 8 + 2 * c + e;
            if (m < p.m) {
              o[m * 16] = acc[nt][e];
              o[m * 16 + 8] = acc[nt][2 + e];
            }
          }
      }
    }
    __syncthreads();  // (the other buffer's readers are a barrier ahead of its next writers)
    const int outs = nf * p.m * 16;
    for (int idx = threadIdx.x; idx < outs; idx += 32 * kGvWarps) {
      const int rr = idx & 15, fm = idx >> 4;
      const int f = p.m == 1 ? fm : fm / p.m, m = fm - f * p.m;
      const int64_t row = (int64_t)(f0 + f) * 16 + rr;
      const float* o = pb + (f * slices * p.m + m) * 16 + rr;
      float sum = 0.f;
#pragma unroll 8
      for (int w = 0; w < slices; ++w) sum += o[w * p.m * 16];
      if (row < p.n) static_cast<T*>(p.out)[m * p.so + row] = from_f32<T>(sum);
    }
  }
}

}  // namespace tc
