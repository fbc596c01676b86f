// Attention of single query rows over two ranges of keys: the plain kernel behind the windowed prefill
// (sinks, then the window) and the shared-prefix decode (the prefix, then the sequence's suffix) for what
// their tensor-core kernels do not take (fp32, other head sizes, unaligned rows, a scale <= 0).
//
//   out = sum_j p_j v_j, p = softmax over the visible j of scale q.k_j
//
// One CTA per query row; each of its warps takes every kRowsWarps-th group of 32 keys, a lane per key for
// the scores (the row is in shared memory as fp32), then a lane per element for P V, with a running
// maximum and sum; the warps' states are joined in shared memory. No visible key, or only scores of -inf: zeros.
#pragma once

#include <stdint.h>

namespace tc {

constexpr int kRowsWarps = 4;
constexpr int kRowsMaxDim = 256;

struct RowsParams {
  const void* q;  // query head i of KV head h of sequence b at b*sq_b + h*sq_h + i*sq_g + pos*sq_p
  void* out;
  int64_t sq_b, sq_h, sq_g, sq_p, so_b, so_h, so_g, so_p;
  const void *k0, *v0, *k1, *v1;  // the two ranges' tensors (the same one for a window)
  int64_t sk0_b, sk0_h, sk0_n, sv0_b, sv0_h, sv0_n;
  int64_t sk1_b, sk1_h, sk1_n, sv1_b, sv1_h, sv1_n;
  int batch, hkv, g, d;
  int64_t lq;
  // window > 0: query pos sees rows [0, min(sinks, w0)) of range 0 and [w0, lk - lq + pos] of range 1,
  // w0 = max(0, lk - lq + pos + 1 - window). window == 0: rows [0, n0) of range 0 and [0, lengths[b]) of
  // range 1 (lengths null: n1; clamped into [0, n1]).
  int64_t window, sinks, lk, n0, n1;
  const int32_t* lengths;
  float c;  // scale * log2(e)
};

template <typename T>
__global__ void __launch_bounds__(32 * kRowsWarps) rows_attn_kernel(const __grid_constant__ RowsParams p) {
  __shared__ float sq[kRowsMaxDim];
  __shared__ float s_m[kRowsWarps], s_l[kRowsWarps], s_o[kRowsWarps][kRowsMaxDim];
  constexpr int E = kRowsMaxDim / 32;
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // rows in the order (batch, KV head, position, query head of the group)
  int64_t r = blockIdx.x;
  const int i = (int)(r % p.g);
  r /= p.g;
  const int64_t pos = r % p.lq;
  r /= p.lq;
  const int h = (int)(r % p.hkv);
  const int64_t b = r / p.hkv;
  int64_t n0 = p.n0, first1 = 0, end1 = p.n1;
  if (p.window > 0) {
    const int64_t limit = p.lk - p.lq + pos;
    first1 = limit + 1 - p.window < 0 ? 0 : limit + 1 - p.window;
    n0 = p.sinks < first1 ? p.sinks : first1;
    end1 = limit + 1;
  } else if (p.lengths != nullptr) {
    end1 = p.lengths[b] < 0 ? 0 : (p.lengths[b] < p.n1 ? p.lengths[b] : p.n1);
  }
  const int64_t total = n0 + end1 - first1;
  const T* q = static_cast<const T*>(p.q) + b * p.sq_b + h * p.sq_h + i * p.sq_g + pos * p.sq_p;
  for (int e = threadIdx.x; e < p.d; e += blockDim.x) sq[e] = to_f32(q[e]);
  __syncthreads();
  const T* k0 = static_cast<const T*>(p.k0) + b * p.sk0_b + h * p.sk0_h;
  const T* v0 = static_cast<const T*>(p.v0) + b * p.sv0_b + h * p.sv0_h;
  const T* k1 = static_cast<const T*>(p.k1) + b * p.sk1_b + h * p.sk1_h;
  const T* v1 = static_cast<const T*>(p.v1) + b * p.sv1_b + h * p.sv1_h;
  float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int x = 0; x < E; ++x) acc[x] = 0.f;
  for (int64_t j0 = 32 * (int64_t)warp; j0 < total; j0 += 32 * kRowsWarps) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    if (j < total) {
      const T* kr = j < n0 ? k0 + j * p.sk0_n : k1 + (j - n0 + first1) * p.sk1_n;
      float dot = 0.f;
      for (int e = 0; e < p.d; ++e) dot = fmaf(sq[e], to_f32(kr[e]), dot);
      s = dot * p.c;
    }
    const float mn = fmaxf(m, warp_max(s));
    const float a = m == -INFINITY ? 0.f : exp2f(m - mn);
    // a group of scores that are all -inf (the first ones of a warp) has weights 0, not exp2(inf - inf)
    const float w = j < total ? exp2f(s - (mn == -INFINITY ? 0.f : mn)) : 0.f;
    l = l * a + warp_sum(w);
#pragma unroll
    for (int x = 0; x < E; ++x) acc[x] *= a;
    m = mn;
    const int cnt = total - j0 < 32 ? (int)(total - j0) : 32;
    for (int t = 0; t < cnt; ++t) {
      const float wt = __shfl_sync(0xffffffffu, w, t);
      const int64_t jj = j0 + t;
      const T* vr = jj < n0 ? v0 + jj * p.sv0_n : v1 + (jj - n0 + first1) * p.sv1_n;
#pragma unroll
      for (int x = 0; x < E; ++x)
        if (lane + 32 * x < p.d) acc[x] = fmaf(wt, to_f32(vr[lane + 32 * x]), acc[x]);
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int x = 0; x < E; ++x) s_o[warp][lane + 32 * x] = acc[x];
  __syncthreads();
  float M = -INFINITY, L = 0.f, f[kRowsWarps];
#pragma unroll
  for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, s_m[w]);
#pragma unroll
  for (int w = 0; w < kRowsWarps; ++w) {
    f[w] = s_l[w] == 0.f ? 0.f : exp2f(s_m[w] - M);  // a warp with no keys, or all at -inf, has l = 0
    L += f[w] * s_l[w];
  }
  T* out = static_cast<T*>(p.out) + b * p.so_b + h * p.so_h + i * p.so_g + pos * p.so_p;
  for (int e = threadIdx.x; e < p.d; e += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) o += f[w] * s_o[w][e];
    out[e] = from_f32<T>(L == 0.f ? 0.f : o / L);
  }
}

}  // namespace tc
