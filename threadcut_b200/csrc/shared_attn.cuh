// Decode attention of a batch over ONE shared prefix and each sequence's own suffix, on the tcgen05 tensor
// cores (sm_100a). The prefix of a KV head meets all batch*g query rows that share it in one product, so
// its K and V are read once for the batch; a suffix meets its sequence's g rows.
//
//   out = sum_parts 2^(m_p - M) o_p / sum_parts 2^(m_p - M) l_p,   M = max m_p
//
// over parts (slices of the prefix, slices of the suffix), each part's o_p = sum_j 2^(s_j - m_p) v_j and
// l_p = sum_j 2^(s_j - m_p) with s_j = scale log2(e) q.k_j and m_p a running maximum: the log-sum-exp merge of
// threadcut/flash_decode.py:68-69 over both kinds of slices.
//
// shared_attn_kernel: a CTA per part (prefix: KV head, tile of up to 128 query rows, slice; suffix: sequence, KV
// head, slice), two resident per SM at d <= 128, one waiting for memory or softmax while the other multiplies:
//   warp 4 (one lane): TMA, the query rows once, then K and V tiles of 64 keys through a ring of slots in the
//                      order the products take them (K0 K1 V0 K2 V1 ...).
//   warp 5 (one lane): tcgen05.mma: S = Q K^T (128 x 64 keys x d, fp32 in TMEM, two S buffers so the next tile's S
//                      is there when a softmax ends), O += P V with P from TMEM.
//   warps 0-3:         softmax, a thread per query row; warps without live rows leave at once (a suffix has g
//                      rows). The maximum is kept until a tile passes it by 2^8, so O is rescaled rarely.
// The weights 2^(s_j - m_p) enter O += P V rounded once to T, as in the causal prefill; the sums l_p add them unrounded.
// (The split-KV decode kernels hand them over in two 16-bit parts.) Half a step of bf16 is 2^-8 of a weight: against
// float64 the result is off by 2.2e-3 of its norm, of which its own rounding to bf16 makes 1.65e-3 (fp16 2.9e-4 of
// 2.1e-4). Two parts, the second in the other half of the S buffer, bring the 1.65e-3 and double the products of P:
// 2 sequences of 1,536 + 40 tokens 9.0 us instead of 8.6, 8 of 16,384 + 700 23.2 instead of 20.0, 64 of 98,304 + 1,024
// 165 instead of 139. A caller who needs the last bits has decode_attention_batched.
// Up to 128 rows the loop runs at the DRAM's pace (b = 1 over 98,304 rows: 66 us, 6.1 TB/s); with more, each row tile
// fetches the tiles from L2 again and 256 rows take 118 us for 98,304 keys. One CTA an SM that multiplied each tile
// with two row tiles moved half the bytes from L2 and took 125 us: its two chains of softmax and products, not
// the fetches, set the pace, and two smaller CTAs overlap start and end better (16,384 keys: 39 us against 50).
// Rows behind a slice's end inside its last tile: the scores are masked and the staged V rows zeroed, so
// whatever memory holds there is not met. shared_merge_kernel joins the parts.
#pragma once

#include <type_traits>

#include "tc_common.cuh"

namespace tc {

constexpr int kShKeys = 64;       // keys per K/V tile
constexpr int kShThreads = 192;   // 4 softmax warps, TMA, MMA
constexpr uint32_t kShSpin = 1u << 20;  // mbarrier polls before a wait gives up (about a second)
constexpr float kShLazyMax = 8.f;

template <int D>
struct SharedGeom {
  static constexpr int kBoxes = D / 64;
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kSlotBytes = kShKeys * D * 2;
  static constexpr int kBoxBytes = kShKeys * 128;
  // two CTAs per SM at D <= 128 (2 x 113 KB of shared memory, 2 x 256 TMEM columns), one at D = 256
  static constexpr int kSlots = D == 64 ? 10 : 5;
  static constexpr int kCtasPerSm = D == 256 ? 1 : 2;
  static constexpr int kTmemCols = D == 256 ? 512 : 256;
  static constexpr int kSmem = 1024 + kQBytes + kSlots * kSlotBytes;
};

struct SharedParams {
  CUtensorMap tmq;   // (d, g, batch, hkv), box (64, g, 128 / g, 1): the rows of a prefix part
  CUtensorMap tmq1;  // the same, box (64, g, 1, 1): the rows of a suffix part
  CUtensorMap tmkp, tmvp;  // prefix: (d, n, hkv, 1), box (64, 64, 1, 1); paged (d, page rows, hkv, pages), box (64, 32, 1, 1)
  CUtensorMap tmk, tmv;    // suffixes: (d, m, hkv, batch), box (64, 64, 1, 1)
  const int32_t* lengths;  // [batch] or null (= m)
  const int32_t* tiles;    // paged prefix: [n_tiles][3] = page, first row, rows <= 32; key tile j is entries 2j, 2j + 1
  int n_tiles;
  int num_pages, page_rows;
  int batch, hkv, g;
  int bt;           // sequences per prefix row tile (128 / g)
  int row_tiles;    // cdiv(batch, bt)
  int n, m;
  int np;           // prefix parts per (KV head, row tile): the first hkv*row_tiles*np CTAs
  int ns;           // suffix parts per (sequence, KV head)
  int warm;         // the whole launch is resident at once
  float c;          // scale * log2(e)
  float* o;         // [np + ns][batch*hkv*g][d] unnormalised
  float2* ml;       // [np + ns][batch*hkv*g] (maximum in log2, sum)
};

// 32 bytes to a 32-byte aligned address: a whole sector a thread.
__device__ __forceinline__ void st_v8(float* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// mbarriers and flags of a CTA.
template <int kSlots>
struct SharedCtl {
  uint64_t q_full, full[kSlots], empty[kSlots], s_full[2], p_full[2], pv_done[2], fin;
  uint32_t tmem;
};

__device__ __forceinline__ int shared_suffix(const SharedParams& p, int b) {
  const int len = p.lengths != nullptr ? __ldcg(p.lengths + b) : p.m;
  return len < 0 ? 0 : (len > p.m ? p.m : len);
}

// Key tiles [t0, t1) of part s of np over `tiles` tiles.
__device__ __forceinline__ void shared_range(int tiles, int s, int np, int& t0, int& t1) {
  t0 = (int)((int64_t)tiles * s / np);
  t1 = (int)((int64_t)tiles * (s + 1) / np);
}

template <typename T, int D, bool kPaged>
__global__ void __launch_bounds__(kShThreads, SharedGeom<D>::kCtasPerSm)
    shared_attn_kernel(const __grid_constant__ SharedParams p) {
  using G = SharedGeom<D>;
  using Ctl = SharedCtl<G::kSlots>;
  constexpr int kSlots = G::kSlots;
  constexpr int kTmaWarp = 4, kMmaWarp = 5;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // All shared memory is dynamic, so that two CTAs fit an SM: the tiles from the first 1 KB boundary on,
  // and the control block in whichever part of the 1 KB of slack is not spent on reaching it.
  extern __shared__ uint8_t smem_raw[];
  const uint32_t gap = (1024 - (smem_u32(smem_raw) & 1023)) & 1023;
  uint8_t* sQ = smem_raw + gap;      // D/64 boxes of 128 rows x 128 B
  uint8_t* sKV = sQ + G::kQBytes;    // slot s: D/64 boxes of 64 rows x 128 B
  static_assert(sizeof(Ctl) <= 512, "the control block must fit either side of the tiles");
  Ctl& ctl = *reinterpret_cast<Ctl*>(gap >= 512 ? smem_raw : sKV + kSlots * G::kSlotBytes);
  uint64_t *full = ctl.full, *empty = ctl.empty, *s_full = ctl.s_full, *p_full = ctl.p_full, *pv_done = ctl.pv_done;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- this CTA's part
  const int prefix_ctas = p.hkv * p.row_tiles * p.np;
  const bool prefix = (int)blockIdx.x < prefix_ctas;
  int part, h, b0, s0 = 0, live;  // b0: first sequence of the rows; live: query rows
  if (prefix) {
    // row tiles of one slice are neighbours in the launch order: the later finds K and V in L2
    int i = blockIdx.x;
    b0 = (i % p.row_tiles) * p.bt;
    i /= p.row_tiles;
    h = i % p.hkv;
    part = i / p.hkv;
    live = (p.batch - b0 < p.bt ? p.batch - b0 : p.bt) * p.g;
  } else {
    int i = blockIdx.x - prefix_ctas;
    s0 = i % p.ns;
    i /= p.ns;
    h = i % p.hkv;
    b0 = i / p.hkv;
    live = p.g;
    part = p.np + s0;
  }
  const int nlive = (live + 31) >> 5;  // softmax warps with rows
  const CUtensorMap* mq = prefix ? &p.tmq : &p.tmq1;
  const CUtensorMap* mk = prefix ? &p.tmkp : &p.tmk;
  const CUtensorMap* mv = prefix ? &p.tmvp : &p.tmv;
  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], nlive);
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(&ctl.fin, 1);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(&ctl.tmem, G::kTmemCols);
  if (warp == kTmaWarp && lane == 0) {
    prefetch_tensormap(mq);
    prefetch_tensormap(mk);
    prefetch_tensormap(mv);
    if (!kPaged && prefix && p.warm) {
      // The first tiles of a prefix part into L2 before the wait below (its range needs no device data; rows still
      // being written are read by the copies later): 8 sequences of 16,384 + 700 tokens 20.9 -> 20.1 us. Not in
      // launches of several waves, whose later CTAs would only fetch twice.
      int w0, w1;
      shared_range((p.n + kShKeys - 1) / kShKeys, part, p.np, w0, w1);
      for (int t = w0; t < w1 && t < w0 + 2; ++t)
        for (int bx = 0; bx < G::kBoxes; ++bx) {
          tma_prefetch_4d(mk, bx * 64, t * kShKeys, h, 0);
          tma_prefetch_4d(mv, bx * 64, t * kShKeys, h, 0);
        }
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = ctl.tmem;  // S buffer i (and P over it) at +64i, O at +128
  const uint32_t tO = tmem + 128;
  // The next kernel is let in after the allocation above: its CTAs may hold TMEM while they wait for this one.
  pdl_launch();
  pdl_wait();  // queries, lengths, tables and the cache may be the previous kernel's
  int t0, t1, end;  // this part's key tiles, and the keys of its source
  if (prefix) {
    end = p.n;
    shared_range(kPaged ? (p.n_tiles + 1) / 2 : (p.n + kShKeys - 1) / kShKeys, part, p.np, t0, t1);
  } else {
    end = shared_suffix(p, b0);
    shared_range((end + kShKeys - 1) / kShKeys, s0, p.ns, t0, t1);
  }
  const int nt = t1 - t0;  // 0: nothing in this slice, every role falls through; the merge knows and skips it
  const bool paged = kPaged && prefix;
  // Place of K_j and V_j in the ring's order K0 K1 V0 K2 V1 ... (the order the products take them).
  auto k_at = [](int j) { return j < 2 ? j : 2 * j - 1; };
  auto v_at = [nt](int j) { return j < nt - 1 ? 2 * j + 2 : 2 * nt - 1; };
  // (page, first row, rows) of sub-tile c of key tile t; a table entry outside the pool counts as empty
  auto sub = [&](int t, int c) -> int3 {
    const int i = 2 * t + c;
    if (i >= p.n_tiles) return make_int3(p.num_pages, 0, 0);
    const int32_t* e = p.tiles + 3 * (int64_t)i;
    const int page = e[0], row = e[1], rows = e[2];
    if (page < 0 || page >= p.num_pages || row < 0 || rows < 0 || rows > 32 || row + rows > p.page_rows)
      return make_int3(p.num_pages, 0, 0);
    return make_int3(page, row, rows);
  };

  if (nt > 0 && warp == kTmaWarp) {
    // ---------------- TMA
    if (lane == 0) {
      const uint64_t pol = policy_evict_first();
      mbar_arrive_expect_tx(&ctl.q_full, (uint32_t)(G::kBoxes * 128 * p.g * (prefix ? p.bt : 1)));
      for (int bx = 0; bx < G::kBoxes; ++bx) tma_load_4d(sQ + bx * 16384, mq, bx * 64, 0, b0, h, &ctl.q_full, pol);
      int armed = 0;
      auto load = [&](const CUtensorMap* map, int t) -> bool {
        const int s = armed % kSlots, r = armed / kSlots;
        if (r > 0 && !mbar_wait(&empty[s], (r - 1) & 1, TC_DEVERR_PIPE_TIMEOUT, kShSpin)) return false;
        mbar_arrive_expect_tx(&full[s], (uint32_t)G::kSlotBytes);
        uint8_t* st = sKV + s * G::kSlotBytes;
        if (paged) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int3 e = sub(t, c);
            for (int bx = 0; bx < G::kBoxes; ++bx)
              tma_load_4d(st + bx * G::kBoxBytes + c * 4096, map, bx * 64, e.y, h, e.x, &full[s], pol);
          }
        } else {
          for (int bx = 0; bx < G::kBoxes; ++bx)
            tma_load_4d(st + bx * G::kBoxBytes, map, bx * 64, t * kShKeys, h, prefix ? 0 : b0, &full[s], pol);
        }
        ++armed;
        return true;
      };
      bool ok = load(mk, t0) && (nt < 2 || load(mk, t0 + 1));
      for (int j = 0; ok && j < nt; ++j) ok = load(mv, t0 + j) && (j + 2 >= nt || load(mk, t0 + j + 2));
      // copies still in flight after a wait gave up must land before the CTA leaves (normally these phases
      // completed long ago and the waits return at once)
      for (int i = armed - kSlots > 0 ? armed - kSlots : 0; i < armed; ++i)
        mbar_wait(&full[i % kSlots], (i / kSlots) & 1, TC_DEVERR_PIPE_TIMEOUT, kShSpin);
      mbar_wait(&ctl.q_full, 0, TC_DEVERR_PIPE_TIMEOUT, kShSpin);
    }
  } else if (nt > 0 && warp == kMmaWarp) {
    // ---------------- tcgen05.mma: S(0) S(1), then per tile P V(j), S(j + 2). Products of one thread run in issue
    // order, so S(j + 2) overwrites P(j) only after P V(j) read it. K and V are waited for before P, while the
    // softmax works: each wait costs this thread some 200 cycles even when the phase is long over.
    if (elect_one()) {
      const uint32_t idS = umma_idesc_f16(kBf16, false, 128, kShKeys);
      const uint32_t idO = umma_idesc_f16(kBf16, true, 128, D);
      // descriptors of the first K step; a byte offset of 16n adds n (the address field does not overflow)
      const uint64_t dq = umma_desc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t dk = umma_desc_sw128(smem_u32(sKV), 16, 1024);
      const uint64_t dv = umma_desc_sw128(smem_u32(sKV), G::kBoxBytes, 1024);
      auto wait = [&](uint64_t* bar, int phase) { return mbar_wait(bar, phase & 1, TC_DEVERR_PIPE_TIMEOUT, kShSpin); };
      auto wait_slot = [&](int i) { return wait(&full[i % kSlots], i / kSlots); };
      auto issue_s = [&](int j) {
        const int s = k_at(j) % kSlots;
        const uint64_t k = dk + s * (G::kSlotBytes >> 4);
#pragma unroll
        for (int kd = 0; kd < D / 16; ++kd)
          umma_f16(tmem + 64 * (j & 1), dq + (((kd >> 2) * 16384 + (kd & 3) * 32) >> 4),
                   k + (((kd >> 2) * G::kBoxBytes + (kd & 3) * 32) >> 4), idS, kd > 0);
        umma_commit(&empty[s]);
        umma_commit(&s_full[j & 1]);
      };
      bool ok = wait(&ctl.q_full, 0);
      for (int j = 0; ok && j < 2 && j < nt; ++j) {
        ok = wait_slot(k_at(j));
        if (ok) issue_s(j);
      }
      for (int j = 0; ok && j < nt; ++j) {
        const int s = v_at(j) % kSlots;
        ok = wait_slot(v_at(j)) && (j + 2 >= nt || wait_slot(k_at(j + 2))) && wait(&p_full[j & 1], j >> 1);
        if (!ok) break;
        tmem_fence_after();
        const uint64_t v = dv + s * (G::kSlotBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kShKeys / 16; ++kk)
          umma_f16_tmem_a(tO, tmem + 64 * (j & 1) + kk * 8, v + ((kk * 2048) >> 4), idO, j > 0 || kk > 0);
        umma_commit(&empty[s]);
        umma_commit(&pv_done[j & 1]);
        if (j + 2 < nt) issue_s(j + 2);
      }
      umma_commit(&ctl.fin);  // completes once every product issued above has
    }
  } else if (nt > 0 && warp < nlive) {
    // ---------------- softmax: thread = TMEM lane = query row (sequence b0 + row / g, head row % g)
    const int row = threadIdx.x;
    const uint32_t lb = (uint32_t)(warp * 32) << 16;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      const uint32_t tS = tmem + lb + 64 * (j & 1);
      // valid keys of the tile's halves of 32
      int v0, v1;
      if (paged) {
        v0 = sub(t0 + j, 0).z;
        v1 = sub(t0 + j, 1).z;
      } else {
        const int left = end - (t0 + j) * kShKeys;
        v0 = left < 32 ? left : 32;
        v1 = left < 64 ? (left > 32 ? left - 32 : 0) : 32;
      }
      // warp-uniform: tcgen05.ld/st and the votes below are warp-collective
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[j & 1], (j >> 1) & 1, TC_DEVERR_PIPE_TIMEOUT, kShSpin));
      if (!ok) break;
      tmem_fence_after();
      uint32_t v[2][32];
      tmem_ld32(tS, v[0]);
      tmem_ld32(tS + 32, v[1]);
      tmem_wait_ld();
      if (v0 + v1 < kShKeys) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          if (e >= v0) v[0][e] = __float_as_uint(-INFINITY);
          if (e >= v1) v[1][e] = __float_as_uint(-INFINITY);
        }
        // the staged V rows behind the end: zeros, so that a zero weight never meets a NaN
        const int i = v_at(j);
        ok = __all_sync(0xffffffffu, mbar_wait(&full[i % kSlots], (i / kSlots) & 1, TC_DEVERR_PIPE_TIMEOUT, kShSpin));
        if (!ok) break;
        uint8_t* st = sKV + (i % kSlots) * G::kSlotBytes;
        for (int y = row; y < kShKeys * (D / 8); y += nlive * 32) {
          const int r = y / (D / 8), cc = y % (D / 8);
          if ((r & 31) >= (r < 32 ? v0 : v1))
            *reinterpret_cast<uint4*>(st + (cc >> 3) * G::kBoxBytes + r * 128 + (cc & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      float mx[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) mx[r] = -INFINITY;
#pragma unroll
      for (int cch = 0; cch < 2; ++cch)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          mx[e & 7] = fmax3(mx[e & 7], __uint_as_float(v[cch][2 * e]), __uint_as_float(v[cch][2 * e + 1]));
      const float mt = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                             fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * p.c;  // exp2 domain (c > 0)
      const bool bump = mt > m + kShLazyMax;
      const float mn = bump ? mt : m;
      const float alpha = !bump ? 1.f : (m == -INFINITY ? 0.f : fast_exp2(m - mn));
      const float mref = mn == -INFINITY ? 0.f : mn;
      float2 rs[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t w[32];  // 16-bit pairs: keys 2e, 2e + 1
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float2 xy = ffma2(make_float2(__uint_as_float(v[e >> 4][2 * (e & 15)]), __uint_as_float(v[e >> 4][2 * (e & 15) + 1])),
                                make_float2(p.c, p.c), make_float2(-mref, -mref));
        const float2 pp = make_float2(fast_exp2(xy.x), fast_exp2(xy.y));
        rs[e & 1] = fadd2(rs[e & 1], pp);
        w[e] = Mma<T>::pack(pp.x, pp.y);
      }
      tmem_st32(tS, w);
      l = l * alpha + ((rs[0].x + rs[1].x) + (rs[0].y + rs[1].y));
      m = mn;
      if (j >= 1 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // O holds P V of the tiles before j once P V(j - 1) is done (P V(j) waits for this warp)
        ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, TC_DEVERR_PIPE_TIMEOUT, kShSpin));
        if (!ok) break;
        tmem_fence_after();
#pragma unroll
        for (int cch = 0; cch < D / 32; ++cch) {
          uint32_t o[32];
          tmem_ld32(tO + lb + cch * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(tO + lb + cch * 32, o);
        }
      }
      tmem_wait_st();
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[j & 1]);
    }
    if (ok)
      ok = __all_sync(0xffffffffu, mbar_wait(&ctl.fin, 0, TC_DEVERR_PIPE_TIMEOUT, kShSpin));
    if (ok) {
      tmem_fence_after();
      const int64_t rows = (int64_t)p.batch * p.hkv * p.g;
      const int bi = row / p.g;
      const int64_t r = ((int64_t)(b0 + bi) * p.hkv + h) * p.g + (row - bi * p.g);
      float* orow = p.o + ((int64_t)part * rows + r) * D;
#pragma unroll
      for (int cch = 0; cch < D / 32; ++cch) {
        uint32_t o[32];
        tmem_ld32(tO + lb + cch * 32, o);
        tmem_wait_ld();
        if (row < live) {
#pragma unroll
          for (int q8 = 0; q8 < 4; ++q8) st_v8(orow + cch * 32 + q8 * 8, o + 8 * q8);
        }
      }
      if (row < live) p.ml[(int64_t)part * rows + r] = make_float2(m, l);
    }
  }
  // every product has completed before the TMEM columns are freed (bounded: a lost commit only errs)
  tmem_fence_before();
  __syncthreads();
  if (warp == 0) {
    if (nt > 0) mbar_wait(&ctl.fin, 0, TC_DEVERR_PIPE_TIMEOUT, kShSpin);
    tmem_fence_after();
    tmem_dealloc(tmem, G::kTmemCols);
  }
}

struct SharedMergeParams {
  const float* o;
  const float2* ml;
  const int32_t* lengths;
  void* out;
  int64_t so_b, so_h, so_g;
  int batch, hkv, g, m, np, ns;
  int wpr;  // warps per query row
};

// p.wpr warps per query row (a power of two <= 8, eight warps a CTA): warp w of a row folds parts w, w + wpr, ...,
// lane l the float4 columns l, l + 32, ...; the warps' states are joined in shared memory in their order.
template <typename T, int D>
__global__ void __launch_bounds__(256) shared_merge_kernel(const __grid_constant__ SharedMergeParams p) {
  constexpr int kCols = D / 4, kPer = (kCols + 31) / 32;  // float4 columns, per lane
  constexpr int kLoads = 4;
  __shared__ float s_m[8], s_l[8];
  __shared__ float4 s_a[8][kCols];
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.batch * p.hkv * p.g;
  const int64_t r = blockIdx.x * (int64_t)(8 / p.wpr) + warp / p.wpr;
  const bool row = r < rows;
  const int i = (int)(r % p.g), h = (int)(r / p.g % p.hkv), b = row ? (int)(r / p.g / p.hkv) : 0;
  int len = p.lengths != nullptr ? p.lengths[b] : p.m;
  len = len < 0 ? 0 : (len > p.m ? p.m : len);
  const int tiles = (len + kShKeys - 1) / kShKeys;
  const int parts = row ? p.np + p.ns : 0;
  float M = -INFINITY, L = 0.f;
  float4 A[kPer];
#pragma unroll
  for (int x = 0; x < kPer; ++x) A[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = warp & (p.wpr - 1); p0 < parts; p0 += kLoads * p.wpr) {
    float2 ml[kLoads];
    float4 o[kLoads][kPer];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int s = p0 + k * p.wpr;
      bool use = s < parts;
      if (use && s >= p.np) {
        int t0, t1;
        shared_range(tiles, s - p.np, p.ns, t0, t1);
        use = t1 > t0;
      }
      ml[k] = use ? __ldcg(p.ml + s * rows + r) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int col = lane + 32 * x;
        o[k][x] = use && col < kCols ? __ldcg(reinterpret_cast<const float4*>(p.o + (s * rows + r) * D) + col)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float mc = M;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) mc = fmaxf(mc, ml[k].x);
    const float a = M == -INFINITY ? 0.f : fast_exp2(M - mc);
    L *= a;
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      A[x].x *= a;
      A[x].y *= a;
      A[x].z *= a;
      A[x].w *= a;
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const float w = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - mc);
      L += w * ml[k].y;
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        A[x].x += w * o[k][x].x;
        A[x].y += w * o[k][x].y;
        A[x].z += w * o[k][x].z;
        A[x].w += w * o[k][x].w;
      }
    }
    M = mc;
  }
  if (p.wpr > 1) {
    if (lane == 0) {
      s_m[warp] = M;
      s_l[warp] = L;
    }
#pragma unroll
    for (int x = 0; x < kPer; ++x)
      if (lane + 32 * x < kCols) s_a[warp][lane + 32 * x] = A[x];
    __syncthreads();
    if ((warp & (p.wpr - 1)) != 0) return;
    float Mt = M;
    for (int w = 1; w < p.wpr; ++w) Mt = fmaxf(Mt, s_m[warp + w]);
    L = 0.f;
#pragma unroll
    for (int x = 0; x < kPer; ++x) A[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < p.wpr; ++w) {
      const float f = s_m[warp + w] == -INFINITY ? 0.f : fast_exp2(s_m[warp + w] - Mt);
      L += f * s_l[warp + w];
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        if (lane + 32 * x < kCols) {
          const float4 v = s_a[warp + w][lane + 32 * x];
          A[x].x += f * v.x;
          A[x].y += f * v.y;
          A[x].z += f * v.z;
          A[x].w += f * v.w;
        }
      }
    }
  }
  if (!row) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* out = static_cast<T*>(p.out) + b * p.so_b + h * p.so_h + i * p.so_g;
#pragma unroll
  for (int x = 0; x < kPer; ++x) {
    const int col = lane + 32 * x;
    if (col < kCols) {
      uint2 w;
      w.x = Mma<T>::pack(A[x].x * inv, A[x].y * inv);
      w.y = Mma<T>::pack(A[x].z * inv, A[x].w * inv);
      *reinterpret_cast<uint2*>(out + 4 * col) = w;
    }
  }
}

}  // namespace tc
