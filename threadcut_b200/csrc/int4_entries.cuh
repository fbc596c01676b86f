// C entry points of the 4-bit cache and the 4-bit projections (kernels: int4.cuh, int4_attn.cuh, int4_gemv.cuh).
// Included at the end of threadcut_b200.cu, whose host helpers it uses.
#pragma once

namespace {

bool i4_dtype(int dtype) { return dtype == TC_BF16 || dtype == TC_F16; }

// Rows of 4-bit caches are copied and stored in whole 16-byte (d = 64: 8-byte) units.
bool i4_aligned(const void* base, int64_t s0, int64_t s1, int64_t s2, int d) {
  const int64_t unit = d == 64 ? 8 : 16;
  return reinterpret_cast<uintptr_t>(base) % unit == 0 && s0 % unit == 0 && s1 % unit == 0 && s2 % unit == 0;
}

bool i4_pool(int hkv, int d, int64_t page_rows, int64_t num_pages) {
  return hkv >= 1 && hkv <= 65535 && mma_dim(d) && page_rows >= 1 && page_rows <= (1 << 30) && num_pages >= 1 &&
         num_pages <= (1 << 30);
}

// fn<T, D>(args...) for the type and head size
#define TC_INT4_DISPATCH(fn, dtype, d, ...)                                                                     \
  ((dtype) == TC_BF16 ? ((d) == 64    ? fn<__nv_bfloat16, 64>(__VA_ARGS__)                                      \
                         : (d) == 128 ? fn<__nv_bfloat16, 128>(__VA_ARGS__)                                     \
                                      : fn<__nv_bfloat16, 256>(__VA_ARGS__))                                    \
                      : ((d) == 64    ? fn<__half, 64>(__VA_ARGS__)                                             \
                         : (d) == 128 ? fn<__half, 128>(__VA_ARGS__)                                            \
                                      : fn<__half, 256>(__VA_ARGS__)))

template <typename T, int D, int U>
cudaError_t launch_int4_append_vec(const Int4AppendParams& p, int sms, cudaStream_t st) {
  const int64_t groups = cdiv(p.hq, 256 / D * U) + 2 * cdiv(p.hkv, 256 / D * i4_kv_heads(U));
  // warps of a token's groups, the tokens shared out evenly over those that are resident at once
  const bool norm = p.q_w != nullptr || p.k_w != nullptr;
  const int64_t resident = (int64_t)sms * 8 * i4_append_ctas(U, norm) / groups;
  const int64_t rounds = cdiv(p.t, resident < 1 ? 1 : resident);
  const dim3 grid((unsigned)cdiv(cdiv(p.t, rounds) * groups, 8));
  auto fn = norm ? int4_append_vec_kernel<T, D, U, true> : int4_append_vec_kernel<T, D, U, false>;
  return launch_ex(fn, grid, dim3(256), 0, st, p);
}

// Four heads a lane, and for keys and values alone the kernel that loads a token ahead, from 64 warps an SM on (a warp for 256/D heads of a
// token). With many heads they pay earlier, with few later: 32 + 8 heads of 128, one and four heads a lane, 128 tokens (21 warps an
// SM) 2.7 and 2.7 us, 256 (42) 3.8 and 2.9, 512 (83) 5.8 and 4.4; 8 + 1 heads 1,024 tokens (42) 5.7 and 5.7, 1,536 (62) 7.8 and 10.1.
// Keys and values of 8 heads, one head a lane, four, and a token ahead: 1,024 tokens (55) 4.1, 3.5 and 3.1 us, 2,048 (111) 5.7, 4.7 and
// 4.8, 8,192 17.7, 12.6 and 10.1.
template <typename T, int D>
cudaError_t launch_int4_append(const Int4AppendParams& p, bool vec, int sms, cudaStream_t st) {
  constexpr int RW = 256 / D;
  const int64_t warps = p.t * (cdiv(p.hq, RW) + 2 * cdiv(p.hkv, RW));
  if (vec && p.hq == 0 && p.rot == 0 && p.k_w == nullptr && warps >= (int64_t)sms * 64) {
    const int64_t groups = 2 * cdiv(p.hkv, RW * kI4WriteHeads), resident = (int64_t)sms * 24 / groups;
    const int64_t rounds = cdiv(p.t, resident < 1 ? 1 : resident);
    return launch_ex(int4_write_kernel<T, D>, dim3((unsigned)cdiv(cdiv(p.t, rounds) * groups, 8)), dim3(256), 0, st, p);
  }
  if (vec)
    return warps < (int64_t)sms * 64 ? launch_int4_append_vec<T, D, 1>(p, sms, st)
                                     : launch_int4_append_vec<T, D, 4>(p, sms, st);
  const int64_t blocks = cdiv(warps, 8);
  return launch_ex(int4_append_kernel<T, D>,
                   dim3((unsigned)(blocks < (int64_t)sms * 64 ? blocks : (int64_t)sms * 64)), dim3(256), 0, st, p);
}

template <typename T, int D>
cudaError_t launch_int4_gather(const Int4GatherParams& p, int sms, cudaStream_t st) {
  const int64_t blocks = cdiv(p.n_tiles * p.hkv, 8);
  return launch_ex(int4_gather_kernel<T, D>, dim3((unsigned)(blocks < (int64_t)sms * 64 ? blocks : (int64_t)sms * 64)),
                   dim3(256), 0, st, p);
}

template <typename T, int D>
cudaError_t launch_int4_rotate(const Int4RotateParams& p, int sms, cudaStream_t st) {
  const int64_t blocks = cdiv(p.layers * p.n_tiles * p.hkv, 8);
  return launch_ex(int4_rotate_kernel<T, D>, dim3((unsigned)(blocks < (int64_t)sms * 8 ? blocks : (int64_t)sms * 8)),
                   dim3(256), 0, st, p);
}

int i4_head_tiles(int g) { return g <= 4 ? 1 : g <= 8 ? 2 : 4; }
// Warps of a CTA. The slices of one long sequence end together, so that one large CTA an SM has the least to merge; short
// ones leave a large CTA's warps with too little each, and those of several sequences end at different times, so that a second
// CTA on the SM works while one begins or ends. One sequence, 8 KV heads of 128, 16 against 8 warps: 4,096 rows 10.4 and
// 8.8 us, 8,192 rows 12.4 and 12.4, 16,384 rows 14.4 and 16.3, 98,304 rows 34.3 and 35.2.
int i4_cta_warps(int batch, int hkv, int64_t rows, int d, int nh, int sms) {
  return batch == 1 && hkv * cdiv(rows, kTile) >= 14 * (int64_t)sms ? i4_warps(d, nh) : 8;
}

template <typename T, int D, int NH, bool kBulk, int kWarps>
cudaError_t launch_int4_decode_w(const Int4DecodeParams& p, dim3 grid, int dev, cudaStream_t st) {
  auto fn = int4_decode_kernel<T, D, NH, kBulk, kWarps>;
  constexpr int smem = I4Geom<D, kBulk, kWarps>::kSmem;
  const cudaError_t e = set_smem(reinterpret_cast<const void*>(fn), smem + 1024, dev);  // beside static shared memory
  if (e != cudaSuccess) return e;
  return launch_ex(fn, grid, dim3(32 * kWarps), smem, st, p);
}
template <typename T, int D, int NH, bool kBulk>
cudaError_t launch_int4_decode_nh(const Int4DecodeParams& p, int warps, dim3 grid, int dev, cudaStream_t st) {
  if constexpr (i4_warps(D, NH) == 16) {
    if (warps == 16) return launch_int4_decode_w<T, D, NH, kBulk, 16>(p, grid, dev, st);
  }
  return launch_int4_decode_w<T, D, NH, kBulk, 8>(p, grid, dev, st);
}
template <typename T, int D, bool kBulk>
cudaError_t launch_int4_decode_bulk(const Int4DecodeParams& p, int warps, dim3 grid, int dev, cudaStream_t st) {
  switch (i4_head_tiles(p.g)) {
    case 1: return launch_int4_decode_nh<T, D, 1, kBulk>(p, warps, grid, dev, st);
    case 2: return launch_int4_decode_nh<T, D, 2, kBulk>(p, warps, grid, dev, st);
  }
  return launch_int4_decode_nh<T, D, 4, kBulk>(p, warps, grid, dev, st);
}
template <typename T, int D>
cudaError_t launch_int4_decode(const Int4DecodeParams& p, int warps, dim3 grid, int dev, cudaStream_t st) {
  if constexpr (D > 64) {  // (rows of d = 64 are 40 bytes, and begin off 16-byte boundaries)
    if (p.sk_n == i4_row_bytes(D) && p.sv_n == i4_row_bytes(D))
      return launch_int4_decode_bulk<T, D, true>(p, warps, grid, dev, st);
  }
  return launch_int4_decode_bulk<T, D, false>(p, warps, grid, dev, st);
}

// KV partition. One sequence: as many slices as are resident at once, none below a tile a warp. Several, whose lengths are
// on the device: slices for about two rounds of CTAs, of 2 to 16 tiles a warp, that the block scheduler balances (64
// sequences of 8,704 rows, 8 KV heads of 128: slices of 32 tiles 191 us, 64 172, 136 154, 272 162; 8 of 2,000 rows:
// slices of 8 tiles 17.1 us, 16 and 32 14.4, 64 16.5).
DecodePlan plan_int4(int batch, int hkv, int g, int d, int64_t rows, int splits_req, int sms) {
  const int nh = i4_head_tiles(g), warps = i4_cta_warps(batch, hkv, rows, d, nh, sms);
  const int per_sm = i4_warps(d, nh) / warps;
  const int64_t tiles = rows > 0 ? cdiv(rows, kTile) : 1;
  if (splits_req > 0) return plan_decode(batch, hkv, rows, 0, false, splits_req, per_sm, sms);
  DecodePlan pl;
  if (batch == 1) {
    pl = plan_decode(1, hkv, rows, 0, false, 0, per_sm, sms);
    if (pl.tps < warps) pl.tps = warps;
  } else {
    const int64_t share = (int64_t)batch * hkv * tiles / (2 * (int64_t)sms * per_sm);
    pl.tps = share < 2 * warps ? 2 * warps : share > 16 * warps ? 16 * warps : share;
    if (pl.tps < cdiv(tiles, kMaxSplits)) pl.tps = cdiv(tiles, kMaxSplits);
  }
  pl.max_splits = cdiv(tiles, pl.tps);
  return pl;
}

int run_int4_decode(Int4DecodeParams& p, int d, int64_t rows, float scale, int splits, int dtype, void* ws,
                    size_t ws_bytes, cudaStream_t st) {
  const int dev = current_device();
  const DecodePlan pl = plan_int4(p.batch, p.hkv, p.g, d, rows, splits, sm_count(dev));
  const WsLayout w = decode_ws_layout(p.batch, p.hkv, p.g, d, pl.max_splits);
  if (pl.max_splits > 1) {
    if (ws == nullptr || ws_bytes < w.total) return TC_ERR_WORKSPACE;
    if (!aligned16(ws)) return TC_ERR_ALIGN;
    uint8_t* wb = static_cast<uint8_t*>(ws);
    p.counters = reinterpret_cast<unsigned int*>(wb + w.counters);
    p.ws_ml = reinterpret_cast<float2*>(wb + w.ml);
    p.ws_o = reinterpret_cast<float*>(wb + w.o);
  }
  p.tiles_per_split = (int)pl.tps;
  p.max_splits = (int)pl.max_splits;
  p.c = scale * kLog2e;
  p.q_vec = aligned16(p.q) && stride16(p.sq_b, dtype) && stride16(p.sq_h, dtype) && stride16(p.sq_g, dtype);
  const dim3 grid((unsigned)pl.max_splits, (unsigned)p.hkv, (unsigned)p.batch);
  const cudaError_t e = TC_INT4_DISPATCH(
      launch_int4_decode, dtype, d, p, i4_cta_warps(p.batch, p.hkv, rows, d, i4_head_tiles(p.g), sm_count(dev)), grid, dev, st);
  return e == cudaSuccess ? TC_OK : TC_ERR_CUDA;
}

constexpr int kGvMaxSmem = 226 * 1024;
constexpr int kGvMaxColumns = 65536;  // one token of them fits
// Up to these, tokens as digits, which two fill the columns of a product with: 151,936 x 2,560 with one token 35.8 us, as 16-bit
// numbers 46.6; two 37.4 and 47.8; 2,560 x 4,096 with one 3.7 and 4.2.
constexpr int kGvIntTokens = 2;

// Row tiles a CTA works on at a time, 16 warps between them: as many as leave each stream 8 to go through, so that few sums
// are added across warps and the streams end together; two at least where there are enough row tiles. 1, 2, 4 and 8 streams:
// 2,560 x 4,096 (one token) 3.7, 3.9, 5.2 and 8.0 us, 6,144 x 2,560 4.3, 3.9, 4.3 and 5.7, 19,456 x 2,560 8.7, 7.5, 7.9 and 9.3,
// 151,936 x 2,560 with 7 tokens 82, 58, 54 and 53.
int gv_streams(int64_t n, int sms) {
  const int64_t tiles = cdiv(n, 16);
  int streams = tiles > 2 * (int64_t)sms ? 2 : 1;
  while (streams < 8 && tiles >= 16 * (int64_t)streams * sms) streams *= 2;
  return streams;
}
int gv_part_bytes(int m, int streams) {
  const int least = kGvWarps * 64 * m;  // a row tile of each stream
  return least > kGvPartBytes ? least : kGvPartBytes;
}
// Shared memory of a launch over m tokens beside the rings.
int64_t gv_fixed(int k, int m, int group, int streams, bool digits) {
  return 2 * gv_part_bytes(m, streams) + gv_sum_bytes(k, m, group, digits) +
         (int64_t)m * (digits ? kGvDigits : 1) * gv_x_bytes(k, digits);
}
// The largest ring that fits beside that; false where none does. A stage holds a warp's run of columns, or an even part of it.
bool gv_ring(int64_t fixed, int k, int group, int streams, int& chunk, int& stages) {
  const int64_t run = cdiv((int64_t)gv_blocks(k) * streams, kGvWarps);
  for (int most = kGvMaxChunk; most >= 1; --most)
    for (stages = kGvMaxStages; stages >= 2; --stages) {
      chunk = (int)cdiv(run, cdiv(run, most));
      if (fixed + (int64_t)kGvWarps * chunk * stages * gv_tile_bytes(group) <= kGvMaxSmem) return true;
    }
  return false;
}

template <typename T, int NT, int G, bool kInt>
cudaError_t launch_int4_gemv_g(Int4GemvParams p, int smem, int dev, cudaStream_t st) {
  auto fn = int4_gemv_kernel<T, NT, G, kInt>;
  // the opt-in is set once per (kernel, device): ask for the most any plan takes
  const cudaError_t e = set_smem(reinterpret_cast<const void*>(fn), kGvMaxSmem, dev);
  if (e != cudaSuccess) return e;
  const int tiles = (int)cdiv(p.n, 16), sms = sm_count(dev);
  int ctas = (int)cdiv(tiles, p.streams);
  if (ctas > sms) ctas = sms;
  p.share = tiles / ctas;
  p.more = tiles - p.share * ctas;
  return launch_ex(fn, dim3((unsigned)ctas), dim3(32 * kGvWarps), smem, st, p);
}
template <typename T, int NT, bool kInt>
cudaError_t launch_int4_gemv_nt(const Int4GemvParams& p, int group, int smem, int dev, cudaStream_t st) {
  return group == 32   ? launch_int4_gemv_g<T, NT, 32, kInt>(p, smem, dev, st)
         : group == 64 ? launch_int4_gemv_g<T, NT, 64, kInt>(p, smem, dev, st)
                       : launch_int4_gemv_g<T, NT, 128, kInt>(p, smem, dev, st);
}
template <typename T>
cudaError_t launch_int4_gemv(const Int4GemvParams& p, int group, bool digits, int smem, int dev, cudaStream_t st) {
  return digits              ? launch_int4_gemv_nt<T, 1, true>(p, group, smem, dev, st)
         : p.m <= 8          ? launch_int4_gemv_nt<T, 1, false>(p, group, smem, dev, st)
         : p.m <= 16         ? launch_int4_gemv_nt<T, 2, false>(p, group, smem, dev, st)
                             : launch_int4_gemv_nt<T, 4, false>(p, group, smem, dev, st);
}

}  // namespace

extern "C" {

int tc_int4_append_rope(const void* q, const void* k, const void* v, void* q_out, void* k_pool, void* v_pool, int hq,
                        int hkv, int d, int64_t t, int64_t q_stride_h, int64_t q_stride_t, int64_t k_stride_h,
                        int64_t k_stride_t, int64_t v_stride_h, int64_t v_stride_t, int64_t q_out_stride_h,
                        int64_t q_out_stride_t, const void* q_norm_weight, const void* k_norm_weight, float eps,
                        const void* cos_t, const void* sin_t, int rot, int64_t cos_stride_t, int64_t sin_stride_t,
                        int table_dtype, int64_t page_rows, int64_t num_pages, int64_t pool_stride_page,
                        int64_t pool_stride_h, int64_t pool_stride_row, const int32_t* slots, int dtype, void* stream) {
  if (!i4_dtype(dtype) || (table_dtype != dtype && table_dtype != TC_F32)) return TC_ERR_DTYPE;
  if (!i4_pool(hkv, d, page_rows, num_pages) || hq < 0 || hq > 65535 || rot < 0 || rot > d || (rot & 1) || t < 0 ||
      t > INT32_MAX || !(eps >= 0.f))
    return TC_ERR_INVALID;
  if (t == 0) return TC_OK;
  if (k == nullptr || v == nullptr || k_pool == nullptr || v_pool == nullptr || slots == nullptr ||
      (rot > 0 && (cos_t == nullptr || sin_t == nullptr)) || (hq > 0 && (q == nullptr || q_out == nullptr)))
    return TC_ERR_INVALID;
  if (!i4_aligned(k_pool, pool_stride_page, pool_stride_h, pool_stride_row, d) ||
      !i4_aligned(v_pool, 0, 0, 0, d))
    return TC_ERR_ALIGN;
  Int4AppendParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.kp = static_cast<uint8_t*>(k_pool);
  p.vp = static_cast<uint8_t*>(v_pool);
  p.q_w = q_norm_weight;
  p.k_w = k_norm_weight;
  p.cos_t = cos_t;
  p.sin_t = sin_t;
  p.hq = hq;
  p.hkv = hkv;
  p.rot = rot;
  p.t = t;
  p.q_sh = q_stride_h;
  p.q_st = q_stride_t;
  p.k_sh = k_stride_h;
  p.k_st = k_stride_t;
  p.v_sh = v_stride_h;
  p.v_st = v_stride_t;
  p.qo_sh = q_out_stride_h;
  p.qo_st = q_out_stride_t;
  p.cos_st = cos_stride_t;
  p.sin_st = sin_stride_t;
  p.page_rows = page_rows;
  p.num_pages = num_pages;
  p.s_page = pool_stride_page;
  p.s_h = pool_stride_h;
  p.s_row = pool_stride_row;
  p.slots = slots;
  p.eps = eps;
  p.inv_d = 1.f / (float)d;
  p.minus_zero = -0.f;
  p.table_f32 = table_dtype == TC_F32;
  bool vec = rot % 16 == 0 && aligned16(k) && aligned16(v) && stride16(k_stride_h, dtype) && stride16(k_stride_t, dtype) &&
             stride16(v_stride_h, dtype) && stride16(v_stride_t, dtype);
  if (hq > 0)
    vec = vec && aligned16(q) && aligned16(q_out) && stride16(q_stride_h, dtype) && stride16(q_stride_t, dtype) &&
          stride16(q_out_stride_h, dtype) && stride16(q_out_stride_t, dtype);
  if (rot > 0)
    vec = vec && aligned16(cos_t) && aligned16(sin_t) && stride16(cos_stride_t, table_dtype) &&
          stride16(sin_stride_t, table_dtype);
  vec = vec && aligned16(q_norm_weight) && aligned16(k_norm_weight) && (reinterpret_cast<uintptr_t>(slots) & 7u) == 0;
  const cudaError_t e = TC_INT4_DISPATCH(launch_int4_append, dtype, d, p, vec, sm_count(current_device()),
                                         static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TC_OK : TC_ERR_CUDA;
}

int tc_int4_gather(const void* k_pool, const void* v_pool, void* k_out, void* v_out, int hkv, int d, int64_t n,
                   int64_t out_stride_h, int64_t out_stride_n, int64_t page_rows, int64_t num_pages,
                   int64_t pool_stride_page, int64_t pool_stride_h, int64_t pool_stride_row, const int32_t* tiles,
                   int64_t n_tiles, int dtype, void* stream) {
  if (!i4_dtype(dtype)) return TC_ERR_DTYPE;
  if (!i4_pool(hkv, d, page_rows, num_pages) || n < 0 || n_tiles < 0 || n_tiles > INT32_MAX) return TC_ERR_INVALID;
  if (n == 0 || n_tiles == 0) return TC_OK;
  if (k_pool == nullptr || v_pool == nullptr || k_out == nullptr || v_out == nullptr || tiles == nullptr)
    return TC_ERR_INVALID;
  if (!i4_aligned(k_pool, pool_stride_page, pool_stride_h, pool_stride_row, d) ||
      !i4_aligned(v_pool, 0, 0, 0, d) ||
      !aligned16(k_out) || !aligned16(v_out) || !stride16(out_stride_h, dtype) || !stride16(out_stride_n, dtype) ||
      !aligned16(tiles))
    return TC_ERR_ALIGN;
  Int4GatherParams p;
  std::memset(&p, 0, sizeof(p));
  p.kp = static_cast<const uint8_t*>(k_pool);
  p.vp = static_cast<const uint8_t*>(v_pool);
  p.k_out = k_out;
  p.v_out = v_out;
  p.hkv = hkv;
  p.n = n;
  p.out_sh = out_stride_h;
  p.out_sn = out_stride_n;
  p.page_rows = page_rows;
  p.num_pages = num_pages;
  p.s_page = pool_stride_page;
  p.s_h = pool_stride_h;
  p.s_row = pool_stride_row;
  p.tiles = tiles;
  p.n_tiles = n_tiles;
  const cudaError_t e =
      TC_INT4_DISPATCH(launch_int4_gather, dtype, d, p, sm_count(current_device()), static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TC_OK : TC_ERR_CUDA;
}

int tc_int4_rotate_keys(void* const* k_pools, int layers, int hkv, int d, int64_t page_rows, int64_t num_pages,
                        int64_t pool_stride_page, int64_t pool_stride_h, int64_t pool_stride_row, const int32_t* tiles,
                        int tile_cols, int64_t n_tiles, const float* cos_sin, int dtype, void* stream) {
  if (!i4_dtype(dtype)) return TC_ERR_DTYPE;
  if (layers < 1 || layers > kMaxLayers || !i4_pool(hkv, d, page_rows, num_pages) || n_tiles < 0 || n_tiles > INT32_MAX ||
      tile_cols < 3 || tile_cols > 65535 || k_pools == nullptr || cos_sin == nullptr)
    return TC_ERR_INVALID;
  if (n_tiles == 0) return TC_OK;
  if (tiles == nullptr) return TC_ERR_INVALID;
  Int4RotateParams p;
  std::memset(&p, 0, sizeof(p));
  for (int l = 0; l < layers; ++l) {
    if (k_pools[l] == nullptr) return TC_ERR_INVALID;
    if (!i4_aligned(k_pools[l], pool_stride_page, pool_stride_h, pool_stride_row, d)) return TC_ERR_ALIGN;
    p.kp[l] = static_cast<uint8_t*>(k_pools[l]);
  }
  p.layers = layers;
  p.hkv = hkv;
  p.page_rows = page_rows;
  p.num_pages = num_pages;
  p.s_page = pool_stride_page;
  p.s_h = pool_stride_h;
  p.s_row = pool_stride_row;
  p.tiles = tiles;
  p.tile_cols = tile_cols;
  p.n_tiles = n_tiles;
  load_cos_sin(p.cs, cos_sin, d);
  p.minus_zero = -0.f;
  const cudaError_t e =
      TC_INT4_DISPATCH(launch_int4_rotate, dtype, d, p, sm_count(current_device()), static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TC_OK : TC_ERR_CUDA;
}

size_t tc_decode_attention_int4_workspace_size(int batch, int hkv, int g, int d, int64_t rows, int splits) {
  if (batch < 1 || batch > 65535 || hkv < 1 || hkv > 65535 || g < 1 || g > 16 || !mma_dim(d) || rows < 0 || splits < 0)
    return 0;
  const DecodePlan pl = plan_int4(batch, hkv, g, d, rows, splits, sm_count(current_device()));
  return pl.max_splits > 1 ? decode_ws_layout(batch, hkv, g, d, pl.max_splits).total : 0;
}

int tc_decode_attention_int4(const void* q, const void* k, const void* v, void* out, int batch, int hkv, int g, int d,
                             int64_t n, const int32_t* lengths, int64_t q_stride_b, int64_t q_stride_h,
                             int64_t q_stride_g, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_n,
                             int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_n, int64_t out_stride_b,
                             int64_t out_stride_h, int64_t out_stride_g, float scale, int splits, int dtype,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (!i4_dtype(dtype)) return TC_ERR_DTYPE;
  if (batch < 1 || batch > 65535 || hkv < 1 || hkv > 65535 || g < 1 || g > 16 || !mma_dim(d) || n < 0 || n > (1 << 30) ||
      splits < 0 || q == nullptr || out == nullptr || (n > 0 && (k == nullptr || v == nullptr)) || !finite_scale(scale))
    return TC_ERR_INVALID;
  if (!i4_aligned(k, k_stride_b, k_stride_h, k_stride_n, d) || !i4_aligned(v, v_stride_b, v_stride_h, v_stride_n, d))
    return TC_ERR_ALIGN;
  Int4DecodeParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = q;
  p.out = out;
  p.k = k;
  p.v = v;
  p.lengths = lengths;
  p.n = n;
  p.sq_b = q_stride_b;
  p.sq_h = q_stride_h;
  p.sq_g = q_stride_g;
  p.so_b = out_stride_b;
  p.so_h = out_stride_h;
  p.so_g = out_stride_g;
  p.sk_b = k_stride_b;
  p.sk_h = k_stride_h;
  p.sk_n = k_stride_n;
  p.sv_b = v_stride_b;
  p.sv_h = v_stride_h;
  p.sv_n = v_stride_n;
  p.hkv = hkv;
  p.g = g;
  p.batch = batch;
  return run_int4_decode(p, d, n, scale, splits, dtype, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int tc_decode_attention_int4_paged(const void* q, const void* k_pool, const void* v_pool, void* out, int hkv, int g, int d,
                                   int64_t page_rows, int64_t num_pages, int64_t pool_stride_page, int64_t pool_stride_h,
                                   int64_t pool_stride_row, const int32_t* tiles, int tile_cols, int64_t n_tiles,
                                   int64_t q_stride_h, int64_t q_stride_g, int64_t out_stride_h, int64_t out_stride_g,
                                   float scale, int splits, int dtype, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (!i4_dtype(dtype)) return TC_ERR_DTYPE;
  if (!i4_pool(hkv, d, page_rows, num_pages) || g < 1 || g > 16 || n_tiles < 0 || n_tiles > (1 << 25) || tile_cols < 3 ||
      tile_cols > 65535 || splits < 0 || q == nullptr || out == nullptr || k_pool == nullptr || v_pool == nullptr ||
      (n_tiles > 0 && tiles == nullptr) || !finite_scale(scale))
    return TC_ERR_INVALID;
  if (!i4_aligned(k_pool, pool_stride_page, pool_stride_h, pool_stride_row, d) ||
      !i4_aligned(v_pool, 0, 0, 0, d))
    return TC_ERR_ALIGN;
  Int4DecodeParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = q;
  p.out = out;
  p.k = k_pool;
  p.v = v_pool;
  p.paged = 1;
  p.tiles = tiles;
  p.tile_cols = tile_cols;
  p.n_tiles = n_tiles;
  p.page_rows = page_rows;
  p.num_pages = num_pages;
  p.sq_h = q_stride_h;
  p.sq_g = q_stride_g;
  p.so_h = out_stride_h;
  p.so_g = out_stride_g;
  p.sk_b = p.sv_b = pool_stride_page;
  p.sk_h = p.sv_h = pool_stride_h;
  p.sk_n = p.sv_n = pool_stride_row;
  p.hkv = hkv;
  p.g = g;
  p.batch = 1;
  return run_int4_decode(p, d, n_tiles * kTile, scale, splits, dtype, workspace, workspace_bytes,
                         static_cast<cudaStream_t>(stream));
}

int tc_gemv_int4(const void* x, const void* codes, const void* params, void* out, int64_t n, int k, int64_t m, int group,
                 int64_t x_stride, int64_t out_stride, int swiglu, int dtype, void* stream) {
  if (!i4_dtype(dtype)) return TC_ERR_DTYPE;
  if (n < 0 || n > INT32_MAX || k < 1 || m < 0 || m > (1 << 20) || (group != 32 && group != 64 && group != 128) ||
      k > kGvMaxColumns)
    return TC_ERR_INVALID;
  if (n == 0 || m == 0) return TC_OK;
  if (x == nullptr || codes == nullptr || params == nullptr || out == nullptr) return TC_ERR_INVALID;
  if (!aligned16(codes) || !aligned16(params)) return TC_ERR_ALIGN;
  const int dev = current_device();
  const int streams = gv_streams(n, sm_count(dev));
  for (int64_t m0 = 0; m0 < m;) {
    Int4GemvParams p;
    std::memset(&p, 0, sizeof(p));
    // as many tokens a launch as fit, 32 at most; one always does as 16-bit numbers
    int now = (int)(m - m0 < 32 ? m - m0 : 32);
    bool digits = now <= kGvIntTokens;
    while (!gv_ring(gv_fixed(k, now, group, streams, digits), k, group, streams, p.chunk, p.stages)) {
      if (digits) {
        digits = false;
      } else if (--now == 0) {
        return TC_ERR_INVALID;
      }
    }
    p.x = static_cast<const uint16_t*>(x) + m0 * x_stride;
    p.codes = static_cast<const uint8_t*>(codes);
    p.params = params;
    p.out = static_cast<uint16_t*>(out) + m0 * out_stride;
    p.n = n;
    p.k = k;
    p.m = now;
    p.sx = x_stride;
    p.so = out_stride;
    p.swiglu = swiglu != 0;
    p.vec = aligned16(p.x) && (p.m == 1 || stride16(x_stride, dtype)) && (!p.swiglu || k % 8 == 0);
    p.streams = streams;
    for (p.slice_bits = 4; (kGvWarps >> p.slice_bits) < streams;) --p.slice_bits;
    p.part_bytes = gv_part_bytes(p.m, streams);
    p.flush = p.part_bytes / (kGvWarps * 64 * p.m) * streams;
    const int smem = (int)(gv_fixed(k, now, group, streams, digits) +
                           (int64_t)kGvWarps * p.chunk * p.stages * gv_tile_bytes(group));
    const cudaError_t e =
        dtype == TC_BF16 ? launch_int4_gemv<__nv_bfloat16>(p, group, digits, smem, dev, static_cast<cudaStream_t>(stream))
                         : launch_int4_gemv<__half>(p, group, digits, smem, dev, static_cast<cudaStream_t>(stream));
    m0 += now;
    if (e != cudaSuccess) return TC_ERR_CUDA;
  }
  return TC_OK;
}

}  // extern "C"
