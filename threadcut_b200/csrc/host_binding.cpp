// Host fast path of threadcut_b200.flash_decode.decode_attention (and decode_attention_partial):
// the tensor checks, the output
// allocation and the C-ABI call in one crossing from Python, instead of a ctypes call with 23
// converted arguments plus a dozen tensor attribute lookups in the interpreter. Host code only (no
// device code); it calls the library's tc_decode_attention_stable through a function pointer handed
// over by the ctypes loader, so it uses the very library instance the rest of the package loaded.
//
// decode(q, k, v, scale, splits, stable_rows, workspace) returns the output tensor, or None when
// anything is off (not CUDA, mixed devices or dtypes, wrong ranks or shapes, a non-contiguous last
// dimension, an unsupported dtype, or a non-zero status from the library): the caller then takes
// the checked Python path, which raises the documented exception for that case.
//
// append_rope, window_decode, window_prefill and shared_decode do the same for paged.append_rope,
// flash_decode.decode_attention_window / decode_attention_shared and prefill.prefill_attention_window.
#include <torch/extension.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <optional>
#include <tuple>

namespace {

using DecodeStableFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int64_t, int64_t,
                               int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, float, int, int,
                               int64_t, void*, size_t, void*);

using PartialStableFn = int (*)(const void*, const void*, const void*, float*, float*, int, int, int, int64_t,
                                int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, float, int,
                                int, int64_t, void*, size_t, void*);

DecodeStableFn g_decode = nullptr;
PartialStableFn g_partial = nullptr;

void init(int64_t decode_stable_addr) { g_decode = reinterpret_cast<DecodeStableFn>(decode_stable_addr); }
void init_partial(int64_t partial_stable_addr) {
  g_partial = reinterpret_cast<PartialStableFn>(partial_stable_addr);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: return -1;
  }
}

py::object decode(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale, int64_t splits,
                  int64_t stable_rows, const at::Tensor& ws) {
  if (g_decode == nullptr) return py::none();
  if (!q.is_cuda() || !k.is_cuda() || !v.is_cuda() || !ws.is_cuda()) return py::none();
  const auto dev = q.device();
  if (k.device() != dev || v.device() != dev || ws.device() != dev) return py::none();
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3) return py::none();
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return py::none();
  const int code = dtype_code(q.scalar_type());
  if (code < 0) return py::none();
  const int64_t hkv = q.size(0), g = q.size(1), d = q.size(2), n = k.size(1);
  if (k.size(0) != hkv || k.size(2) != d || v.sizes() != k.sizes()) return py::none();
  if (q.stride(2) != 1 || k.stride(2) != 1 || v.stride(2) != 1) return py::none();
  if (stable_rows < 0) return py::none();
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({hkv, g, d}, q.options());
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int rc = g_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), (int)hkv, (int)g, (int)d, n,
                          q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                          out.stride(0), out.stride(1), (float)scale, (int)splits, code, stable_rows,
                          ws.data_ptr(), (size_t)ws.numel(), st);
  if (rc != 0) return py::none();
  return py::cast(out);
}

// The same for decode_attention_partial: (out fp32 [hkv, g, d], lse fp32 [hkv, g]) through
// tc_decode_attention_partial_stable, or None.
py::object partial(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale, int64_t splits,
                   int64_t stable_rows, const at::Tensor& ws) {
  if (g_partial == nullptr) return py::none();
  if (!q.is_cuda() || !k.is_cuda() || !v.is_cuda() || !ws.is_cuda()) return py::none();
  const auto dev = q.device();
  if (k.device() != dev || v.device() != dev || ws.device() != dev) return py::none();
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3) return py::none();
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return py::none();
  const int code = dtype_code(q.scalar_type());
  if (code < 0) return py::none();
  const int64_t hkv = q.size(0), g = q.size(1), d = q.size(2), n = k.size(1);
  if (k.size(0) != hkv || k.size(2) != d || v.sizes() != k.sizes()) return py::none();
  if (q.stride(2) != 1 || k.stride(2) != 1 || v.stride(2) != 1) return py::none();
  if (stable_rows < 0) return py::none();
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({hkv, g, d}, q.options().dtype(at::kFloat));
  at::Tensor lse = at::empty({hkv, g}, q.options().dtype(at::kFloat));
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int rc = g_partial(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr<float>(), lse.data_ptr<float>(),
                           (int)hkv, (int)g, (int)d, n, q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                           v.stride(0), v.stride(1), out.stride(0), out.stride(1), (float)scale, (int)splits, code,
                           stable_rows, ws.data_ptr(), (size_t)ws.numel(), st);
  if (rc != 0) return py::none();
  return py::make_tuple(out, lse);
}

// ---- the serving operators. Each returns None where an argument is not of the plain kind; the Python path
// then converts it or raises.
using AppendFn = int (*)(const void*, const void*, const void*, void*, void*, void*, int, int, int, int64_t,
                         int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, const void*,
                         const void*, float, const void*, const void*, int, int64_t, int64_t, int, int64_t,
                         int64_t, int64_t, int64_t, int64_t, const int32_t*, int, void*);

using WindowFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int, int64_t, const int32_t*,
                         int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                         int64_t, int64_t, int64_t, int64_t, float, int, int, void*, size_t, void*);

using WindowSizeFn = size_t (*)(int, int, int, int, int64_t, int64_t, int64_t, int, int);

using PrefillFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int, int, int, int64_t,
                          int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                          int64_t, int64_t, int64_t, float, int, int, void*, size_t, void*);

using PrefillSizeFn = size_t (*)(int, int, int, int, int, int, int64_t, int64_t, int);

using SharedFn = int (*)(const void*, const void*, const void*, const void*, const void*, void*, int, int, int,
                         int, int64_t, int64_t, const int32_t*, int64_t, int64_t, int64_t, int64_t, int64_t,
                         int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                         int64_t, float, int, void*, size_t, void*);

using SharedSizeFn = size_t (*)(int, int, int, int, int64_t, int64_t, int);

AppendFn g_append = nullptr;
WindowFn g_window = nullptr;
WindowSizeFn g_window_size = nullptr;
PrefillFn g_prefill = nullptr;
PrefillSizeFn g_prefill_size = nullptr;
SharedFn g_shared = nullptr;
SharedSizeFn g_shared_size = nullptr;

void init_ops(int64_t append, int64_t window, int64_t window_size, int64_t prefill, int64_t prefill_size, int64_t shared,
              int64_t shared_size) {
  g_append = reinterpret_cast<AppendFn>(append);
  g_window = reinterpret_cast<WindowFn>(window);
  g_window_size = reinterpret_cast<WindowSizeFn>(window_size);
  g_prefill = reinterpret_cast<PrefillFn>(prefill);
  g_prefill_size = reinterpret_cast<PrefillSizeFn>(prefill_size);
  g_shared = reinterpret_cast<SharedFn>(shared);
  g_shared_size = reinterpret_cast<SharedSizeFn>(shared_size);
}

using OptTensor = std::optional<at::Tensor>;

// On `dev`, of type `t`, with a contiguous last dimension.
bool plain(const at::Tensor& x, const c10::Device& dev, at::ScalarType t) {
  return x.device() == dev && x.scalar_type() == t && x.dim() > 0 && x.stride(-1) == 1;
}

bool plain_lengths(const OptTensor& n, const c10::Device& dev, int64_t b) {
  return !n || (n->device() == dev && n->scalar_type() == at::kInt && n->dim() == 1 && n->size(0) == b && n->is_contiguous());
}
const int32_t* lengths_ptr(const OptTensor& n) { return n ? n->data_ptr<int32_t>() : nullptr; }

// x itself if a tensor map can describe it (rows on 16-byte boundaries, no broadcast dimension), else a copy that one
// can; the strides of extents of 1 count too, since the library checks them all. (rows16 of the Python side.)
at::Tensor rows16(const at::Tensor& x) {
  const int64_t es = x.element_size();
  bool ok = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < x.dim(); ++i)
    ok = ok && x.stride(i) * es % 16 == 0 && (x.stride(i) > 0 || x.size(i) <= 1);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

bool broadcast(const at::Tensor& x) {
  for (int64_t i = 0; i < x.dim(); ++i)
    if (x.stride(i) == 0 && x.size(i) > 1) return true;
  return false;
}

// Scratch with no initial contents.
at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

py::object append_rope(const at::Tensor& k, const at::Tensor& v, const at::Tensor& cos, const at::Tensor& sin,
                       const at::Tensor& k_pool, const at::Tensor& v_pool, const at::Tensor& slots, const at::Tensor& q,
                       const OptTensor& q_norm, const OptTensor& k_norm, double eps) {
  if (g_append == nullptr || !k.is_cuda()) return py::none();
  const auto dev = k.device();
  const auto dt = k.scalar_type();
  const int code = dtype_code(dt);
  // [h, t, d], or [1, h, t, d] throughout
  const int64_t o = k.dim() - 3;
  if (code < 0 || (o != 0 && o != 1) || q.dim() != k.dim() || v.sizes() != k.sizes()) return py::none();
  if (o == 1 && (k.size(0) != 1 || q.size(0) != 1)) return py::none();
  const int64_t hkv = k.size(o), t = k.size(o + 1), d = k.size(o + 2), hq = q.size(o);
  if (q.size(o + 1) != t || q.size(o + 2) != d) return py::none();
  if (!plain(k, dev, dt) || !plain(v, dev, dt) || !plain(q, dev, dt) || !plain(k_pool, dev, dt) ||
      !plain(v_pool, dev, dt))
    return py::none();
  const auto tab = cos.scalar_type();
  const int64_t c = cos.dim() - 2, s = sin.dim() - 2;
  if ((tab != dt && tab != at::kFloat) || (c != 0 && c != 1) || (s != 0 && s != 1) || (c == 1 && cos.size(0) != 1) ||
      (s == 1 && sin.size(0) != 1) || !plain(cos, dev, tab) || !plain(sin, dev, tab))
    return py::none();
  const int64_t rot = cos.size(c + 1);
  if (cos.size(c) != t || sin.size(s) != t || sin.size(s + 1) != rot) return py::none();
  if (k_pool.dim() != 4 || k_pool.size(1) != hkv || k_pool.size(3) != d || v_pool.sizes() != k_pool.sizes() ||
      v_pool.strides() != k_pool.strides())
    return py::none();
  if (slots.device() != dev || slots.scalar_type() != at::kInt || slots.dim() != 2 || slots.size(0) != t ||
      slots.size(1) != 2 || !slots.is_contiguous())
    return py::none();
  for (const OptTensor* w : {&q_norm, &k_norm})
    if (*w && (!plain(**w, dev, dt) || (*w)->dim() != 1 || (*w)->size(0) != d)) return py::none();
  if (hq > 65535 || hkv > 65535 || d > 65535 || rot > 65535) return py::none();
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = o == 0 ? at::empty_strided({hq, t, d}, {d, hq * d, 1}, q.options())
                          : at::empty_strided({1, hq, t, d}, {t * hq * d, d, hq * d, 1}, q.options());
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int rc = g_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                          (int)hq, (int)hkv, (int)d, t, q.stride(o), q.stride(o + 1), k.stride(o), k.stride(o + 1),
                          v.stride(o), v.stride(o + 1), d, hq * d, q_norm ? q_norm->data_ptr() : nullptr,
                          k_norm ? k_norm->data_ptr() : nullptr, (float)eps, cos.data_ptr(), sin.data_ptr(), (int)rot,
                          cos.stride(c), sin.stride(s), dtype_code(tab), k_pool.size(2), k_pool.size(0),
                          k_pool.stride(0), k_pool.stride(1), k_pool.stride(2), slots.data_ptr<int32_t>(), code, st);
  if (rc != 0) return py::none();
  return py::cast(out);
}

// Zeroed decode workspaces, one per (device, stream, sequences x heads) as the Python side keeps them; never
// freed with the process, whose CUDA context may go first.
at::Tensor& decode_workspace(const c10::Device& dev, cudaStream_t st, int64_t rows, size_t bytes, const at::Tensor& like) {
  static auto* cache = new std::map<std::tuple<int, cudaStream_t, int64_t>, at::Tensor>();
  at::Tensor& ws = (*cache)[{(int)dev.index(), st, rows}];
  if (!ws.defined() || (size_t)ws.numel() < bytes)
    ws = at::zeros({(int64_t)bytes}, like.options().dtype(at::kByte));
  return ws;
}

py::object window_decode(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale, int64_t window,
                         int64_t sinks, const OptTensor& lengths, int64_t splits) {
  if (g_window == nullptr || !q.is_cuda() || q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes()) return py::none();
  const auto dev = q.device();
  const auto dt = q.scalar_type();
  const int code = dtype_code(dt);
  const int64_t b = q.size(0), hkv = q.size(1), g = q.size(2), d = q.size(3), n = k.size(2);
  if (code < 0 || k.size(0) != b || k.size(1) != hkv || k.size(3) != d || !plain(q, dev, dt) || !plain(k, dev, dt) ||
      !plain(v, dev, dt) || !plain_lengths(lengths, dev, b) || window < 1 || sinks < 0 || b < 1 || b > 65535 ||
      hkv > 65535 || g > 65535 || d > 65535 || splits < 0 || splits > 65535)
    return py::none();
  c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  window = std::min(window, std::max<int64_t>(n, 1));
  sinks = std::min(sinks, n);
  const size_t nb = g_window_size((int)b, (int)hkv, (int)g, (int)d, n, window, sinks, (int)splits, code);
  void* ws = nullptr;
  if (nb > 0) {
    // a captured call gets a workspace of its graph's own
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return py::none();
    ws = decode_workspace(dev, st, b * hkv, nb, q).data_ptr();
  }
  at::Tensor out = at::empty({b, hkv, g, d}, q.options());
  const int rc = g_window(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), (int)b, (int)hkv, (int)g, (int)d, n,
                          lengths_ptr(lengths), window, sinks, q.stride(0), q.stride(1), q.stride(2), k.stride(0),
                          k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2), out.stride(0), out.stride(1),
                          out.stride(2), (float)scale, (int)splits, code, ws, nb, st);
  if (rc != 0) return py::none();
  return py::cast(out);
}

py::object window_prefill(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, double scale, int64_t window,
                          int64_t sinks, int64_t splits) {
  if (g_prefill == nullptr || !q_in.is_cuda() || q_in.dim() != 4 || k_in.dim() != 4 || v_in.sizes() != k_in.sizes()) return py::none();
  const auto dev = q_in.device();
  const auto dt = q_in.scalar_type();
  const int code = dtype_code(dt);
  const int64_t b = q_in.size(0), hq = q_in.size(1), lq = q_in.size(2), d = q_in.size(3), hkv = k_in.size(1), lk = k_in.size(2);
  if (code < 0 || k_in.size(0) != b || k_in.size(3) != d || hkv < 1 || hq % hkv != 0 || lq < 1 || lq > lk || lk > INT32_MAX ||
      !plain(q_in, dev, dt) || !plain(k_in, dev, dt) || !plain(v_in, dev, dt) || window < 1 || sinks < 0 || b < 1 || b > 65535 ||
      hq > 65535 || d > 65535 || splits < 0 || splits > 65535)
    return py::none();
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = rows16(q_in);
  // for the tensor cores, as on the Python side
  const bool map = code != dtype_code(at::kFloat) && (d == 64 || d == 128);
  const at::Tensor k = map && !broadcast(k_in) ? rows16(k_in) : k_in, v = map && !broadcast(v_in) ? rows16(v_in) : v_in;
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  window = std::min(window, lk);
  sinks = std::min(sinks, lk);
  at::Tensor out = at::empty({b, lq, hq, d}, q.options());
  const size_t nb = g_prefill_size((int)b, (int)hq, (int)hkv, (int)lq, (int)lk, (int)d, window, sinks, (int)splits);
  at::Tensor ws;
  if (nb > 0) ws = scratch(nb, q);
  const int rc = g_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), (int)b, (int)hq, (int)hkv, (int)lq,
                           (int)lk, (int)d, window, sinks, q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1),
                           k.stride(2), v.stride(0), v.stride(1), v.stride(2), out.stride(0), out.stride(1),
                           out.stride(2), (float)scale, (int)splits, code, nb > 0 ? ws.data_ptr() : nullptr, nb, st);
  if (rc != 0) return py::none();
  return py::cast(out);
}

py::object shared_decode(const at::Tensor& q_in, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& k,
                         const at::Tensor& v, double scale, const OptTensor& lengths) {
  if (g_shared == nullptr || !q_in.is_cuda() || q_in.dim() != 4 || kp.dim() != 3 || k.dim() != 4 || vp.sizes() != kp.sizes() ||
      v.sizes() != k.sizes())
    return py::none();
  const auto dev = q_in.device();
  const auto dt = q_in.scalar_type();
  const int code = dtype_code(dt);
  const int64_t b = q_in.size(0), hkv = q_in.size(1), g = q_in.size(2), d = q_in.size(3), n = kp.size(1), m = k.size(2);
  if (code < 0 || kp.size(0) != hkv || kp.size(2) != d || k.size(0) != b || k.size(1) != hkv || k.size(3) != d ||
      !plain(q_in, dev, dt) || !plain(kp, dev, dt) || !plain(vp, dev, dt) || !plain(k, dev, dt) || !plain(v, dev, dt) ||
      !plain_lengths(lengths, dev, b) || b < 1 || b > 65535 || hkv > 65535 || g > 65535 || d > 65535)
    return py::none();
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = rows16(q_in);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  at::Tensor out = at::empty({b, hkv, g, d}, q.options());
  const size_t nb = g_shared_size((int)b, (int)hkv, (int)g, (int)d, n, m, code);
  at::Tensor ws;
  if (nb > 0) ws = scratch(nb, q);
  const int rc = g_shared(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), (int)b,
                          (int)hkv, (int)g, (int)d, n, m, lengths_ptr(lengths), q.stride(0), q.stride(1), q.stride(2),
                          kp.stride(0), kp.stride(1), vp.stride(0), vp.stride(1), k.stride(0), k.stride(1), k.stride(2),
                          v.stride(0), v.stride(1), v.stride(2), out.stride(0), out.stride(1), out.stride(2),
                          (float)scale, code, nb > 0 ? ws.data_ptr() : nullptr, nb, st);
  if (rc != 0) return py::none();
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("init", &init, "set the address of tc_decode_attention_stable");
  m.def("init_partial", &init_partial, "set the address of tc_decode_attention_partial_stable");
  m.def("decode", &decode, "checked decode_attention fast path; None means: take the Python path");
  m.def("init_ops", &init_ops, "set the addresses of the serving operators' entry points");
  m.def("append_rope", &append_rope, "checked paged.append_rope fast path; None means: take the Python path");
  m.def("window_decode", &window_decode, "checked decode_attention_window fast path; None means: take the Python path");
  m.def("window_prefill", &window_prefill, "checked prefill_attention_window fast path; None means: take the Python path");
  m.def("shared_decode", &shared_decode, "checked decode_attention_shared fast path; None means: take the Python path");
  m.def("partial", &partial, "checked decode_attention_partial fast path; None means: take the Python path");
}
