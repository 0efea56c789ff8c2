// Python binding of the per-call hot path (marlin_gemm_fp4 / marlin_gemm_int4,
// the fused QKV and gate/up projections, the row-packed product, their input
// gradients and the low-rank adapters) for callers
// that issue one projection per Python call.  It does in C++ what the
// ctypes path does in Python -- shape checks, the output allocation, the
// per-(device, stream) workspace -- and calls the same C ABI entry points of
// libmmfp4.so (mm_fp4_gemm / mm_u4_gemm).  torch is used only for tensor
// arguments and the output allocation; the stream comes from the caller.
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <map>
#include <mutex>
#include <sstream>
#include <utility>

#include "mmfp4.h"

namespace {

[[noreturn]] void fail(int rc) {
  const char* msg = mm_last_error();
  if (rc == 1) throw pybind11::value_error(msg);
  throw std::runtime_error(msg);
}

std::mutex g_mu;
std::map<std::pair<int, int64_t>, at::Tensor> g_ws;   // (device index, stream) -> workspace
struct Captured {
  unsigned long long id;   // of the capture
  at::Tensor buf;
};
std::map<std::pair<int, int64_t>, Captured> g_captured;

// One workspace per (device, stream), shared with the ctypes path (which
// asks for it through workspace_for below); kept until release_workspaces().
// Under capture one per capture and stream, from the graph's pool, its counters cleared by a
// node of that graph: graphs never share one, with one another or with eager calls, and none
// relies on a fill that only another one replays.  It is held until the stream is used again
// outside that capture; the graph's pool keeps the memory as long as the graph lives.
at::Tensor workspace_dev(int dev, int64_t stream, size_t nbytes, const at::TensorOptions& opt) {
  std::lock_guard<std::mutex> lock(g_mu);
  const auto key = std::make_pair(dev, stream);
  if (const unsigned long long id = mm_capture_id((void*)stream)) {
    Captured& c = g_captured[key];
    if (c.id == id && (size_t)c.buf.numel() >= nbytes) return c.buf;
    size_t size = std::max(nbytes, (size_t)1 << 20);
    if (c.id == id) size = std::max(size, 2 * (size_t)c.buf.numel());
    c = Captured{0, at::Tensor()};
    at::Tensor buf = at::empty({(int64_t)size}, opt.dtype(at::kByte));
    if (const int rc = mm_clear_counters(buf.data_ptr(), size, (void*)stream)) fail(rc);
    c = Captured{id, buf};
    return buf;
  }
  if (!g_captured.empty()) g_captured.erase(key);
  auto it = g_ws.find(key);
  if (it != g_ws.end() && (size_t)it->second.numel() >= nbytes) return it->second;
  size_t size = nbytes < ((size_t)1 << 20) ? ((size_t)1 << 20) : nbytes;
  if (it != g_ws.end() && size < 2 * (size_t)it->second.numel()) size = 2 * it->second.numel();
  // Zero-filled once: the split-K arrival counters at its head must start at
  // zero, and every call leaves them at zero.
  at::Tensor buf = at::zeros({(int64_t)size}, opt.dtype(at::kByte));
  g_ws[key] = buf;
  return buf;
}

at::Tensor workspace(const at::Tensor& like, int64_t stream, size_t nbytes) {
  return workspace_dev((int)like.get_device(), stream, nbytes, like.options());
}

at::Tensor workspace_for(int64_t device, int64_t stream, int64_t nbytes) {
  return workspace_dev((int)device, stream, (size_t)nbytes,
                       at::TensorOptions().device(at::kCUDA, (int)device));
}

void release_workspaces() {
  std::lock_guard<std::mutex> lock(g_mu);
  g_ws.clear();
  g_captured.clear();
}

void check_groups(const char* name, const at::Tensor& t, int64_t K, int64_t N, int64_t g) {
  if (g <= 0 || K % g != 0) {
    std::ostringstream os;
    os << name << ": K=" << K << " must be divisible by group_size=" << g;
    throw pybind11::value_error(os.str());
  }
  if (t.dim() != 2 || t.size(0) != K / g || t.size(1) != N) {
    std::ostringstream os;
    os << name << ": " << name << " shape " << t.sizes() << " != (" << K / g << ", " << N
       << ") for K=" << K << ", group_size=" << g;
    throw pybind11::value_error(os.str());
  }
}

at::Tensor half_contig(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf && t.is_contiguous() ? t : t.to(at::kHalf).contiguous();
}

// C = A . dequant(B, S[, Z]) for A [*, K], B [K/8, N] words; fp16 [*, N].
// SZ (INT4 only, optional): the scales and zeros interleaved [K/g, N/4, 8]
// for the decode kernels (mm_u4_gemm_sz).
at::Tensor gemm(const at::Tensor& A, const at::Tensor& B, const at::Tensor& S,
                const c10::optional<at::Tensor>& Z, const c10::optional<at::Tensor>& SZ,
                int64_t group_size, int64_t stream) {
  const int dev = A.get_device();
  if (dev < 0 || B.get_device() != dev || S.get_device() != dev ||
      (Z && Z->get_device() != dev)) {
    std::ostringstream os;
    os << "tensor on " << (dev < 0 ? A.device() : B.device())
       << ": the FP4/INT4 kernels run on the GPU only, with every operand on one device";
    throw std::runtime_error(os.str());
  }
  if (B.dim() != 2) throw pybind11::value_error("B_packed must be [K/8, N]");
  if (B.scalar_type() != at::kInt && B.scalar_type() != at::kUInt32)
    throw pybind11::type_error("packed weights must be int32/uint32 words");
  const int64_t K = A.size(-1);
  const int64_t M = K ? A.numel() / K : 0;
  const int64_t N = B.size(1);
  if (B.size(0) * 8 != K) {
    std::ostringstream os;
    os << "Packed K " << B.size(0) * 8 << " does not match activations K " << K;
    throw pybind11::value_error(os.str());
  }
  check_groups("scales", S, K, N, group_size);
  if (Z) check_groups("zeros", *Z, K, N, group_size);
  const at::Tensor a = half_contig(A);
  const at::Tensor b = B.is_contiguous() ? B : B.contiguous();
  const at::Tensor s = half_contig(S);
  std::vector<int64_t> oshape(A.sizes().begin(), A.sizes().end());
  oshape.back() = N;
  at::Tensor out = at::empty(oshape, a.options());
  const size_t need = mm_gemm_workspace_bytes((int)M, (int)N, (int)K);
  at::Tensor ws = workspace(a, stream, need);
  int rc;
  if (!Z) {
    rc = mm_fp4_gemm((const uint16_t*)a.data_ptr(), (const uint32_t*)b.data_ptr(),
                     (const uint16_t*)s.data_ptr(), (uint16_t*)out.data_ptr(), (int)M, (int)N,
                     (int)K, (int)group_size, ws.data_ptr(), (size_t)ws.numel(),
                     (void*)stream);
  } else if (SZ) {
    const at::Tensor z = half_contig(*Z);
    if (SZ->scalar_type() != at::kHalf || !SZ->is_contiguous() || SZ->numel() != 2 * z.numel() ||
        SZ->get_device() != dev)
      throw pybind11::value_error("SZ must be contiguous fp16 [K/g, 2N] on the operands' device");
    rc = mm_u4_gemm_sz((const uint16_t*)a.data_ptr(), (const uint32_t*)b.data_ptr(),
                       (const uint16_t*)s.data_ptr(), (const uint16_t*)z.data_ptr(),
                       (const uint16_t*)SZ->data_ptr(), (uint16_t*)out.data_ptr(), (int)M,
                       (int)N, (int)K, (int)group_size, ws.data_ptr(), (size_t)ws.numel(),
                       (void*)stream);
  } else {
    const at::Tensor z = half_contig(*Z);
    rc = mm_u4_gemm((const uint16_t*)a.data_ptr(), (const uint32_t*)b.data_ptr(),
                    (const uint16_t*)s.data_ptr(), (const uint16_t*)z.data_ptr(),
                    (uint16_t*)out.data_ptr(), (int)M, (int)N, (int)K, (int)group_size,
                    ws.data_ptr(), (size_t)ws.numel(), (void*)stream);
  }
  if (rc) fail(rc);
  return out;
}

// The fused projections below take the plain form of their operands only --
// contiguous fp16 activations and scales and packed words on one device, shapes
// that agree -- and return None for anything else, which their Python callers
// then convert or refuse.
bool plain(const at::Tensor& t, at::ScalarType type, int dev, int64_t d0, int64_t d1) {
  return t.dim() == 2 && t.size(0) == d0 && t.size(1) == d1 && t.get_device() == dev &&
         t.is_contiguous() && t.scalar_type() == type;
}
bool plain_words(const at::Tensor& t, int dev, int64_t d0, int64_t d1) {
  return plain(t, t.scalar_type() == at::kUInt32 ? at::kUInt32 : at::kInt, dev, d0, d1);
}
// [M, K] of the activations, or M = -1.
std::pair<int64_t, int64_t> plain_acts(const at::Tensor& A) {
  if (A.dim() != 2 || A.get_device() < 0 || !A.is_contiguous() || A.scalar_type() != at::kHalf ||
      A.size(0) == 0 || A.size(1) == 0)
    return {-1, 0};
  return {A.size(0), A.size(1)};
}

// Q, K, V = A . dequant(W[p], S[p]) in one mm_fp4_gemm_multi call.
pybind11::object qkv(const at::Tensor& A, const std::array<at::Tensor, 3>& W,
                     const std::array<at::Tensor, 3>& S, int64_t g, int64_t stream) {
  const auto [M, K] = plain_acts(A);
  if (M < 0 || g <= 0 || K % g != 0 || K % 8 != 0) return pybind11::none();
  const int dev = (int)A.get_device();
  const uint32_t* b[3];
  const uint16_t* s[3];
  uint16_t* c[3];
  int n[3];
  int64_t ntot = 0;
  for (int p = 0; p < 3; ++p) {
    const int64_t N = W[p].dim() == 2 ? W[p].size(1) : 0;
    if (N <= 0 || N % 4 != 0 || !plain_words(W[p], dev, K / 8, N) ||
        !plain(S[p], at::kHalf, dev, K / g, N))
      return pybind11::none();
    n[p] = (int)N;
    ntot += N;
  }
  at::Tensor out[3];
  size_t need = mm_gemm_workspace_bytes((int)M, (int)ntot, (int)K);
  for (int p = 0; p < 3; ++p) {
    out[p] = at::empty({M, n[p]}, A.options());
    need = std::max(need, mm_gemm_workspace_bytes((int)M, n[p], (int)K));
    b[p] = (const uint32_t*)W[p].data_ptr();
    s[p] = (const uint16_t*)S[p].data_ptr();
    c[p] = (uint16_t*)out[p].data_ptr();
  }
  at::Tensor ws = workspace(A, stream, need);
  const int rc = mm_fp4_gemm_multi((const uint16_t*)A.data_ptr(), 3, b, s, c, n, (int)M, (int)K,
                                   (int)g, ws.data_ptr(), (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::make_tuple(out[0], out[1], out[2]);
}

// The gate/up pair: Marlin [K/8, N] words, or row-packed [N, K/8] ones.
pybind11::object gate_up(const at::Tensor& A, const at::Tensor& Wg, const at::Tensor& Sg,
                         const at::Tensor& Wu, const at::Tensor& Su, int64_t g, bool rows,
                         bool act, int64_t stream) {
  const auto [M, K] = plain_acts(A);
  if (M < 0 || g <= 0 || K % g != 0 || K % 8 != 0 || Wg.dim() != 2) return pybind11::none();
  const int dev = (int)A.get_device();
  const int64_t N = Wg.size(rows ? 0 : 1), d0 = rows ? N : K / 8, d1 = rows ? K / 8 : N;
  if (N <= 0 || N % 8 != 0 || !plain_words(Wg, dev, d0, d1) || !plain_words(Wu, dev, d0, d1) ||
      !plain(Sg, at::kHalf, dev, K / g, N) || !plain(Su, at::kHalf, dev, K / g, N))
    return pybind11::none();
  at::Tensor out = at::empty({M, act ? N : 2 * N}, A.options());
  at::Tensor ws = workspace(A, stream, mm_gemm_workspace_bytes((int)M, (int)(2 * N), (int)K));
  const auto fn = rows ? mm_fp4_gate_up_rowpacked : mm_fp4_gate_up;
  const int rc = fn((const uint16_t*)A.data_ptr(), (const uint32_t*)Wg.data_ptr(),
                    (const uint16_t*)Sg.data_ptr(), (const uint32_t*)Wu.data_ptr(),
                    (const uint16_t*)Su.data_ptr(), (uint16_t*)out.data_ptr(), (int)M, (int)N,
                    (int)K, (int)g, act, ws.data_ptr(), (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

// Row-packed product: W [N, K/8], scales [K/g, N].
pybind11::object rowpacked(const at::Tensor& A, const at::Tensor& W, const at::Tensor& S,
                           int64_t g, int64_t stream) {
  const auto [M, K] = plain_acts(A);
  if (M < 0 || g <= 0 || K % g != 0 || K % 8 != 0 || W.dim() != 2) return pybind11::none();
  const int dev = (int)A.get_device();
  const int64_t N = W.size(0);
  if (N <= 0 || !plain_words(W, dev, N, K / 8) || !plain(S, at::kHalf, dev, K / g, N))
    return pybind11::none();
  at::Tensor out = at::empty({M, N}, A.options());
  at::Tensor ws = workspace(A, stream, mm_gemm_workspace_bytes((int)M, (int)N, (int)K));
  const int rc = mm_fp4_gemm_rowpacked(
      (const uint16_t*)A.data_ptr(), (const uint32_t*)W.data_ptr(), (const uint16_t*)S.data_ptr(),
      (uint16_t*)out.data_ptr(), (int)M, (int)N, (int)K, (int)g, 0, ws.data_ptr(),
      (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

// ---------------------------------------------------------------------------
// Training and adapters.  As above: plain operands on the current device (contiguous,
// 16-byte aligned, N % 8 == 0), or None.
// ---------------------------------------------------------------------------
int type_code(at::ScalarType t) {
  return t == at::kFloat ? 0 : (t == at::kHalf ? 1 : (t == at::kBFloat16 ? 2 : -1));
}
bool on_current_device(int dev) {
  return dev >= 0 &&
         c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index() == dev;
}
bool aligned(const at::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
// [*, n] rows in plain form: their number, or -1.
int64_t plain_rows(const at::Tensor& t, int dev, int64_t n) {
  if (t.dim() < 1 || t.size(-1) != n || t.get_device() != dev || !t.is_contiguous() ||
      !aligned(t) || type_code(t.scalar_type()) < 0)
    return -1;
  return t.numel() / n;
}
// Whether t is [*, n] with x's leading axes, plain but for its alignment.
bool same_rows(const at::Tensor& t, const at::Tensor& x, int64_t n) {
  return t.dim() == x.dim() && t.get_device() == x.get_device() && t.is_contiguous() &&
         t.size(-1) == n && t.sizes().slice(0, t.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
}
at::Tensor rows_like(const at::Tensor& t, int64_t n, at::ScalarType type) {
  std::vector<int64_t> shape(t.sizes().begin(), t.sizes().end());
  shape.back() = n;
  return at::empty(shape, t.options().dtype(type));
}
struct Matrix {
  const uint32_t* w;
  const uint16_t *s, *z;
  int64_t N, K;
};
// A quantized matrix in plain form; N = 0 if it is none.
Matrix plain_matrix(const at::Tensor& W, const at::Tensor& S, const c10::optional<at::Tensor>& Z,
                    bool rows, int64_t g, int dev) {
  Matrix m{nullptr, nullptr, nullptr, 0, 0};
  if (W.dim() != 2 || g <= 0) return m;
  const int64_t N = W.size(rows ? 0 : 1), K = 8 * W.size(rows ? 1 : 0);
  if (N <= 0 || N % 8 != 0 || K <= 0 || K % g != 0 || (rows && K % 32 != 0) ||
      !plain_words(W, dev, W.size(0), W.size(1)) || !plain(S, at::kHalf, dev, K / g, N) ||
      !aligned(W) || !aligned(S))
    return m;
  if (Z && (!plain(*Z, at::kHalf, dev, K / g, N) || !aligned(*Z))) return m;
  m.w = (const uint32_t*)W.data_ptr();
  m.s = (const uint16_t*)S.data_ptr();
  m.z = Z ? (const uint16_t*)Z->data_ptr() : nullptr;
  m.N = N;
  m.K = K;
  return m;
}
// dA of up to three matrices from fp16 gradients.
at::Tensor backward(const at::Tensor& like, int nmat, const uint16_t* const* dC, const int* ldc,
                    const float* mul, const Matrix* mats, bool rows, int64_t M, int64_t g,
                    at::ScalarType out_type, int64_t stream) {
  const int64_t K = mats[0].K;
  at::Tensor out = rows_like(like, K, out_type);
  if (M == 0) return out;
  const uint32_t* w[3];
  const uint16_t *s[3], *z[3];
  int n[3];
  for (int i = 0; i < nmat; ++i) {
    w[i] = mats[i].w;
    s[i] = mats[i].s;
    z[i] = mats[i].z;
    n[i] = (int)mats[i].N;
  }
  at::Tensor ws = workspace(like, stream, mm_gemm_backward_workspace_bytes(nmat, n, (int)M, (int)K));
  const int rc = mm_gemm_backward(dC, ldc, mul, nmat, w, s, z[0] ? z : nullptr, n, rows,
                                  out.data_ptr(), type_code(out_type), (int)M, (int)K, (int)g,
                                  ws.data_ptr(), (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return out;
}
// fp16 values [M, sum N] of gradients side by side, and their rows' factors.
std::pair<at::Tensor, at::Tensor> carried(const at::Tensor* d, const int* N, int nmat, int64_t M,
                                          int64_t stream) {
  int64_t n = 0;
  const void* x[3];
  for (int i = 0; i < nmat; ++i) {
    n += N[i];
    x[i] = d[i].data_ptr();
  }
  at::Tensor y = at::empty({M, n}, d[0].options().dtype(at::kHalf));
  at::Tensor mul = at::empty({M}, d[0].options().dtype(at::kFloat));
  const int rc = mm_grad_rows_multi(x, type_code(d[0].scalar_type()), nmat, N,
                                    (uint16_t*)y.data_ptr(), (float*)mul.data_ptr(), (int)M,
                                    (void*)stream);
  if (rc) fail(rc);
  return {y, mul};
}
// dA of up to three matrices, all gradients of one type.
at::Tensor backward_any(const at::Tensor* dC, int nmat, const Matrix* mats, bool rows, int64_t M,
                        int64_t g, int64_t stream) {
  const uint16_t* p[3];
  int n[3], ld[3];
  for (int i = 0; i < nmat; ++i) {
    p[i] = (const uint16_t*)dC[i].data_ptr();
    ld[i] = n[i] = (int)mats[i].N;
  }
  const auto type = dC[0].scalar_type();
  if (type == at::kHalf) return backward(dC[0], nmat, p, ld, nullptr, mats, rows, M, g, type, stream);
  const auto [y, mul] = carried(dC, n, nmat, M, stream);
  const uint16_t* at = (const uint16_t*)y.data_ptr();
  for (int i = 0; i < nmat; ++i) {
    p[i] = at;
    at += n[i];
    ld[i] = (int)y.size(1);
  }
  return backward(dC[0], nmat, p, ld, (const float*)mul.data_ptr(), mats, rows, M, g, type, stream);
}

pybind11::object linear_backward(const at::Tensor& dC, const at::Tensor& W, const at::Tensor& S,
                                 const c10::optional<at::Tensor>& Z, bool rows, int64_t g,
                                 int64_t stream) {
  const int dev = (int)dC.get_device();
  if (!on_current_device(dev)) return pybind11::none();
  const Matrix m = plain_matrix(W, S, Z, rows, g, dev);
  const int64_t M = m.N ? plain_rows(dC, dev, m.N) : -1;
  if (M < 0) return pybind11::none();
  return pybind11::cast(backward_any(&dC, 1, &m, rows, M, g, stream));
}

pybind11::object qkv_backward(const std::array<at::Tensor, 3>& dC,
                              const std::array<at::Tensor, 3>& W,
                              const std::array<at::Tensor, 3>& S, int64_t g, int64_t stream) {
  const int dev = (int)dC[0].get_device();
  if (!on_current_device(dev)) return pybind11::none();
  Matrix m[3];
  int64_t M = 0;
  for (int i = 0; i < 3; ++i) {
    m[i] = plain_matrix(W[i], S[i], c10::nullopt, false, g, dev);
    const int64_t rows = m[i].N ? plain_rows(dC[i], dev, m[i].N) : -1;
    if (rows < 0 || dC[i].scalar_type() != dC[0].scalar_type() || m[i].K != m[0].K ||
        dC[i].sizes().slice(0, dC[i].dim() - 1) != dC[0].sizes().slice(0, dC[0].dim() - 1))
      return pybind11::none();
    M = rows;
  }
  return pybind11::cast(backward_any(dC.data(), 3, m, false, M, g, stream));
}

pybind11::object gate_up_keep(const at::Tensor& A, const at::Tensor& Wg, const at::Tensor& Sg,
                              const at::Tensor& Wu, const at::Tensor& Su, int64_t g, bool rows,
                              int64_t stream) {
  const int dev = (int)A.get_device();
  if (!on_current_device(dev) || A.scalar_type() != at::kHalf) return pybind11::none();
  const Matrix mg = plain_matrix(Wg, Sg, c10::nullopt, rows, g, dev);
  const Matrix mu = plain_matrix(Wu, Su, c10::nullopt, rows, g, dev);
  const int64_t N = mg.N, K = mg.K, M = N ? plain_rows(A, dev, K) : -1;
  if (M <= 0 || mu.N != N || mu.K != K || (M > 32 && K % 64 != 0) ||
      (rows && g % (M <= 32 ? 32 : 64) != 0))
    return pybind11::none();
  at::Tensor h = rows_like(A, N, at::kHalf), keep = rows_like(A, 2 * N, at::kHalf);
  at::Tensor ws = workspace(A, stream, mm_gemm_workspace_bytes((int)M, (int)(2 * N), (int)K));
  const int rc = mm_fp4_gate_up_keep((const uint16_t*)A.data_ptr(), mg.w, mg.s, mu.w, mu.s,
                                     (uint16_t*)h.data_ptr(), (uint16_t*)keep.data_ptr(), rows,
                                     (int)M, (int)N, (int)K, (int)g, ws.data_ptr(),
                                     (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::make_tuple(h, keep);
}

pybind11::object gate_up_backward(const at::Tensor& dH, const at::Tensor& keep,
                                  const at::Tensor& Wg, const at::Tensor& Sg,
                                  const at::Tensor& Wu, const at::Tensor& Su, int64_t g, bool rows,
                                  int64_t stream) {
  const int dev = (int)dH.get_device();
  if (!on_current_device(dev)) return pybind11::none();
  const Matrix m[2] = {plain_matrix(Wg, Sg, c10::nullopt, rows, g, dev),
                       plain_matrix(Wu, Su, c10::nullopt, rows, g, dev)};
  const int64_t N = m[0].N, M = N ? plain_rows(dH, dev, N) : -1;
  if (M <= 0 || m[1].N != N || m[1].K != m[0].K || keep.scalar_type() != at::kHalf ||
      !same_rows(keep, dH, 2 * N) || !aligned(keep))
    return pybind11::none();
  at::Tensor d = at::empty({M, 2 * N}, keep.options());
  at::Tensor mul = at::empty({M}, keep.options().dtype(at::kFloat));
  const int rc = mm_swiglu_grad(dH.data_ptr(), type_code(dH.scalar_type()),
                                (const uint16_t*)keep.data_ptr(), (uint16_t*)d.data_ptr(),
                                (float*)mul.data_ptr(), (int)M, (int)N, (void*)stream);
  if (rc) fail(rc);
  const uint16_t* p[2] = {(const uint16_t*)d.data_ptr(), (const uint16_t*)d.data_ptr() + N};
  const int ld[2] = {(int)(2 * N), (int)(2 * N)};
  return pybind11::cast(backward(dH, 2, p, ld, (const float*)mul.data_ptr(), m, rows, M, g,
                                 dH.scalar_type(), stream));
}

// The adapters' operands in plain form.
struct Lora {
  int64_t T, K, N, r, L;
  int type, ids64;
  const void* ids;
  const float* scaling;
};
bool plain_lora(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                const c10::optional<at::Tensor>& ids, const c10::optional<at::Tensor>& scaling,
                Lora* l) {
  const int dev = (int)x.get_device();
  const auto t = x.scalar_type();
  if (!on_current_device(dev) || (t != at::kHalf && t != at::kBFloat16) || a.dim() != 3 ||
      b.dim() != 3)
    return false;
  *l = Lora{0, a.size(2), b.size(1), a.size(1), a.size(0), type_code(t), 0, nullptr, nullptr};
  if (l->K <= 0 || l->N <= 0 || l->r <= 0 || l->L <= 0 || x.dim() < 1 || x.size(-1) != l->K ||
      !x.is_contiguous() || b.size(0) != l->L || b.size(2) != l->r)
    return false;
  l->T = x.numel() / l->K;
  for (const at::Tensor* w : {&a, &b})
    if (w->get_device() != dev || w->scalar_type() != t || !w->is_contiguous()) return false;
  if (ids) {
    l->ids64 = ids->scalar_type() == at::kLong;
    if (ids->get_device() != dev || (!l->ids64 && ids->scalar_type() != at::kInt) ||
        !ids->is_contiguous() || ids->dim() != 1 || ids->numel() != l->T)
      return false;
    l->ids = ids->data_ptr();
  } else if (l->L != 1) {
    return false;
  }
  if (scaling) {
    if (scaling->get_device() != dev || scaling->scalar_type() != at::kFloat ||
        !scaling->is_contiguous() || scaling->dim() != 1 || scaling->numel() != l->L)
      return false;
    l->scaling = (const float*)scaling->data_ptr();
  }
  return l->T > 0;
}

pybind11::object lora_add(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a,
                          const at::Tensor& b, const c10::optional<at::Tensor>& ids,
                          const c10::optional<at::Tensor>& scaling, double factor,
                          int64_t stream) {
  Lora l;
  if (!plain_lora(x, a, b, ids, scaling, &l) || !same_rows(base, x, l.N) ||
      (base.scalar_type() != at::kHalf && base.scalar_type() != x.scalar_type()))
    return pybind11::none();
  at::Tensor out = rows_like(x, l.N, x.scalar_type());
  at::Tensor ws = workspace(x, stream, mm_lora_workspace_bytes((int)l.T, (int)l.K, (int)l.N,
                                                               (int)l.r, (int)l.L, 0));
  const int rc = mm_lora_add((const uint16_t*)x.data_ptr(), l.type,
                             (const uint16_t*)base.data_ptr(), type_code(base.scalar_type()),
                             (uint16_t*)out.data_ptr(), (const uint16_t*)a.data_ptr(),
                             (const uint16_t*)b.data_ptr(), l.ids, l.ids64, l.scaling,
                             (float)factor, (int)l.T, (int)l.K, (int)l.N, (int)l.r, (int)l.L,
                             ws.data_ptr(), (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

pybind11::object lora_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& a,
                               const at::Tensor& b, const c10::optional<at::Tensor>& ids,
                               const c10::optional<at::Tensor>& scaling, double factor,
                               const c10::optional<at::Tensor>& dx_base, int64_t stream) {
  Lora l;
  if (!plain_lora(x, a, b, ids, scaling, &l) || !same_rows(dy, x, l.N) ||
      dy.scalar_type() != x.scalar_type() ||
      (dx_base && (!same_rows(*dx_base, x, l.K) || dx_base->scalar_type() != x.scalar_type())))
    return pybind11::none();
  at::Tensor dx = at::empty_like(x), da = at::empty_like(a), db = at::empty_like(b);
  at::Tensor ws = workspace(x, stream, mm_lora_workspace_bytes((int)l.T, (int)l.K, (int)l.N,
                                                               (int)l.r, (int)l.L, 1));
  const int rc = mm_lora_backward(
      (const uint16_t*)dy.data_ptr(), (const uint16_t*)x.data_ptr(), l.type,
      (const uint16_t*)a.data_ptr(), (const uint16_t*)b.data_ptr(), l.ids, l.ids64, l.scaling,
      (float)factor, dx_base ? (const uint16_t*)dx_base->data_ptr() : nullptr,
      (uint16_t*)dx.data_ptr(), da.data_ptr(), db.data_ptr(), l.type, (int)l.T, (int)l.K, (int)l.N,
      (int)l.r, (int)l.L, ws.data_ptr(), (size_t)ws.numel(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::make_tuple(dx, da, db);
}

// ---------------------------------------------------------------------------
// Microscaled 4-bit floating point: plain operands on the current device, or None.
// ---------------------------------------------------------------------------
// The words [.., N, K/8] and scales [.., N, K/32] of weights, of n axes.
bool plain_mx(const at::Tensor& W, const at::Tensor& S, int dev, int n) {
  if (W.dim() != n || S.dim() != n || W.get_device() != dev || S.get_device() != dev ||
      (W.scalar_type() != at::kInt && W.scalar_type() != at::kUInt32) ||
      S.scalar_type() != at::kByte || !W.is_contiguous() || !S.is_contiguous() || !aligned(W) ||
      !aligned(S) ||
      W.numel() == 0 || W.size(n - 1) != 4 * S.size(n - 1))
    return false;
  return W.sizes().slice(0, n - 1) == S.sizes().slice(0, n - 1);
}
at::ScalarType scalar_type_of(int64_t code) {
  return code == 0 ? at::kFloat : (code == 1 ? at::kHalf : at::kBFloat16);
}

// out_type: 0 fp32, 1 fp16, 2 bf16, -1 x's.
pybind11::object mx_gemm(const at::Tensor& x, const at::Tensor& W, const at::Tensor& S,
                         int64_t out_type, int64_t stream) {
  const int dev = (int)x.get_device();
  if (!on_current_device(dev) || !plain_mx(W, S, dev, 2)) return pybind11::none();
  const int64_t N = W.size(0), K = 8 * W.size(1), M = plain_rows(x, dev, K);
  if (M < 0 || M > INT32_MAX || N > INT32_MAX) return pybind11::none();
  const int type = type_code(x.scalar_type()), ot = out_type < 0 ? type : (int)out_type;
  at::Tensor out = rows_like(x, N, scalar_type_of(ot));
  if (M == 0) return pybind11::cast(out);
  const size_t need = mm_mxfp4_gemm_workspace_bytes((int)M, (int)N, (int)K);
  at::Tensor ws;
  if (need) ws = workspace(x, stream, need);
  const int rc = mm_mxfp4_gemm(x.data_ptr(), type, (const uint32_t*)W.data_ptr(),
                               (const uint8_t*)S.data_ptr(), out.data_ptr(), ot, (int)M, (int)N,
                               (int)K, need ? ws.data_ptr() : nullptr, need ? ws.numel() : 0,
                               (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

// The gradient of x for dy [*, N].
pybind11::object mx_gemm_backward(const at::Tensor& dy, const at::Tensor& W, const at::Tensor& S,
                                  int64_t out_type, int64_t stream) {
  const int dev = (int)dy.get_device();
  if (!on_current_device(dev) || !plain_mx(W, S, dev, 2)) return pybind11::none();
  const int64_t N = W.size(0), K = 8 * W.size(1), M = plain_rows(dy, dev, N);
  if (M < 0 || M > INT32_MAX || N > INT32_MAX || N * dy.element_size() % 16 != 0)
    return pybind11::none();
  const int type = type_code(dy.scalar_type()), ot = out_type < 0 ? type : (int)out_type;
  at::Tensor out = rows_like(dy, K, scalar_type_of(ot));
  if (M == 0) return pybind11::cast(out);
  const size_t need = mm_mxfp4_gemm_backward_workspace_bytes((int)M, (int)N, (int)K, type);
  at::Tensor ws;
  if (need) ws = workspace(dy, stream, need);
  const int rc = mm_mxfp4_gemm_backward(dy.data_ptr(), type, (int)N, (const uint32_t*)W.data_ptr(),
                                        (const uint8_t*)S.data_ptr(), out.data_ptr(), ot, (int)M,
                                        (int)N, (int)K, need ? ws.data_ptr() : nullptr,
                                        need ? ws.numel() : 0, (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

pybind11::object mx_quantize(const at::Tensor& x, int64_t stream) {
  const int dev = (int)x.get_device();
  if (!on_current_device(dev) || x.dim() < 1 || x.size(-1) == 0 || x.size(-1) % 32 != 0)
    return pybind11::none();
  const int64_t K = x.size(-1), rows = plain_rows(x, dev, K);
  if (rows < 0 || K > INT32_MAX) return pybind11::none();
  at::Tensor words = rows_like(x, K / 8, at::kInt), scales = rows_like(x, K / 32, at::kByte);
  if (rows == 0) return pybind11::make_tuple(words, scales);
  const int rc = mm_mxfp4_quantize(x.data_ptr(), type_code(x.scalar_type()), rows, (int)K,
                                   (uint32_t*)words.data_ptr(), (uint8_t*)scales.data_ptr(),
                                   (void*)stream);
  if (rc) fail(rc);
  return pybind11::make_tuple(words, scales);
}

pybind11::object mx_dequantize(const at::Tensor& W, const at::Tensor& S, int64_t type,
                               int64_t stream) {
  const int dev = (int)W.get_device();
  if (!on_current_device(dev) || W.dim() < 1 || !plain_mx(W, S, dev, (int)W.dim()))
    return pybind11::none();
  const int64_t K = 8 * W.size(-1);
  if (K > INT32_MAX) return pybind11::none();
  at::Tensor out = rows_like(W, K, scalar_type_of(type));
  const int rc = mm_mxfp4_dequantize((const uint32_t*)W.data_ptr(), (const uint8_t*)S.data_ptr(),
                                     W.numel() / W.size(-1), (int)K, out.data_ptr(), (int)type,
                                     (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

// The experts' block on MXFP4 weights: plain operands, ids and probs [T, k].
pybind11::object mx_moe_mlp(const at::Tensor& x, const at::Tensor& Wgu, const at::Tensor& Sgu,
                            const at::Tensor& Wdn, const at::Tensor& Sdn, const at::Tensor& ids,
                            const at::Tensor& probs, int64_t stream) {
  const int dev = (int)x.get_device();
  if (!on_current_device(dev) || x.dim() != 2 || !plain_mx(Wgu, Sgu, dev, 3) ||
      !plain_mx(Wdn, Sdn, dev, 3) || ids.dim() != 2 || probs.sizes() != ids.sizes() ||
      ids.get_device() != dev || probs.get_device() != dev || !ids.is_contiguous() ||
      !probs.is_contiguous() || probs.scalar_type() != at::kFloat ||
      (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt))
    return pybind11::none();
  const int64_t E = Wgu.size(0), I = 8 * Wdn.size(2), H = 8 * Wgu.size(2);
  const int64_t T = plain_rows(x, dev, H), k = ids.size(1);
  if (T <= 0 || k == 0 || ids.size(0) != T || Wgu.size(1) != 2 * I || Wdn.size(0) != E ||
      Wdn.size(1) != H || std::max({E, I, H, T, T * k}) > INT32_MAX)
    return pybind11::none();
  const int type = type_code(x.scalar_type());
  at::Tensor out = at::empty_like(x);
  const size_t need = mm_moe_mlp_mxfp4_scratch_bytes((int)T, (int)k, (int)E, (int)H, (int)I);
  at::Tensor scratch = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
  const int rc = mm_moe_mlp_mxfp4(
      x.data_ptr(), type, ids.data_ptr(), ids.scalar_type() == at::kLong,
      (const float*)probs.data_ptr(), (int)T, (int)k, (int)E, (int)H, (int)I,
      (const uint32_t*)Wgu.data_ptr(), (const uint8_t*)Sgu.data_ptr(),
      (const uint32_t*)Wdn.data_ptr(), (const uint8_t*)Sdn.data_ptr(), scratch.data_ptr(), need,
      out.data_ptr(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(out);
}

// Routing: logits [*, E] and a bias [E] in plain form, or None.
pybind11::object moe_route(const at::Tensor& logits, int64_t k, bool softmax,
                           const c10::optional<at::Tensor>& bias, int64_t groups, int64_t keep,
                           bool renorm, double scale, int64_t stream) {
  const int dev = (int)logits.get_device();
  const int type = type_code(logits.scalar_type());
  if (!on_current_device(dev) || logits.dim() < 1 || type < 0 || !logits.is_contiguous() ||
      logits.size(-1) == 0)
    return pybind11::none();
  const int64_t E = logits.size(-1), T = logits.numel() / E;
  if (T > INT32_MAX || E > INT32_MAX || k < 0 || k > INT32_MAX || groups < 0 ||
      groups > INT32_MAX || keep < 0 || keep > INT32_MAX ||
      (bias && (bias->dim() != 1 || bias->numel() != E || bias->get_device() != dev ||
                bias->scalar_type() != at::kFloat || !bias->is_contiguous())))
    return pybind11::none();
  at::Tensor w = rows_like(logits, k, at::kFloat), ids = rows_like(logits, k, at::kLong);
  const int rc = mm_moe_route(logits.data_ptr(), type, bias ? (const float*)bias->data_ptr() : nullptr,
                              (int)T, (int)E, (int)k, softmax, (int)groups, (int)keep, renorm,
                              (float)scale, (int64_t*)ids.data_ptr(), (float*)w.data_ptr(),
                              (void*)stream);
  if (rc) fail(rc);
  return pybind11::make_tuple(w, ids);
}

pybind11::object moe_route_backward(const at::Tensor& dw, const at::Tensor& logits,
                                    const at::Tensor& ids, bool softmax, bool renorm, double scale,
                                    int64_t stream) {
  const int dev = (int)logits.get_device();
  const int type = type_code(logits.scalar_type());
  if (!on_current_device(dev) || logits.dim() < 1 || type < 0 || !logits.is_contiguous() ||
      logits.size(-1) == 0 || dw.dim() != logits.dim() || dw.get_device() != dev ||
      ids.get_device() != dev || dw.scalar_type() != at::kFloat || ids.scalar_type() != at::kLong ||
      !dw.is_contiguous() || !ids.is_contiguous() || dw.sizes() != ids.sizes() ||
      dw.sizes().slice(0, dw.dim() - 1) != logits.sizes().slice(0, dw.dim() - 1))
    return pybind11::none();
  const int64_t E = logits.size(-1), T = logits.numel() / E, k = dw.size(-1);
  if (T > INT32_MAX || E > INT32_MAX || k > INT32_MAX) return pybind11::none();
  at::Tensor dl = at::empty_like(logits);
  const int rc = mm_moe_route_backward((const float*)dw.data_ptr(), logits.data_ptr(), type,
                                       (const int64_t*)ids.data_ptr(), (int)T, (int)E, (int)k,
                                       softmax, renorm, (float)scale, dl.data_ptr(), (void*)stream);
  if (rc) fail(rc);
  return pybind11::cast(dl);
}

// Stream id of a leaf's gradient accumulator, or -1 where it has none (yet).
int64_t accumulator_stream(const at::Tensor& leaf) {
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!node) return -1;
  const auto stream = node->stream();
  return stream ? (int64_t)stream->id() : -1;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Per-call binding of libmmfp4's FP4 / INT4 GEMM entry points";
  m.def("gemm", &gemm, "C = A . dequant(B, S[, Z]) on the given stream", pybind11::arg("A"),
        pybind11::arg("B"), pybind11::arg("S"), pybind11::arg("Z"), pybind11::arg("SZ"),
        pybind11::arg("group_size"), pybind11::arg("stream"));
  m.def("qkv", &qkv, "mm_fp4_gemm_multi on plain operands, else None");
  m.def("gate_up", &gate_up, "mm_fp4_gate_up[_rowpacked] on plain operands, else None");
  m.def("rowpacked", &rowpacked, "mm_fp4_gemm_rowpacked on plain operands, else None");
  m.def("linear_backward", &linear_backward, "mm_gemm_backward on plain operands, else None");
  m.def("qkv_backward", &qkv_backward, "mm_gemm_backward over three matrices, else None");
  m.def("gate_up_keep", &gate_up_keep, "mm_fp4_gate_up_keep on plain operands, else None");
  m.def("gate_up_backward", &gate_up_backward,
        "mm_swiglu_grad and mm_gemm_backward on plain operands, else None");
  m.def("lora_add", &lora_add, "mm_lora_add on plain operands, else None");
  m.def("lora_backward", &lora_backward, "mm_lora_backward on plain operands, else None");
  m.def("mx_gemm", &mx_gemm, "mm_mxfp4_gemm on plain operands, else None");
  m.def("mx_gemm_backward", &mx_gemm_backward, "mm_mxfp4_gemm_backward on plain operands, else None");
  m.def("mx_quantize", &mx_quantize, "mm_mxfp4_quantize on a plain operand, else None");
  m.def("mx_dequantize", &mx_dequantize, "mm_mxfp4_dequantize on plain operands, else None");
  m.def("mx_moe_mlp", &mx_moe_mlp, "mm_moe_mlp_mxfp4 on plain operands, else None");
  m.def("moe_route", &moe_route, "mm_moe_route on plain operands, else None");
  m.def("moe_route_backward", &moe_route_backward,
        "mm_moe_route_backward on plain operands, else None");
  m.def("accumulator_stream", &accumulator_stream,
        "stream id of a leaf's gradient accumulator, -1 without one");
  m.def("workspace", &workspace_for,
        "the zero-initialised workspace of (device index, raw stream), at least nbytes",
        pybind11::arg("device"), pybind11::arg("stream"), pybind11::arg("nbytes"));
  m.def("release_workspaces", &release_workspaces, "drop every cached workspace");
}
