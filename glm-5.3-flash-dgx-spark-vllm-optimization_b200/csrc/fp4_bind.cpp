// Python bindings of the 4-bit floating-point operators: argument checks, dispatch by row count, launches on the current
// stream of the tensors' device.  Temporaries come from the caching allocator inside the call, so calls on different
// streams, and captured graphs, never share one.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "launchers.h"

namespace {

using at::Tensor;
using OptT = c10::optional<Tensor>;

constexpr int64_t kTileRows = 128, kTileK = 256, kTileBytes = 16384;
constexpr int64_t kFourRows = 16;      // rows above which act4 quantises the activations
constexpr int64_t kFewRows = 96;       // rows up to which exact activations are expanded into 4-bit terms (24576 x 4096: 96 rows
                                       // 48 us, 55 widened; 112 rows 67, 56.  4096 x 4096: 96 rows 15.9, 15.8; 112 rows 18.0,
                                       // 16.4.  A 4096 x 12288 weight would gain from 64 rows on)
constexpr int64_t kFour = 128;         // rows up to which 4-bit activations go through the small-M kernel (24576 x 4096: 100 rows
                                       // 28.8 us, 36.3 on the GEMM; 200 rows 42.6, 35.5)

void ok(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, "glm53 kernel ", what, " failed: ", cudaGetErrorString(e));
}
cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }
// numbers in messages are formatted here: streaming one into a string stream crashes in the process when the extension is
// built with a C++ library that differs from the one torch loaded
std::string num(int64_t v) { return std::to_string(v); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int64_t n_tiles(int64_t rows, int64_t k) { return ((rows + kTileRows - 1) / kTileRows) * ((k + kTileK - 1) / kTileK); }
int64_t scale_bytes(bool nv) { return kTileRows * (kTileK / (nv ? 16 : 32)); }

// a 4-bit matrix: its arrays and shape, checked once when it is made.  Matrices made here keep their three arrays in one
// buffer; the views that Python sees are made when asked for
struct Matrix4 {
  Tensor parts[3];                     // codes, scales, row scale; or the one buffer in parts[0]
  bool whole = false;
  int64_t rows = 0, k = 0;
  bool nv = false;
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  float* row_scale = nullptr;

  static void check_shape(int64_t rows, int64_t k, bool nv) {
    const int64_t block = nv ? 16 : 32;
    TORCH_CHECK(rows >= 1 && k >= block && k % block == 0, "Matrix4: rows >= 1 and K a multiple of ", num(block), ", got [",
                num(rows), ", ", num(k), "]");
    TORCH_CHECK(rows < (int64_t)1 << 31 && k < (int64_t)1 << 31, "Matrix4: at most 2^31 - 1 rows and columns");
  }
  Matrix4(int64_t rows_, int64_t k_, bool nv_, const Tensor& like) : whole(true), rows(rows_), k(k_), nv(nv_) {
    check_shape(rows, k, nv);
    const int64_t c = n_tiles(rows, k) * kTileBytes, s = n_tiles(rows, k) * scale_bytes(nv);
    parts[0] = at::empty({c + s + (nv ? 4 * rows : 0)}, like.options().dtype(at::kByte));
    codes = parts[0].data_ptr<uint8_t>();
    scales = codes + c;
    if (nv) row_scale = reinterpret_cast<float*>(scales + s);
  }
  Matrix4(const Tensor& c, const Tensor& s, const OptT& r, int64_t rows_, int64_t k_, bool nv_)
      : rows(rows_), k(k_), nv(nv_) {
    check_shape(rows, k, nv);
    const int64_t t = n_tiles(rows, k);
    TORCH_CHECK(c.is_cuda() && c.scalar_type() == at::kByte && c.is_contiguous() && c.numel() == t * kTileBytes &&
                    aligned16(c.data_ptr()),
                "Matrix4: codes must be ", num(t * kTileBytes), " contiguous, 16-byte aligned uint8 on a CUDA device");
    TORCH_CHECK(s.device() == c.device() && s.scalar_type() == at::kByte && s.is_contiguous() &&
                    s.numel() == t * scale_bytes(nv) && aligned16(s.data_ptr()),
                "Matrix4: scales must be ", num(t * scale_bytes(nv)),
                " contiguous, 16-byte aligned uint8 on the codes' device");
    TORCH_CHECK(nv == r.has_value(), "Matrix4: nvfp4 has a row scale, mxfp4 none");
    if (nv) {
      TORCH_CHECK(r->device() == c.device() && r->scalar_type() == at::kFloat && r->is_contiguous() &&
                      r->numel() == rows && aligned16(r->data_ptr()),
                  "Matrix4: row_scale must be fp32 [rows], contiguous, 16-byte aligned, on the codes' device");
      parts[2] = *r;
      row_scale = r->data_ptr<float>();
    }
    parts[0] = c;
    parts[1] = s;
    codes = c.data_ptr<uint8_t>();
    scales = s.data_ptr<uint8_t>();
  }
  at::Device device() const { return parts[0].device(); }
  Tensor codes_view() const { return whole ? parts[0].narrow(0, 0, n_tiles(rows, k) * kTileBytes) : parts[0]; }
  Tensor scales_view() const {
    const int64_t t = n_tiles(rows, k);
    return whole ? parts[0].narrow(0, t * kTileBytes, t * scale_bytes(nv)) : parts[1];
  }
  OptT row_scale_view() const {
    if (!nv) return c10::nullopt;
    const int64_t t = n_tiles(rows, k);
    return whole ? parts[0].narrow(0, t * (kTileBytes + scale_bytes(nv)), 4 * rows).view(at::kFloat) : parts[2];
  }
};

void check_x(const Tensor& x, const char* op) {
  TORCH_CHECK(x.is_cuda(), op, ": x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1), op, ": x must be [rows, K] with unit inner stride");
  TORCH_CHECK(x.size(0) < (int64_t)1 << 31, op, ": at most 2^31 - 1 rows");
}

Matrix4 quantize(const Tensor& x, bool nv) {
  check_x(x, "quantize4");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "quantize4: x must be bf16 or f16");
  const c10::cuda::CUDAGuard guard(x.device());
  Matrix4 m(x.size(0), x.size(1), nv, x);
  Fp4QuantArgs a{};
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  a.R = m.rows;
  a.K = m.k;
  a.nv = nv;
  a.f16 = x.scalar_type() == at::kHalf;
  a.vec = aligned16(a.x) && a.ldx % 8 == 0;
  a.codes = m.codes;
  a.scales = m.scales;
  a.row_scale = m.row_scale;
  ok(g53_fp4_quantize(a, stream()), "fp4_quantize");
  return m;
}

void dequant(const Matrix4& m, const Tensor& y) {
  Fp4DequantArgs a{};
  a.codes = m.codes;
  a.scales = m.scales;
  a.row_scale = m.row_scale;
  a.R = m.rows;
  a.K = m.k;
  a.nv = m.nv;
  a.out = y.scalar_type() == at::kBFloat16 ? 0 : y.scalar_type() == at::kHalf ? 1 : 2;
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.vec = aligned16(a.y) && (a.ldy * y.element_size()) % 16 == 0;
  ok(g53_fp4_dequant(a, stream()), "fp4_dequant");
}

Tensor dequantize(const Matrix4& m, const OptT& out, at::ScalarType dtype) {
  const c10::cuda::CUDAGuard guard(m.device());
  TORCH_CHECK(out.has_value() || dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat,
              "dequantize4: the output must be bf16, f16 or fp32");
  const Tensor y = out.has_value() ? *out : at::empty({m.rows, m.k}, m.parts[0].options().dtype(dtype));
  TORCH_CHECK(y.device() == m.device(), "dequantize4: the output must be on the matrix's device");
  TORCH_CHECK(y.scalar_type() == at::kBFloat16 || y.scalar_type() == at::kHalf || y.scalar_type() == at::kFloat,
              "dequantize4: the output must be bf16, f16 or fp32");
  TORCH_CHECK(y.dim() == 2 && y.size(0) == m.rows && y.size(1) == m.k && y.stride(1) == 1 &&
                  (m.rows == 1 || y.stride(0) >= m.k),
              "dequantize4: the output must be [", num(m.rows), ", ", num(m.k), "], rows contiguous and apart");
  dequant(m, y);
  return y;
}

void check_xy(const Tensor& x, const Matrix4& w, const Tensor& y, int64_t n, int64_t mode, const char* op) {
  check_x(x, op);
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, op, ": x must be bf16");
  TORCH_CHECK(x.device() == w.device() && y.device() == x.device(), op, ": x, y and the weights must be on one device");
  TORCH_CHECK(x.size(1) == w.k, op, ": K mismatch: x ", num(x.size(1)), ", weights ", num(w.k));
  TORCH_CHECK(mode == GEMV_BF16 || mode == GEMV_F32 || mode == GEMV_F32_ACC, op, ": mode must be GEMV_BF16, GEMV_F32 or "
              "GEMV_F32_ACC");
  TORCH_CHECK(y.scalar_type() == (mode == GEMV_BF16 ? at::kBFloat16 : at::kFloat), op,
              ": y must be bf16 (GEMV_BF16) or fp32 (the other modes)");
  TORCH_CHECK(y.dim() == 2 && y.size(0) == x.size(0) && y.size(1) == n && (y.stride(1) == 1 || n == 1) &&
                  (y.size(0) <= 1 || y.stride(0) >= n),
              op, ": y must be [", num(x.size(0)), ", ", num(n), "], rows contiguous and apart");
}

// small-M product: the arguments that do not depend on the form of x
Fp4SkinnyArgs skinny_args(int64_t M, const Matrix4& w, const Tensor& y, int64_t width, int64_t mode, double limit) {
  Fp4SkinnyArgs a{};
  a.codes = w.codes;
  a.scales = w.scales;
  a.row_scale = w.row_scale;
  a.nv = w.nv;
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.M = (int)M;
  a.N = (int)w.rows;
  a.K = (int)w.k;
  a.width = (int)width;
  a.mode = (int)mode;
  a.limit = (float)limit;
  return a;
}

// exact activations, few rows: expanded into 4-bit terms, by the product itself or in a launch of their own
void skinny(const Tensor& x, const Matrix4& w, const Tensor& y, int64_t width, int64_t mode, double limit) {
  Fp4SkinnyArgs a = skinny_args(x.size(0), w, y, width, mode, limit);
  const __nv_bfloat16* rows = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  const int vec = aligned16(rows) && x.stride(0) % 8 == 0;
  Tensor buf;
  if (g53_fp4_expand_inline(a.M, a.N, a.K, a.nv, mode == GEMV_SWIGLU)) {
    a.x = rows;
    a.ldx = x.stride(0);
    a.xvec = vec;
  } else {
    // whole groups of 256 image rows: the product fetches them
    const int64_t tiles = n_tiles((x.size(0) * g53_fp4_terms() + 255) / 256 * 256, w.k);
    buf = at::empty({tiles * (kTileBytes + scale_bytes(w.nv)) + a.M * 4}, x.options().dtype(at::kByte));
    uint8_t* b = buf.data_ptr<uint8_t>();
    Fp4ExpandArgs e{};
    e.x = rows;
    e.ldx = x.stride(0);
    e.M = a.M;
    e.K = a.K;
    e.nv = a.nv;
    e.vec = vec;
    a.x_codes = e.codes = b;
    a.x_scales = e.scales = b + tiles * kTileBytes;
    a.x_factor = e.factor = reinterpret_cast<float*>(b + tiles * (kTileBytes + scale_bytes(w.nv)));
    a.terms = g53_fp4_terms();
    ok(g53_fp4_expand(e, stream()), "fp4_expand");
  }
  ok(g53_fp4_skinny(a, stream()), "fp4_skinny");
}

// 4-bit activations, few rows, with their row scales, or (null: x's own are not set, or there are none) one for all rows
void skinny4(const Matrix4& x, const float* row_scale, float one, const Matrix4& w, const Tensor& y, int64_t mode) {
  Fp4SkinnyArgs a = skinny_args(x.rows, w, y, 0, mode, 0.0);
  a.x_codes = x.codes;
  a.x_scales = x.scales;
  a.x_factor = row_scale;
  a.x_const = one;
  a.terms = 1;
  ok(g53_fp4_skinny(a, stream()), "fp4_skinny");
}

// exact activations, more rows: the weights widened inside the product
void exact(const Tensor& x, const Matrix4& w, const Tensor& y, int64_t width, int64_t mode, double limit) {
  // rows that the tensor map cannot describe (unaligned, or broadcast) are copied
  const bool direct = aligned16(x.data_ptr()) && x.stride(0) % 8 == 0 && x.stride(0) >= w.k;
  const Tensor xx = direct ? x : x.clone(at::MemoryFormat::Contiguous);
  Fp4ExactArgs a{};
  a.x = reinterpret_cast<const __nv_bfloat16*>(xx.data_ptr());
  a.ldx = xx.stride(0);
  a.codes = w.codes;
  a.scales = w.scales;
  a.row_scale = w.row_scale;
  a.nv = w.nv;
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.M = (int)x.size(0);
  a.N = (int)w.rows;
  a.K = (int)w.k;
  a.width = (int)width;
  a.mode = (int)mode;
  a.limit = (float)limit;
  ok(g53_fp4_exact(a, stream()), "fp4_exact");
}

Fp4GemmArgs gemm_args(const Matrix4& a, const Matrix4& w, int64_t mode) {
  Fp4GemmArgs p{};
  p.a_codes = a.codes;
  p.a_scales = a.scales;
  p.a_row = a.row_scale;
  p.a_const = 1.f;
  p.b_codes = w.codes;
  p.b_scales = w.scales;
  p.b_row = w.row_scale;
  p.nv = w.nv;
  p.M = (int)a.rows;
  p.N = (int)w.rows;
  p.K = (int)w.k;
  p.mode = (int)mode;
  return p;
}

void linear(const Tensor& x, const Matrix4& w, const Tensor& y, int64_t mode, bool act4) {
  check_xy(x, w, y, w.rows, mode, "linear4");
  const int64_t M = x.size(0);
  if (M == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  if (M > kFourRows && act4) {
    const Matrix4 a = quantize(x, w.nv);
    if (M <= kFour) {
      skinny4(a, a.row_scale, 1.f, w, y, mode);
      return;
    }
    Fp4GemmArgs p = gemm_args(a, w, mode);
    p.y = y.data_ptr();
    p.ldy = y.stride(0);
    ok(g53_fp4_gemm(p, stream()), "fp4_gemm");
  } else if (M > kFewRows) {
    exact(x, w, y, 0, mode, 0.0);
  } else {
    skinny(x, w, y, 0, mode, 0.0);
  }
}

// smallest k with bound <= 448 * 6 * 2^k (fp4.cuh: nv_row_exp)
int row_exp(float bound) {
  uint32_t b;
  std::memcpy(&b, &bound, 4);
  const int k = (int)(b >> 23) - 127 - 11 + ((b & 0x7fffffu) > 0x280000u ? 1 : 0);
  return std::max(k, -100);
}

void mlp(const Tensor& x, const Matrix4& gu, const Matrix4& down, const Tensor& y, double limit, int64_t mode, bool act4) {
  const int64_t W = down.k;
  TORCH_CHECK(gu.nv == down.nv && gu.device() == down.device(), "mlp4: both matrices in one format, on one device");
  TORCH_CHECK(W % 32 == 0 && gu.rows == (W + 63) / 64 * 128, "mlp4: the gate/up image must have ", num((W + 63) / 64 * 128),
              " rows for a width of ", num(W), " (a multiple of 32)");
  check_xy(x, gu, y, down.rows, mode, "mlp4");
  TORCH_CHECK(limit > 0, "mlp4: limit must be positive (infinity: no clamp)");
  const int64_t M = x.size(0);
  // bounds |h|: |u| <= limit, and silu(min(g, limit)) lies in [-0.27847, limit]
  const float h_max = std::max((float)limit, 0.2785f) * (float)limit;
  const bool four = act4 && M > kFourRows;
  TORCH_CHECK(!four || !gu.nv || (std::isfinite(h_max) && h_max >= 1e-30f),
              "mlp4: 4-bit nvfp4 activations need a finite limit (their row scale comes from it)");
  if (M == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  if (four) {
    const Matrix4 a = quantize(x, gu.nv);
    const Matrix4 h(M, W, gu.nv, x);
    Fp4GemmArgs p = gemm_args(a, gu, GEMV_SWIGLU);
    p.limit = (float)limit;
    p.width = (int)W;
    p.out_codes = h.codes;
    p.out_scales = h.scales;
    p.h_exp = gu.nv ? row_exp(h_max) : 0;
    ok(g53_fp4_gemm(p, stream()), "fp4_gemm");
    const float factor = gu.nv ? std::ldexp(1.f, p.h_exp) : 1.f;
    if (M <= kFour) {
      skinny4(h, nullptr, factor, down, y, mode);
      return;
    }
    Fp4GemmArgs d = gemm_args(h, down, mode);
    d.a_row = nullptr;
    d.a_const = factor;
    d.y = y.data_ptr();
    d.ldy = y.stride(0);
    ok(g53_fp4_gemm(d, stream()), "fp4_gemm");
    return;
  }
  const Tensor h = at::empty({M, W}, x.options());
  if (M > kFewRows) {
    exact(x, gu, h, W, GEMV_SWIGLU, limit);
    exact(h, down, y, 0, mode, 0.0);
    return;
  }
  skinny(x, gu, h, W, GEMV_SWIGLU, limit);
  skinny(h, down, y, 0, mode, 0.0);
}

int64_t error(int64_t device) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  cudaError_t (*const words[])(int*, cudaStream_t) = {g53_fp4_skinny_error, g53_fp4_gemm_error, g53_fp4_exact_error};
  // pinned, so the three copies cost one wait
  const Tensor host = at::empty({3}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
  int* code = host.data_ptr<int>();
  for (int i = 0; i < 3; ++i) ok(words[i](code + i, stream()), "fp4_error");
  ok(cudaStreamSynchronize(stream()), "fp4_error");
  int64_t first = 0;
  for (int i = 0; i < 3; ++i) {
    if (!code[i]) continue;
    if (!first) first = code[i];
    ok(words[i](nullptr, stream()), "fp4_error");
  }
  return first;
}

}  // namespace

void register_fp4(pybind11::module& m) {
  namespace py = pybind11;
  py::class_<Matrix4>(m, "Matrix4")
      .def(py::init<const Tensor&, const Tensor&, const OptT&, int64_t, int64_t, bool>())
      .def_property_readonly("codes", &Matrix4::codes_view)
      .def_property_readonly("scales", &Matrix4::scales_view)
      .def_property_readonly("row_scale", &Matrix4::row_scale_view)
      .def_readonly("rows", &Matrix4::rows)
      .def_readonly("k", &Matrix4::k)
      .def_readonly("nv", &Matrix4::nv);
  m.def("fp4_quantize", &quantize);
  m.def("fp4_dequantize", &dequantize);
  m.def("fp4_linear", &linear);
  m.def("fp4_mlp", &mlp);
  m.def("fp4_error", &error);
}
