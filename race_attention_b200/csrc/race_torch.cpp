// race_torch.cpp -- the 8-bit operators on torch tensors: what race_attention_b200/fp8.py
// and optim.py call.  It allocates results, lays out descriptors, calls the C
// entry points of librace_b200.so on the current stream and holds the two
// autograd functions.  Small calls are bound by the host, and a call costs some
// 5 us here where the same steps through ctypes cost 15 to 30 (and an autograd
// pass 30 us in place of 150 to 270).  Arguments are checked by the Python layer unless
// a check needs the tensors' memory.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "race_b200.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kBlock = 128;
constexpr int64_t kRowsAtOnce = 65535 * kBlock;    // of race_quantize
constexpr auto kF8 = at::kFloat8_e4m3fn;

struct RaceFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int rc) {
  if (rc == RACE_OK) return;
  std::string text = "race_b200 error " + std::to_string(rc) + ": " + race_strerror(rc);
  const char* more = race_last_cuda_error();
  if ((rc == RACE_ERR_UNSUPPORTED || rc == RACE_ERR_CUDA) && more[0] != '\0') text += std::string(": ") + more;
  throw RaceFailure(text);
}

cudaStream_t stream_of(const Tensor& x) {
  return c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
}

int32_t code_of(const Tensor& x) { return x.scalar_type() == at::kFloat ? RACE_F32 : RACE_BF16; }

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// x as [rows, columns] with contiguous columns; x is float32 or bfloat16
Tensor rows_of(const Tensor& x) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  Tensor r = x.dim() == 2 ? x : x.reshape({rows, x.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) r = r.contiguous();
  return r;
}

race_rows_t rr(const Tensor& x) {
  return x.defined() ? race_rows_t{x.data_ptr(), x.stride(0)} : race_rows_t{nullptr, 0};
}

struct Held {
  Tensor codes, scales;
};

// codes of [rows, cols], every row on 16 bytes
Tensor new_codes(int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t pitch = up16(cols);
  Tensor c = at::empty({rows, pitch}, like.options().dtype(kF8));
  return pitch == cols ? c : c.narrow(1, 0, cols);
}
Tensor new_scales(int64_t rows, int64_t cols, const Tensor& like) {
  return at::empty_strided({rows, blocks_of(cols)}, {1, std::max<int64_t>(rows, 1)}, like.options().dtype(at::kFloat));
}

race_blocks_t rb(const Held& h) {
  if (!h.codes.defined()) return race_blocks_t{nullptr, 0, nullptr, 0, 0};
  const int64_t pitch = h.codes.size(0) > 1 ? h.codes.stride(0) : up16(h.codes.size(1));
  return race_blocks_t{h.codes.data_ptr(), pitch, static_cast<float*>(h.scales.data_ptr()), h.scales.stride(0),
                       h.scales.stride(1)};
}

// Autograd's version check has to see what a kernel wrote into a caller's tensor.
void written(const Tensor& x) { x.unsafeGetTensorImpl()->bump_version(); }

enum Mode { kRows = 0, kBoth = 1, kCols = 2 };

std::pair<Held, Held> quantize_rows(const Tensor& x, bool square, int mode) {
  const int64_t r = x.size(0), k = x.size(1);
  Held a, t;
  Tensor s;
  if (square) s = at::empty({blocks_of(r), blocks_of(k)}, x.options().dtype(at::kFloat));
  if (mode != kCols) a = {new_codes(r, k, x), square ? s : new_scales(r, k, x)};
  if (mode != kRows) t = {new_codes(k, r, x), square ? s.t() : new_scales(k, r, x)};
  // A launch takes kRowsAtOnce rows, whole blocks, so that longer tensors go in parts.
  for (int64_t r0 = 0; r0 < r; r0 += kRowsAtOnce) {
    race_rows_t part{static_cast<char*>(x.data_ptr()) + r0 * x.stride(0) * x.element_size(), x.stride(0)};
    race_blocks_t by_rows = rb(a), by_cols = rb(t);
    if (r0 > 0 && mode != kCols) {
      by_rows.codes = static_cast<char*>(by_rows.codes) + r0 * by_rows.ld;
      by_rows.scales += (square ? r0 / kBlock : r0) * by_rows.stride_row;
    }
    if (r0 > 0 && mode != kRows) {
      by_cols.codes = static_cast<char*>(by_cols.codes) + r0;
      by_cols.scales += r0 / kBlock * by_cols.stride_block;
    }
    check(race_quantize(part, code_of(x), std::min(r - r0, kRowsAtOnce), k, square, by_rows, by_cols, stream_of(x)));
  }
  return {a, t};
}

// The operand itself if the copy engine can walk its codes, else a copy that it can.
Held in_place(const Held& h) {
  const Tensor& c = h.codes;
  const int64_t r = c.size(0), k = c.size(1);
  if ((k <= 1 || c.stride(1) == 1) && reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 &&
      (r <= 1 || (c.stride(0) % 16 == 0 && c.stride(0) >= k)))
    return h;
  Tensor n = new_codes(r, k, c);
  n.view(at::kByte).copy_(c.view(at::kByte));
  return {n, h.scales};
}

// The product in `y` ([m, n], any row stride).
void product_into(const Tensor& y, int64_t ld, const Held& a, const Held& b, bool square, bool f32, uint32_t* status) {
  const int64_t m = a.codes.size(0), n = b.codes.size(0), k = a.codes.size(1);
  const race_matmul_desc_t d{f32 ? RACE_F32 : RACE_BF16, square, m, n, k, 0, 0};
  const size_t need = race_scaled_matmul_workspace(&d);
  Tensor ws;
  if (need > 0) ws = at::empty({(int64_t)need}, a.codes.options().dtype(at::kByte));
  check(race_scaled_matmul(&d, rb(a), rb(b), race_rows_t{y.data_ptr(), ld}, status, need > 0 ? ws.data_ptr() : nullptr,
                           need, stream_of(y)));
}

// The product as a tensor of `shape`, whose last axis is n.  Results are allocated
// with their shape: autograd refuses to change a view in place that an autograd
// function has made.
Tensor product(const Held& a, const Held& b, bool square, bool f32, uint32_t* status, at::IntArrayRef shape) {
  const Tensor y = at::empty(shape, a.codes.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  product_into(y, b.codes.size(0), a, b, square, f32, status);
  return y;
}

// x's sizes with n in the place of the last one
std::vector<int64_t> shape_of(const Tensor& x, int64_t n) {
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  return shape;
}

// ------------------------------------------------------------------ entry points

std::tuple<Tensor, Tensor, Tensor, Tensor> quantize(const Tensor& x, bool square, int mode) {
  c10::cuda::CUDAGuard guard(x.device());
  at::NoGradGuard no_grad;
  const auto [a, t] = quantize_rows(rows_of(x), square, mode);
  return {a.codes, a.scales, t.codes, t.scales};
}

Tensor matmul(const Tensor& ac, const Tensor& as, bool a_square, const Tensor& bc, const Tensor& bs, bool b_square,
              bool f32, const Maybe& out, int64_t status) {
  TORCH_CHECK_VALUE(!a_square, "a must have a scale for each row; only b may have square blocks");
  TORCH_CHECK_VALUE(ac.size(1) == bc.size(1), "a ", ac.sizes(), " and b ", bc.sizes(),
                    " must have the same number of columns");
  TORCH_CHECK_VALUE(ac.device() == bc.device(), "a and b must be on the same device");
  if (out.has_value()) {
    const int64_t m = ac.size(0), n = bc.size(0);
    TORCH_CHECK_VALUE(out->dim() == 2 && out->size(0) == m && out->size(1) == n && out->device() == ac.device() &&
                          out->scalar_type() == (f32 ? at::kFloat : at::kBFloat16) &&
                          (n <= 1 || out->stride(1) == 1) && (m <= 1 || out->stride(0) >= n),
                      "out must be a [", m, ", ", n, "] tensor of out_dtype with contiguous columns");
  }
  c10::cuda::CUDAGuard guard(ac.device());
  at::NoGradGuard no_grad;
  auto* word = reinterpret_cast<uint32_t*>(status);
  const Held a = in_place({ac, as}), b = in_place({bc, bs});
  if (!out.has_value()) return product(a, b, b_square, f32, word, {ac.size(0), bc.size(0)});
  product_into(*out, out->stride(0), a, b, b_square, f32, word);
  written(*out);
  return *out;
}

// The gradients are computed outside torch, so they have none of their own.
void once() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "the 8-bit operators have no second derivatives (create_graph=True)");
}

bool has_tangent(const Tensor& x) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(/*level=*/0).defined();
}
// Calls that need no gradient skip the autograd functions, which would refuse a tangent.
void no_tangent(const Tensor& x) {
  TORCH_CHECK(!has_tangent(x), "the 8-bit operators have no forward-mode derivatives");
}

struct Linear : torch::autograd::Function<Linear> {
  // x [..., K]; weight [N, K], or none with its held form (codes, scales and those of its transpose)
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& wc, const Maybe& ws,
                        const Maybe& tc, const Maybe& ts, bool f32, bool need_x, bool need_w, int64_t status) {
    const Tensor x2 = rows_of(x), none;
    const auto [xr, xt] = quantize_rows(x2, false, need_w ? kBoth : kRows);
    Held w{wc.value_or(none), ws.value_or(none)}, t{tc.value_or(none), ts.value_or(none)};
    if (weight.has_value()) std::tie(w, t) = quantize_rows(rows_of(*weight), true, need_x ? kBoth : kRows);
    const Tensor y = product(xr, in_place(w), true, f32, reinterpret_cast<uint32_t*>(status),
                             shape_of(x, w.codes.size(0)));
    if (need_x || need_w) {
      ctx->save_for_backward({need_w ? xt.codes : Tensor(), need_w ? xt.scales : Tensor(),
                              need_x ? t.codes : Tensor(), need_x ? t.scales : Tensor()});
      // status word, types and needs, then x's sizes
      std::vector<int64_t> meta{status, x.scalar_type() == at::kFloat,
                                weight.has_value() && weight->scalar_type() == at::kFloat, need_x, need_w};
      meta.insert(meta.end(), x.sizes().begin(), x.sizes().end());
      ctx->saved_data["meta"] = meta;
    }
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> meta = ctx->saved_data["meta"].toIntVector();
    auto* status = reinterpret_cast<uint32_t*>(meta[0]);
    const bool need_x = meta[3] && ctx->needs_input_grad(0), need_w = meta[4] && ctx->needs_input_grad(1);
    Tensor dx, dw;
    if (grads[0].defined() && (need_x || need_w)) {
      c10::cuda::CUDAGuard guard(grads[0].device());
      const auto [r, c] = quantize_rows(rows_of(grads[0]), false, need_x ? need_w ? kBoth : kRows : kCols);
      if (need_x)
        dx = product(r, in_place({saved[2], saved[3]}), true, meta[1] != 0, status, at::IntArrayRef(meta).slice(5));
      if (need_w)
        dw = product(c, {saved[0], saved[1]}, false, meta[2] != 0, status, {c.codes.size(0), saved[0].size(0)});
    }
    return {dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Maybe& weight, const Maybe& wc, const Maybe& ws, const Maybe& tc, const Maybe& ts,
              bool f32, int64_t status) {
  no_tangent(x);
  if (weight.has_value()) no_tangent(*weight);
  c10::cuda::CUDAGuard guard(x.device());
  const bool grad = at::GradMode::is_enabled(), need_x = grad && x.requires_grad();
  const bool need_w = grad && weight.has_value() && weight->requires_grad();
  if (need_x || need_w) return Linear::apply(x, weight, wc, ws, tc, ts, f32, need_x, need_w, status);
  at::NoGradGuard no_grad;
  const Held w = weight.has_value() ? quantize_rows(rows_of(*weight), true, kRows).first : Held{*wc, *ws};
  return product(quantize_rows(rows_of(x), false, kRows).first, in_place(w), true, f32,
                 reinterpret_cast<uint32_t*>(status), shape_of(x, w.codes.size(0)));
}

struct NormOut {
  Tensor y, h, rstd;
  Held y8;
};

// x and residual as rows; y and h get `shape` (see product).
NormOut norm_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, bool quant,
                     bool want_rstd, at::IntArrayRef shape) {
  const int64_t r = x.size(0), k = x.size(1);
  const auto whole = [k](const Tensor& t) { return race_rows_t{t.defined() ? t.data_ptr() : nullptr, k}; };
  NormOut o;
  if (residual.defined()) o.h = at::empty(shape, x.options());
  if (quant)
    o.y8 = {new_codes(r, k, x), new_scales(r, k, x)};
  else
    o.y = at::empty(shape, x.options());
  if (want_rstd) o.rstd = at::empty({r}, x.options().dtype(at::kFloat));
  const race_norm_desc_t d{code_of(x), code_of(weight), r, k, (float)eps};
  check(race_rms_norm(&d, rr(x), rr(residual), weight.data_ptr(), whole(o.y), rb(o.y8), whole(o.h),
                      want_rstd ? static_cast<float*>(o.rstd.data_ptr()) : nullptr, stream_of(x)));
  return o;
}

struct Norm : torch::autograd::Function<Norm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& residual,
                               double eps) {
    ctx->set_materialize_grads(false);
    const Tensor x2 = rows_of(x), w = weight.contiguous();
    const NormOut o = norm_forward(x2, w, residual.has_value() ? rows_of(*residual) : Tensor(), eps, false, true,
                                   x.sizes());
    ctx->save_for_backward({o.h.defined() ? o.h : x2, w, o.rstd});
    variable_list out{o.y};
    if (o.h.defined()) out.push_back(o.h);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const variable_list saved = ctx->get_saved_variables();
    const Tensor h = rows_of(saved[0]), &w = saved[1], &rstd = saved[2];
    const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy.defined())   // y was not used: the norm passes dh through
      return {dh, dh.defined() ? at::zeros_like(w) : Tensor(), dh, Tensor()};
    c10::cuda::CUDAGuard guard(h.device());
    const Tensor dx = at::empty(dy.sizes(), h.options()), dw = at::empty_like(w);
    const race_norm_desc_t d{code_of(h), code_of(w), h.size(0), h.size(1), 0.f};   // rstd has eps in it
    const size_t need = race_rms_norm_workspace(&d);
    const Tensor ws = at::empty({(int64_t)std::max<size_t>(need, 16)}, h.options().dtype(at::kByte));
    check(race_rms_norm_backward(&d, rr(rows_of(dy)), dh.defined() ? rr(rows_of(dh)) : rr(dh), rr(h), w.data_ptr(),
                                 static_cast<const float*>(rstd.data_ptr()), race_rows_t{dx.data_ptr(), h.size(1)},
                                 dw.data_ptr(), ws.data_ptr(), (size_t)ws.numel(), stream_of(h)));
    return {dx, dw, grads.size() > 1 ? dx : Tensor(), Tensor()};
  }
};

// (y or codes, scales, h), the unused ones undefined
std::tuple<Tensor, Tensor, Tensor> norm(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps,
                                        bool quant, bool grad) {
  no_tangent(x);
  no_tangent(weight);
  if (residual.has_value()) no_tangent(*residual);
  c10::cuda::CUDAGuard guard(x.device());
  if (grad) {
    const variable_list out = Norm::apply(x, weight, residual, eps);
    return {out[0], Tensor(), out.size() > 1 ? out[1] : Tensor()};
  }
  at::NoGradGuard no_grad;
  const NormOut o = norm_forward(rows_of(x), weight.contiguous(), residual.has_value() ? rows_of(*residual) : Tensor(),
                                 eps, quant, false, x.sizes());
  if (quant) return {o.y8.codes, o.y8.scales, o.h};
  return {o.y, Tensor(), o.h};
}

// One step of a parameter group.  first[i]: where parameter i's states begin;
// steps: int32, on the host, counted up for the parameters that have a gradient.
void adamw(const std::vector<Tensor>& params, const std::vector<int64_t>& first, const std::vector<int64_t>& sizes,
           const Tensor& steps, const Tensor& m, const Tensor& v, const Maybe& ms,
           const Maybe& vs, double lr, double b1, double b2, double eps, double decay, int64_t seed,
           int64_t bits) {
  c10::cuda::CUDAGuard guard(m.device());
  at::NoGradGuard no_grad;
  std::vector<race_adamw_tensor_t> table;
  std::vector<size_t> moved;
  std::vector<Tensor> kept;
  table.reserve(params.size());
  moved.reserve(params.size());
  int32_t* step = steps.data_ptr<int32_t>();
  const int64_t size = bits == 8 ? 1 : 4;
  char *mp = static_cast<char*>(m.data_ptr()), *vp = static_cast<char*>(v.data_ptr());
  float *msp = ms.has_value() ? ms->data_ptr<float>() : nullptr, *vsp = vs.has_value() ? vs->data_ptr<float>() : nullptr;
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor& p = params[i];
    Tensor g = p.grad();
    if (!g.defined()) continue;
    const auto t = p.scalar_type();
    TORCH_CHECK_VALUE(g.scalar_type() == t && g.layout() == at::kStrided && g.device() == p.device(),
                      "gradients must be dense, on their parameter's device and of its type");
    TORCH_CHECK_VALUE(p.is_contiguous() && p.numel() == sizes[i] && g.numel() == sizes[i] && p.device() == m.device() &&
                          (t == at::kFloat || t == at::kBFloat16),
                      "a parameter changed its size, layout, type or device since the optimizer was built");
    if (!g.is_contiguous()) {
      g = g.contiguous();
      kept.push_back(g);
    }
    const int64_t at = first[i];
    table.push_back({p.data_ptr(), g.data_ptr(), mp + at * size, vp + at * size, msp ? msp + at / kBlock : nullptr,
                     vsp ? vsp + at / kBlock : nullptr, sizes[i], (uint64_t)at, t == at::kFloat ? RACE_F32 : RACE_BF16,
                     step[i]});
    moved.push_back(i);
  }
  const race_adamw_desc_t d{lr, b1, b2, eps, decay, (uint32_t)seed, (int32_t)bits};
  check(race_adamw(&d, table.data(), (int64_t)table.size(), stream_of(m)));
  for (const size_t i : moved) {
    ++step[i];
    written(params[i]);
  }
}

}  // namespace

PYBIND11_MODULE(_race_torch, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const RaceFailure& e) {
      const py::object type = py::module_::import("race_attention_b200._lib").attr("RaceError");
      PyErr_SetString(type.ptr(), e.what());
    }
  });
  m.def("quantize", &quantize);
  m.def("matmul", &matmul);
  m.def("linear", &linear);
  m.def("norm", &norm);
  m.def("adamw", &adamw);
  m.def("has_tangent", &has_tangent);
}
