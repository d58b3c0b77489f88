// Bindings and autograd functions of the rotary positions, the gated feed-forward block and the 8-bit products.  As in bindings.cpp, what
// would otherwise become a device fault is checked here, and the functions are C++ so that a backward pass does not wait for the interpreter.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "bindings.h"
#include "fp8.h"
#include "gated_mlp.h"
#include "himuon.h"
#include "rotary.h"

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

#define HM_CHECK(cond, msg) TORCH_CHECK(cond, "himuon: ", msg)

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

void check_once(const char* op) {
  TORCH_CHECK(!c10::GradMode::is_enabled(), "himuon_b200.ops.", op, ": its gradient cannot be differentiated again (create_graph=True)");
}
bool any_grad(std::initializer_list<const at::Tensor*> all) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : all)
    if (t->requires_grad()) return true;
  return false;
}

// ------------------------------------------------------------------------------------------------ rotary positions
// `positions`: one for each row, or none: row % seq_len.
at::Tensor rotate(const at::Tensor& x, const c10::optional<at::Tensor>& positions, const at::Tensor& turns, int64_t seq_len, int64_t heads, int64_t rotary_dim,
                  bool interleaved, double cos_factor, double sin_factor) {
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  HM_CHECK(x.is_cuda() && (bf16 || x.scalar_type() == at::kFloat) && x.dim() == 2 && heads > 0 && heads < (1LL << 30) && x.size(1) % heads == 0 && x.size(1) < (1LL << 30),
           "rotary: (rows, heads * head_dim) of bf16 or fp32 expected");
  HM_CHECK(x.stride(1) == 1 || x.size(1) <= 1, "rotary: unit inner stride expected");
  const int64_t hd = x.size(1) / heads;
  HM_CHECK(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= hd, "rotary: an even part of the head expected");
  HM_CHECK(turns.device() == x.device() && turns.scalar_type() == at::kLong && turns.is_contiguous() && turns.numel() == rotary_dim / 2, "rotary: one int64 frequency for each pair");
  if (positions.has_value()) {
    HM_CHECK(positions->device() == x.device() && positions->scalar_type() == at::kLong && positions->is_contiguous() && positions->numel() == x.size(0), "rotary: one int64 position for each row");
  } else {
    HM_CHECK(seq_len > 0, "rotary: sequences of one token or more");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (!x.numel()) return y;
  himuon::RotaryArgs a;
  a.x = x.data_ptr(); a.y = y.data_ptr();
  a.positions = positions.has_value() ? reinterpret_cast<const long long*>(positions->data_ptr<int64_t>()) : nullptr;
  a.turns = reinterpret_cast<const unsigned long long*>(turns.data_ptr<int64_t>());
  a.rows = x.size(0); a.ld_x = x.stride(0); a.ld_y = x.size(1); a.seq_len = seq_len;
  a.heads = static_cast<int>(heads); a.head_dim = static_cast<int>(hd); a.rotary_dim = static_cast<int>(rotary_dim);
  a.interleaved = interleaved; a.fp32 = !bf16;
  a.cos_factor = static_cast<float>(cos_factor); a.sin_factor = static_cast<float>(sin_factor);
  himuon::rotary(a, cur_stream());
  autograd_launched += 1;
  return y;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& positions, const at::Tensor& turns, int64_t seq_len, int64_t heads,
                            int64_t rotary_dim, bool interleaved, double cos_factor, double sin_factor) {
    if (positions.has_value()) ctx->save_for_backward({turns, *positions});
    else ctx->save_for_backward({turns});
    ctx->saved_data["sizes"] = std::vector<int64_t>{seq_len, heads, rotary_dim, interleaved};
    ctx->saved_data["factors"] = std::vector<double>{cos_factor, sin_factor};
    return rotate(x, positions, turns, seq_len, heads, rotary_dim, interleaved, cos_factor, sin_factor);
  }

  // The transposed rotation, which is one itself: differentiable as often as anyone likes.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    at::Tensor dy = grads[0];
    if (dy.stride(1) != 1 && dy.size(1) > 1) dy = dy.contiguous();
    variable_list out(9);
    const c10::optional<at::Tensor> positions = saved.size() > 1 ? c10::optional<at::Tensor>(saved[1]) : c10::nullopt;
    const std::vector<int64_t> n = ctx->saved_data["sizes"].toIntVector();
    const std::vector<double> f = ctx->saved_data["factors"].toDoubleVector();
    out[0] = c10::GradMode::is_enabled() ? apply(dy, positions, saved[0], n[0], n[1], n[2], n[3] != 0, f[0], -f[1])
                                         : rotate(dy, positions, saved[0], n[0], n[1], n[2], n[3] != 0, f[0], -f[1]);
    return out;
  }
};

// ------------------------------------------------------------------------------------------------ gated feed-forward block
void check_rows(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like, int64_t rows, int64_t cols) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1 &&
                  t.stride(0) % 8 == 0 && (rows <= 1 || t.stride(0) >= cols) && aligned16(t),
              std::string("himuon: ") + op + ": " + name + " must be (" + std::to_string(rows) + ", " + std::to_string(cols) + ") bf16, its rows on 16-byte boundaries with unit inner stride");
}
// The same, for a gradient: copied where it lies otherwise.
at::Tensor with_rows(const at::Tensor& t) {
  if (t.stride(1) == 1 && t.stride(0) % 8 == 0 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) && aligned16(t)) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

struct GatedSizes { int64_t rows, hidden, inter; };
GatedSizes gated_sizes(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation) {
  HM_CHECK(x.dim() == 2 && wg.dim() == 2, "gated_mlp: (rows, hidden) and (inter, hidden) expected");
  const GatedSizes n{x.size(0), x.size(1), wg.size(0)};
  HM_CHECK(n.rows < (1LL << 30) && n.hidden > 0 && n.hidden % 8 == 0 && n.hidden < (1LL << 28) && n.inter > 0 && n.inter % 8 == 0 && n.inter < (1LL << 28),
           "gated_mlp: sizes of multiples of 8 expected");
  HM_CHECK(activation >= himuon::kSilu && activation <= himuon::kRelu, "gated_mlp: unknown activation");
  check_rows("gated_mlp", "x", x, x, n.rows, n.hidden);
  check_rows("gated_mlp", "w_gate", wg, x, n.inter, n.hidden);
  check_rows("gated_mlp", "w_up", wu, x, n.inter, n.hidden);
  check_rows("gated_mlp", "w_down", wd, x, n.hidden, n.inter);
  return n;
}
// y; with `kept`, h and what is kept of g | u are left there.
struct GatedKept { at::Tensor h, gu, gu_low; };
at::Tensor gated_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation, GatedKept* kept) {
  const GatedSizes n = gated_sizes(x, wg, wu, wd, activation);
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor h = at::empty({n.rows, n.inter}, x.options()), y = at::empty({n.rows, n.hidden}, x.options());
  if (kept) *kept = {h, at::empty({n.rows, 2 * n.inter}, x.options()), at::empty({n.rows, 2 * himuon::gated_low(static_cast<int>(n.inter))}, x.options().dtype(at::kByte))};
  if (!n.rows) return y;
  himuon::GatedUpArgs a;
  a.x = x.data_ptr(); a.wg = wg.data_ptr(); a.wu = wu.data_ptr();
  a.h = h.data_ptr(); a.gu = kept ? kept->gu.data_ptr() : nullptr; a.gu_low = kept ? kept->gu_low.data_ptr() : nullptr;
  a.ld_x = x.stride(0); a.ld_wg = wg.stride(0); a.ld_wu = wu.stride(0);
  a.rows = static_cast<int>(n.rows); a.hidden = static_cast<int>(n.hidden); a.inter = static_cast<int>(n.inter); a.activation = static_cast<int>(activation);
  if (n.rows <= himuon::kFewProductRows) {
    himuon::few_rows_gated_up(a, cur_stream());
    himuon::few_rows_product(h.data_ptr(), n.inter, wd.data_ptr(), wd.stride(0), y.data_ptr(), a.rows, a.inter, a.hidden, cur_stream());
  } else {
    himuon::gated_up(a, cur_stream());
    gemm_into(h, wd, y, false, true);
  }
  autograd_launched += 2;
  return y;
}

struct GatedMlp : torch::autograd::Function<GatedMlp> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation) {
    GatedKept kept;
    const at::Tensor y = gated_forward(x, wg, wu, wd, activation, &kept);
    ctx->save_for_backward({x, wg, wu, wd, kept.h, kept.gu, kept.gu_low});
    ctx->saved_data["activation"] = activation;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_mlp");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &wd = saved[3], &h = saved[4], &gu = saved[5];
    const GatedSizes n{x.size(0), x.size(1), wg.size(0)};
    const c10::cuda::CUDAGuard guard(x.device());
    variable_list out(5);
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    if (!n.rows) {
      for (int i = 0; i < 4; ++i)
        if (ctx->needs_input_grad(i)) out[i] = at::zeros(saved[i].sizes(), saved[i].options());
      return out;
    }
    const at::Tensor dy = with_rows(grads[0]);
    if (ctx->needs_input_grad(3)) {
      out[3] = at::empty(wd.sizes(), wd.options());
      gemm_into(dy, h, out[3], true, false);
      autograd_launched += 1;
    }
    if (!need_x && !need_w) return out;
    at::Tensor dgu = at::empty_like(gu);
    himuon::GatedDownGradArgs a;
    a.dy = dy.data_ptr(); a.wd = wd.data_ptr(); a.gu = gu.data_ptr(); a.gu_low = saved[6].data_ptr(); a.dgu = dgu.data_ptr();
    a.ld_dy = dy.stride(0); a.ld_wd = wd.stride(0);
    a.rows = static_cast<int>(n.rows); a.hidden = static_cast<int>(n.hidden); a.inter = static_cast<int>(n.inter);
    a.activation = static_cast<int>(ctx->saved_data["activation"].toInt());
    himuon::gated_down_grad(a, cur_stream());
    autograd_launched += 1;
    if (need_x) {
      out[0] = at::empty(x.sizes(), x.options());
      himuon::GemmArgs g;                                // dx = dg Wg + du Wu
      g.A = dgu.data_ptr(); g.A2 = static_cast<char*>(dgu.data_ptr()) + 2 * n.inter;
      g.B = wg.data_ptr(); g.B2 = wu.data_ptr(); g.C = out[0].data_ptr();
      g.M = a.rows; g.N = a.hidden; g.K = a.inter;
      g.lda = 2 * n.inter; g.ldb = wg.stride(0); g.ldb2 = wu.stride(0); g.ldc = n.hidden;
      g.b_mn = true;
      at::Tensor parts;
      if (const int64_t floats = himuon::gemm2_parts_floats(g)) {
        parts = at::empty({floats}, x.options().dtype(at::kFloat));
        g.parts = parts.data_ptr<float>();
      }
      himuon::gemm2_bf16(g, cur_stream());
      autograd_launched += 1;
    }
    if (need_w) {
      at::Tensor dw = at::empty({2 * n.inter, n.hidden}, x.options());
      gemm_into(dgu, x, dw, true, false);
      autograd_launched += 1;
      if (ctx->needs_input_grad(1)) out[1] = dw.narrow(0, 0, n.inter);
      if (ctx->needs_input_grad(2)) out[2] = dw.narrow(0, n.inter, n.inter);
    }
    return out;
  }
};

// ------------------------------------------------------------------------------------------------ 8 bits
struct Fp8 { at::Tensor values, scales; int64_t block_rows = 1; bool powers = false; };      // powers: scales known to be powers of two

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }

// Room for (rows, cols) values, their rows padded to 16 bytes, and their scales: of rows along rows, which is how a product reads them.
Fp8 fp8_empty(const at::Tensor& like, int64_t rows, int64_t cols, int64_t block_rows) {
  Fp8 m;
  m.block_rows = block_rows;
  m.powers = true;                                       // (that is what it will be filled with)
  m.values = at::empty({rows, up(cols, 16) * 16}, like.options().dtype(at::kFloat8_e4m3fn)).narrow(1, 0, cols);
  const auto fp32 = like.options().dtype(at::kFloat);
  m.scales = block_rows == 1 ? at::empty({up(cols, 128), rows}, fp32).t() : at::empty({up(rows, 128), up(cols, 128)}, fp32);
  return m;
}
himuon::Fp8Out fp8_out(const Fp8& m) {
  himuon::Fp8Out o;
  o.values = m.values.data_ptr();
  o.scales = m.scales.data_ptr<float>();
  o.ld = m.values.stride(0); o.scale_row = m.scales.stride(0); o.scale_col = m.scales.stride(1);
  o.block_rows = static_cast<int>(m.block_rows);
  return o;
}
// Fills the copies that are given.
void quantize(const at::Tensor& x, const Fp8* straight, const Fp8* turned) {
  HM_CHECK(x.is_cuda() && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat) && x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1) &&
               (x.size(0) <= 1 || x.stride(0) >= x.size(1)), "quantize_fp8: a bf16 or fp32 matrix with unit inner stride expected");
  if (!x.numel() || (!straight && !turned)) return;
  const c10::cuda::CUDAGuard guard(x.device());
  himuon::Fp8QuantizeArgs a;
  a.x = x.data_ptr(); a.rows = x.size(0); a.cols = x.size(1); a.ld = x.stride(0); a.fp32 = x.scalar_type() == at::kFloat;
  if (straight) a.straight = fp8_out(*straight);
  if (turned) a.turned = fp8_out(*turned);
  himuon::fp8_quantize(a, cur_stream());
  autograd_launched += 1;
}
std::tuple<at::Tensor, at::Tensor> quantize_fp8(const at::Tensor& x, int64_t block_rows, bool transpose) {
  HM_CHECK(x.dim() == 2 && (block_rows == 1 || block_rows == 128), "quantize_fp8: a matrix and blocks of 1 or 128 rows expected");
  const Fp8 m = transpose ? fp8_empty(x, x.size(1), x.size(0), block_rows) : fp8_empty(x, x.size(0), x.size(1), block_rows);
  quantize(x, transpose ? nullptr : &m, transpose ? &m : nullptr);
  return {m.values, m.scales};
}

void check_fp8(const char* op, const Fp8& m, const at::Device& device) {
  TORCH_CHECK((m.block_rows == 1 || m.block_rows == 128) && m.values.device() == device && m.values.is_cuda() && m.values.scalar_type() == at::kFloat8_e4m3fn && m.values.dim() == 2 &&
                  m.values.size(0) < (1LL << 30) && m.values.size(1) < (1LL << 30),
              std::string("himuon: ") + op + ": a float8_e4m3fn matrix on " + device.str() + " with blocks of 1 or 128 rows expected");
  TORCH_CHECK(m.scales.device() == device && m.scales.scalar_type() == at::kFloat && m.scales.dim() == 2 && m.scales.size(0) == up(m.values.size(0), m.block_rows) &&
                  m.scales.size(1) == up(m.values.size(1), 128),
              std::string("himuon: ") + op + ": scales must be fp32, one for each block of (" + std::to_string(m.block_rows) + ", 128) values");
}
// Rows on 16-byte boundaries, each with memory of its own; copied where they lie otherwise.
at::Tensor fp8_rows(const at::Tensor& v) {
  if (v.stride(1) == 1 && v.stride(0) % 16 == 0 && (v.size(0) <= 1 || v.stride(0) >= v.size(1)) && aligned16(v)) return v;
  at::Tensor to = at::empty({v.size(0), up(v.size(1), 16) * 16}, v.options()).narrow(1, 0, v.size(1));
  to.copy_(v);
  return to;
}
himuon::Fp8Matrix fp8_matrix(const Fp8& m) {
  himuon::Fp8Matrix a;
  a.values = m.values.data_ptr(); a.scales = m.scales.data_ptr<float>();
  a.ld = m.values.stride(0); a.scale_row = m.scales.stride(0); a.scale_col = m.scales.stride(1);
  a.rows = static_cast<int>(m.values.size(0)); a.cols = static_cast<int>(m.values.size(1)); a.block_rows = static_cast<int>(m.block_rows);
  return a;
}
// a b^T in bf16 or fp32.
at::Tensor product(const char* op, Fp8 a, Fp8 b, bool out_fp32) {
  check_fp8(op, a, a.values.device());
  check_fp8(op, b, a.values.device());
  TORCH_CHECK(a.values.size(1) == b.values.size(1), "himuon: ", op, ": inner dimensions disagree");
  TORCH_CHECK(b.block_rows == 128, "himuon: ", op, ": the second operand needs blocks of 128 rows");
  const c10::cuda::CUDAGuard guard(a.values.device());
  const int64_t rows = a.values.size(0), cols = b.values.size(0), inner = a.values.size(1);
  const auto type = a.values.options().dtype(out_fp32 ? at::kFloat : at::kBFloat16);
  if (!rows || !cols) return at::empty({rows, cols}, type);
  if (!inner) return at::zeros({rows, cols}, type);
  a.values = fp8_rows(a.values);
  b.values = fp8_rows(b.values);
  autograd_launched += 1;
  if (rows <= himuon::kFewFp8Rows) {
    at::Tensor c = at::empty({rows, cols}, type);
    himuon::few_rows_fp8_product(fp8_matrix(a), fp8_matrix(b), c.data_ptr(), out_fp32, cur_stream());
    return c;
  }
  // (rows of the result are stored in groups of 16 bytes)
  const int64_t group = out_fp32 ? 4 : 8, ld = up(cols, group) * group;
  at::Tensor c = at::empty({rows, ld}, type);
  himuon::fp8_product(fp8_matrix(a), fp8_matrix(b), c.data_ptr(), ld, out_fp32, a.powers && b.powers, cur_stream());
  return ld == cols ? c : c.narrow(1, 0, cols).contiguous();
}
at::Tensor fp8_matmul(const at::Tensor& a, const at::Tensor& a_scales, int64_t a_block, bool a_powers, const at::Tensor& b, const at::Tensor& b_scales, int64_t b_block,
                      bool b_powers, bool out_fp32) {
  return product("fp8_matmul", Fp8{a, a_scales, a_block, a_powers}, Fp8{b, b_scales, b_block, b_powers}, out_fp32);
}
at::Tensor fp8_dequantize(const at::Tensor& values, const at::Tensor& scales, int64_t block_rows, bool out_fp32) {
  const Fp8 m{values, scales, block_rows};
  check_fp8("dequantize", m, values.device());
  HM_CHECK((values.stride(1) == 1 || values.size(1) <= 1), "dequantize: unit inner stride expected");
  const c10::cuda::CUDAGuard guard(values.device());
  at::Tensor out = at::empty(values.sizes(), values.options().dtype(out_fp32 ? at::kFloat : at::kBFloat16));
  if (out.numel()) {
    himuon::fp8_dequantize(fp8_matrix(m), out.data_ptr(), out.size(1), out_fp32, cur_stream());
    autograd_launched += 1;
  }
  return out;
}

// x w^T with w kept in 8 bits.
at::Tensor fp8_linear_kept(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scales, int64_t w_block, bool w_powers) {
  HM_CHECK(x.dim() == 2 && x.scalar_type() == at::kBFloat16, "fp8_linear: bf16 rows expected");
  const Fp8 q = fp8_empty(x, x.size(0), x.size(1), 1);
  quantize(x, &q, nullptr);
  return product("fp8_linear", q, Fp8{w, w_scales, w_block, w_powers}, false);
}
// x w^T with both put into 8 bits; copies turned around for the gradients' products are made on the way.
at::Tensor fp8_linear_forward(const at::Tensor& x, const at::Tensor& w, Fp8* xt, Fp8* wt) {
  HM_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16 && x.device() == w.device(),
           "fp8_linear: (rows, in) and (out, in) of bf16 on one device expected");
  const Fp8 q = fp8_empty(x, x.size(0), x.size(1), 1), v = fp8_empty(w, w.size(0), w.size(1), 128);
  if (xt) *xt = fp8_empty(x, x.size(1), x.size(0), 128);
  if (wt) *wt = fp8_empty(w, w.size(1), w.size(0), 128);
  quantize(x, &q, xt);
  quantize(w, &v, wt);
  return product("fp8_linear", q, v, false);
}

struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w) {
    Fp8 xt, wt;
    const bool need_x = x.requires_grad(), need_w = w.requires_grad();
    const at::Tensor y = fp8_linear_forward(x, w, need_w ? &xt : nullptr, need_x ? &wt : nullptr);
    variable_list keep;
    if (need_x) keep.insert(keep.end(), {wt.values, wt.scales});
    if (need_w) keep.insert(keep.end(), {xt.values, xt.scales});
    ctx->save_for_backward(keep);
    ctx->saved_data["need_x"] = need_x;
    ctx->saved_data["need_w"] = need_w;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("fp8_linear");
    const variable_list saved = ctx->get_saved_variables();
    const bool kept_x = ctx->saved_data["need_x"].toBool(), kept_w = ctx->saved_data["need_w"].toBool();
    const bool need_x = kept_x && ctx->needs_input_grad(0), need_w = kept_w && ctx->needs_input_grad(1);
    at::Tensor dy = grads[0];
    if ((dy.stride(1) != 1 && dy.size(1) > 1) || (dy.size(0) > 1 && dy.stride(0) < dy.size(1))) dy = dy.clone(at::MemoryFormat::Contiguous);
    const c10::cuda::CUDAGuard guard(dy.device());
    Fp8 q, qt;
    if (need_x) q = fp8_empty(dy, dy.size(0), dy.size(1), 1);
    if (need_w) qt = fp8_empty(dy, dy.size(1), dy.size(0), 1);
    quantize(dy, need_x ? &q : nullptr, need_w ? &qt : nullptr);
    variable_list out(2);
    if (need_x) out[0] = product("fp8_linear", q, Fp8{saved[0], saved[1], 128, true}, false);
    if (need_w) out[1] = product("fp8_linear", qt, Fp8{saved[kept_x ? 2 : 0], saved[kept_x ? 3 : 1], 128, true}, false);
    return out;
  }
};

}  // namespace

void bind_layer_ops(pybind11::module& m) {
  m.def("rotary", [](const at::Tensor& x, const c10::optional<at::Tensor>& positions, const at::Tensor& turns, int64_t seq_len, int64_t heads, int64_t rotary_dim,
                     bool interleaved, double factor) {
    if (any_grad({&x})) return Rotary::apply(x, positions, turns, seq_len, heads, rotary_dim, interleaved, factor, factor);
    return rotate(x, positions, turns, seq_len, heads, rotary_dim, interleaved, factor, factor);
  });
  m.def("gated_mlp", [](const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation) {
    if (any_grad({&x, &wg, &wu, &wd})) return GatedMlp::apply(x, wg, wu, wd, activation);
    return gated_forward(x, wg, wu, wd, activation, nullptr);
  });
  m.def("quantize_fp8", &quantize_fp8);
  m.def("fp8_dequantize", &fp8_dequantize);
  m.def("fp8_matmul", &fp8_matmul);
  m.def("fp8_linear_kept", &fp8_linear_kept);
  m.def("fp8_linear", [](const at::Tensor& x, const at::Tensor& w) {
    if (any_grad({&x, &w})) return Fp8Linear::apply(x, w);
    return fp8_linear_forward(x, w, nullptr, nullptr);
  });
}
