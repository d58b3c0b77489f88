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
                  t.stride(0) % 8 == 0 && t.stride(0) >= cols && aligned16(t),
              std::string("himuon: ") + op + ": " + name + " must be (" + std::to_string(rows) + ", " + std::to_string(cols) + ") bf16, its rows on 16-byte boundaries with unit inner stride");
}
// Rows of all dimensions but the last.
int64_t flat_rows(const at::Tensor& t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  return n;
}
// Rows as check_rows() wants them: copied where they lie otherwise (a single row too, whose stride may be anything: a tensor map takes none below its width).
at::Tensor with_rows(const at::Tensor& t) {
  if (t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && aligned16(t)) return t;
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
// A product with rows of c one behind the other, on CTA pairs or where gemm() sends it.
void product_into(himuon::GemmArgs& g, bool pairs, const at::Tensor& like) {
  at::Tensor parts;
  if (const int64_t floats = pairs ? himuon::gemm2_parts_floats(g) : himuon::gemm_parts_floats(g)) {
    parts = at::empty({floats}, like.options().dtype(at::kFloat));
    g.parts = parts.data_ptr<float>();
  }
  if (pairs) himuon::gemm2_bf16(g, cur_stream());
  else himuon::gemm_bf16(g, cur_stream());
  autograd_launched += 1;
}
himuon::GemmArgs product_of(const void* a, int64_t lda, bool a_mn, const void* b, int64_t ldb, bool b_mn, const at::Tensor& c, int64_t inner) {
  himuon::GemmArgs g;
  g.A = a; g.B = b; g.C = c.data_ptr();
  g.M = static_cast<int>(c.size(0)); g.N = static_cast<int>(c.size(1)); g.K = static_cast<int>(inner);
  g.lda = lda; g.ldb = ldb; g.ldc = c.size(1);
  g.a_mn = a_mn; g.b_mn = b_mn;
  return g;
}
// h and, for a backward pass, what is kept of g | u, in one piece of memory.
struct GatedKept {
  char *h, *gu, *low;
  static int64_t bytes(const GatedSizes& n, bool all) { return n.rows * (2 * n.inter + (all ? 4 * n.inter + 2 * himuon::gated_low(static_cast<int>(n.inter)) : 0)); }
  GatedKept(const at::Tensor& piece, const GatedSizes& n)
      : h(static_cast<char*>(piece.data_ptr())), gu(h + 2 * n.rows * n.inter), low(gu + 4 * n.rows * n.inter) {}
};
// y; `piece` is left there if it is asked for.
at::Tensor gated_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation, at::Tensor* piece) {
  const GatedSizes n = gated_sizes(x, wg, wu, wd, activation);
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor memory = at::empty({GatedKept::bytes(n, piece != nullptr)}, x.options().dtype(at::kByte));
  const GatedKept kept(memory, n);
  at::Tensor y = at::empty({n.rows, n.hidden}, x.options());
  if (piece) *piece = memory;
  if (!n.rows) return y;
  himuon::GatedUpArgs a;
  a.x = x.data_ptr(); a.wg = wg.data_ptr(); a.wu = wu.data_ptr();
  a.h = kept.h; a.gu = piece ? kept.gu : nullptr; a.gu_low = piece ? kept.low : nullptr;
  a.ld_x = x.stride(0); a.ld_wg = wg.stride(0); a.ld_wu = wu.stride(0);
  a.rows = static_cast<int>(n.rows); a.hidden = static_cast<int>(n.hidden); a.inter = static_cast<int>(n.inter); a.activation = static_cast<int>(activation);
  autograd_launched += 1;
  if (himuon::few_gated_rows(n.rows, n.hidden, n.inter)) {
    himuon::few_rows_gated_up(a, cur_stream());
    himuon::few_rows_product(kept.h, n.inter, wd.data_ptr(), wd.stride(0), y.data_ptr(), a.rows, a.inter, a.hidden, true, cur_stream());
    autograd_launched += 1;
    return y;
  }
  himuon::gated_up(a, cur_stream());
  himuon::GemmArgs g = product_of(kept.h, n.inter, false, wd.data_ptr(), wd.stride(0), false, y, n.inter);
  // Where the pair GEMM has tiles for less than half of the pairs it is taken all the same, as it cuts them along the inner dimension.
  // Gated and back, 80 rows of 4096 x 12288: 94 us for 109 where gemm() sends it, 139 rows of 472 x 5648 30 for 45.
  const int64_t tiles = (n.rows + 255) / 256 * ((n.hidden + 255) / 256), pairs = himuon::num_sms() / 2, blocks = (n.inter + 63) / 64, cuts = std::min(pairs / tiles, blocks / 8);
  const bool cut = 2 * tiles <= pairs && cuts >= 2 && (cuts - 1) * blocks / cuts >= 40;
  g.ordered = cut;
  product_into(g, cut, x);
  return y;
}

struct GatedMlp : torch::autograd::Function<GatedMlp> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation) {
    at::Tensor piece;
    const at::Tensor y = gated_forward(x, wg, wu, wd, activation, &piece);
    ctx->save_for_backward({x, wg, wu, wd, piece});
    ctx->saved_data["activation"] = activation;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_mlp");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &wd = saved[3], &piece = saved[4];
    const int64_t activation = ctx->saved_data["activation"].toInt();
    const GatedSizes n = gated_sizes(x, wg, wu, wd, activation);       // (hooks may have moved what was kept)
    HM_CHECK(piece.device() == x.device() && piece.scalar_type() == at::kByte && piece.is_contiguous() && piece.numel() == GatedKept::bytes(n, true) && aligned16(piece),
             "gated_mlp: what was kept has changed");
    const GatedKept kept(piece, n);
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
      out[3] = at::empty({n.hidden, n.inter}, wd.options());
      himuon::GemmArgs g = product_of(dy.data_ptr(), dy.stride(0), true, kept.h, n.inter, true, out[3], n.rows);
      product_into(g, false, x);
    }
    if (!need_x && !need_w) return out;
    const at::Tensor dgu = at::empty({n.rows, 2 * n.inter}, x.options());
    himuon::GatedDownGradArgs a;
    a.dy = dy.data_ptr(); a.wd = wd.data_ptr(); a.gu = kept.gu; a.gu_low = kept.low; a.dgu = dgu.data_ptr();
    a.ld_dy = dy.stride(0); a.ld_wd = wd.stride(0);
    a.rows = static_cast<int>(n.rows); a.hidden = static_cast<int>(n.hidden); a.inter = static_cast<int>(n.inter);
    a.activation = static_cast<int>(activation);
    himuon::gated_down_grad(a, cur_stream());
    autograd_launched += 1;
    if (need_x) {                                        // dx = dg Wg + du Wu
      out[0] = at::empty({n.rows, n.hidden}, x.options());
      himuon::GemmArgs g = product_of(dgu.data_ptr(), 2 * n.inter, false, wg.data_ptr(), wg.stride(0), true, out[0], n.inter);
      g.A2 = static_cast<char*>(dgu.data_ptr()) + 2 * n.inter;
      g.B2 = wu.data_ptr(); g.ldb2 = wu.stride(0);
      g.ordered = 1;                                     // (so that few tiles are cut along the inner dimension too: 777 rows, 640 x 1728 17 us for 23)
      product_into(g, true, x);
    }
    if (need_w) {
      const at::Tensor dw = at::empty({2 * n.inter, n.hidden}, x.options());
      himuon::GemmArgs g = product_of(dgu.data_ptr(), 2 * n.inter, true, x.data_ptr(), x.stride(0), true, dw, n.rows);
      product_into(g, false, x);
      if (ctx->needs_input_grad(1)) out[1] = dw.narrow(0, 0, n.inter);
      if (ctx->needs_input_grad(2)) out[2] = dw.narrow(0, n.inter, n.inter);
    }
    return out;
  }
};

// ------------------------------------------------------------------------------------------------ 8 bits
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }

// A matrix in 8 bits and what holds its memory.  `powers`: its scales are known to be powers of two.
struct Fp8 {
  himuon::Fp8Matrix m;
  bool powers = false;
  at::Tensor values, scales;             // or all in `values`
};

// Where values, with rows padded to 16 bytes, and scales of a matrix lie in one piece of memory; scales of rows one behind the other, which is how a
// product reads them.
int64_t fp8_scales_at(int64_t rows, int64_t cols) { return rows * up(cols, 16) * 16; }
int64_t fp8_scale_count(int64_t rows, int64_t cols, int64_t block_rows) { return up(rows, block_rows) * up(cols, 128); }
Fp8 fp8_in(const at::Tensor& piece, int64_t rows, int64_t cols, int64_t block_rows) {
  Fp8 q;
  char* at = static_cast<char*>(piece.data_ptr());
  q.m.values = at;
  q.m.scales = reinterpret_cast<float*>(at + fp8_scales_at(rows, cols));
  q.m.ld = up(cols, 16) * 16;
  q.m.scale_row = block_rows == 1 ? 1 : up(cols, 128);
  q.m.scale_col = block_rows == 1 ? rows : 1;
  q.m.rows = static_cast<int>(rows); q.m.cols = static_cast<int>(cols); q.m.block_rows = static_cast<int>(block_rows);
  q.powers = true;                       // (that is what it will be filled with)
  q.values = piece;
  return q;
}
Fp8 fp8_piece(const at::Tensor& like, int64_t rows, int64_t cols, int64_t block_rows) {
  HM_CHECK(rows < (1LL << 30) && cols < (1LL << 30), "a matrix in 8 bits is too large");
  return fp8_in(at::empty({fp8_scales_at(rows, cols) + 4 * fp8_scale_count(rows, cols, block_rows)}, like.options().dtype(at::kByte)), rows, cols, block_rows);
}
himuon::Fp8Out fp8_out(const himuon::Fp8Matrix& m) {
  himuon::Fp8Out o;
  o.values = const_cast<void*>(m.values);
  o.scales = const_cast<float*>(m.scales);
  o.ld = m.ld; o.scale_row = m.scale_row; o.scale_col = m.scale_col;
  o.block_rows = m.block_rows;
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
  if (straight) a.straight = fp8_out(straight->m);
  if (turned) a.turned = fp8_out(turned->m);
  himuon::fp8_quantize(a, cur_stream());
  autograd_launched += 1;
}
// Rows with unit inner stride that share no memory: copied where they lie otherwise.
at::Tensor apart(const at::Tensor& t) {
  if ((t.stride(1) == 1 || t.size(1) <= 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}
std::tuple<at::Tensor, at::Tensor> quantize_fp8(const at::Tensor& given, int64_t block_rows, bool transpose) {
  HM_CHECK(given.dim() == 2 && (block_rows == 1 || block_rows == 128), "quantize_fp8: a matrix and blocks of 1 or 128 rows expected");
  const at::Tensor x = apart(given);
  const int64_t rows = transpose ? x.size(1) : x.size(0), cols = transpose ? x.size(0) : x.size(1), ld = up(cols, 16) * 16;
  HM_CHECK(rows < (1LL << 30) && cols < (1LL << 30), "quantize_fp8: matrix too large");
  const auto fp32 = x.options().dtype(at::kFloat);
  const std::vector<int64_t> blocks = {up(rows, block_rows), up(cols, 128)};
  at::Tensor values = at::empty({rows, ld}, x.options().dtype(at::kFloat8_e4m3fn));
  const at::Tensor scales = block_rows == 1 ? at::empty_strided(blocks, {1, std::max<int64_t>(rows, 1)}, fp32) : at::empty(blocks, fp32);
  Fp8 q;
  q.m.values = values.data_ptr(); q.m.scales = scales.data_ptr<float>();
  q.m.ld = ld; q.m.scale_row = scales.stride(0); q.m.scale_col = scales.stride(1);
  q.m.block_rows = static_cast<int>(block_rows);
  quantize(x, transpose ? nullptr : &q, transpose ? &q : nullptr);
  return {ld == cols ? values : values.narrow(1, 0, cols), scales};
}

// A matrix as a caller has it, checked.  `rows16`: with its rows on 16-byte boundaries, each with memory of its own; copied where they lie otherwise.
Fp8 fp8_given(const char* op, const at::Tensor& values, const at::Tensor& scales, int64_t block_rows, bool powers, const at::Device& device, bool rows16) {
  TORCH_CHECK((block_rows == 1 || block_rows == 128) && values.device() == device && values.is_cuda() && values.scalar_type() == at::kFloat8_e4m3fn && values.dim() == 2 &&
                  values.size(0) < (1LL << 30) && values.size(1) < (1LL << 30),
              std::string("himuon: ") + op + ": a float8_e4m3fn matrix on " + device.str() + " with blocks of 1 or 128 rows expected");
  TORCH_CHECK(scales.device() == device && scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == up(values.size(0), block_rows) &&
                  scales.size(1) == up(values.size(1), 128),
              std::string("himuon: ") + op + ": scales must be fp32, one for each block of (" + std::to_string(block_rows) + ", 128) values");
  Fp8 q;
  q.values = values;
  const bool unit = values.stride(1) == 1 || (!rows16 && values.size(1) <= 1);
  if (rows16 && !(unit && values.stride(0) % 16 == 0 && values.stride(0) >= values.size(1) && aligned16(values))) {
    q.values = at::empty({values.size(0), up(values.size(1), 16) * 16}, values.options()).narrow(1, 0, values.size(1));
    q.values.copy_(values);
  } else if (!unit) {
    q.values = values.contiguous();
  }
  q.scales = scales;
  q.powers = powers;
  q.m.values = q.values.data_ptr(); q.m.scales = scales.data_ptr<float>();
  q.m.ld = q.values.stride(0); q.m.scale_row = scales.stride(0); q.m.scale_col = scales.stride(1);
  q.m.rows = static_cast<int>(values.size(0)); q.m.cols = static_cast<int>(values.size(1)); q.m.block_rows = static_cast<int>(block_rows);
  return q;
}
// a b^T in bf16 or fp32.
// `early`: b was there before the launch before this one, which makes a.
at::Tensor product(const char* op, const Fp8& a, const Fp8& b, bool out_fp32, bool early = false) {
  TORCH_CHECK(a.m.cols == b.m.cols, "himuon: ", op, ": inner dimensions disagree");
  TORCH_CHECK(b.m.block_rows == 128, "himuon: ", op, ": the second operand needs blocks of 128 rows");
  const c10::cuda::CUDAGuard guard(a.values.device());
  const int64_t rows = a.m.rows, cols = b.m.rows;
  const auto type = a.values.options().dtype(out_fp32 ? at::kFloat : at::kBFloat16);
  if (!rows || !cols) return at::empty({rows, cols}, type);
  if (!a.m.cols) return at::zeros({rows, cols}, type);
  autograd_launched += 1;
  if (himuon::few_fp8_rows(a.m, b.m)) {
    at::Tensor c = at::empty({rows, cols}, type);
    himuon::few_rows_fp8_product(a.m, b.m, c.data_ptr(), out_fp32, early, cur_stream());
    return c;
  }
  // (rows of the result are stored in groups of 16 bytes)
  const int64_t group = out_fp32 ? 4 : 8, ld = up(cols, group) * group;
  at::Tensor c = at::empty({rows, ld}, type);
  const bool powers = a.powers && b.powers;
  at::Tensor parts;
  if (const int64_t floats = himuon::fp8_parts_floats(a.m, b.m)) parts = at::empty({floats}, a.values.options().dtype(at::kFloat));
  himuon::fp8_product(a.m, b.m, c.data_ptr(), ld, out_fp32, powers, parts.defined() ? parts.data_ptr<float>() : nullptr, cur_stream());
  return ld == cols ? c : c.narrow(1, 0, cols).contiguous();
}
at::Tensor fp8_matmul(const at::Tensor& a, const at::Tensor& a_scales, int64_t a_block, bool a_powers, const at::Tensor& b, const at::Tensor& b_scales, int64_t b_block,
                      bool b_powers, bool out_fp32) {
  return product("fp8_matmul", fp8_given("fp8_matmul", a, a_scales, a_block, a_powers, a.device(), true), fp8_given("fp8_matmul", b, b_scales, b_block, b_powers, a.device(), true),
                 out_fp32);
}
at::Tensor fp8_dequantize(const at::Tensor& values, const at::Tensor& scales, int64_t block_rows, bool out_fp32) {
  const Fp8 q = fp8_given("dequantize", values, scales, block_rows, false, values.device(), false);
  const c10::cuda::CUDAGuard guard(values.device());
  at::Tensor out = at::empty(values.sizes(), values.options().dtype(out_fp32 ? at::kFloat : at::kBFloat16));
  if (out.numel()) {
    himuon::fp8_dequantize(q.m, out.data_ptr(), out.size(1), out_fp32, cur_stream());
    autograd_launched += 1;
  }
  return out;
}

// x w^T with w kept in 8 bits.
at::Tensor fp8_linear_kept(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scales, int64_t w_block, bool w_powers) {
  HM_CHECK(x.dim() == 2 && x.is_cuda() && x.scalar_type() == at::kBFloat16, "fp8_linear: bf16 rows expected");
  const Fp8 v = fp8_given("fp8_linear", w, w_scales, w_block, w_powers, x.device(), true);
  const Fp8 q = fp8_piece(x, x.size(0), x.size(1), 1);
  quantize(x, &q, nullptr);
  return product("fp8_linear", q, v, false, true);
}
// x w^T with both put into 8 bits; copies turned around for the gradients' products are made on the way.
at::Tensor fp8_linear_forward(const at::Tensor& x, const at::Tensor& w, const Fp8* xt, const Fp8* wt) {
  const Fp8 q = fp8_piece(x, x.size(0), x.size(1), 1), v = fp8_piece(w, w.size(0), w.size(1), 128);
  quantize(x, &q, xt);
  quantize(w, &v, wt);
  return product("fp8_linear", q, v, false);
}

struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w) {
    const bool need_x = x.requires_grad(), need_w = w.requires_grad();
    Fp8 xt, wt;
    if (need_w) xt = fp8_piece(x, x.size(1), x.size(0), 128);
    if (need_x) wt = fp8_piece(w, w.size(1), w.size(0), 128);
    const at::Tensor y = fp8_linear_forward(x, w, need_w ? &xt : nullptr, need_x ? &wt : nullptr);
    variable_list keep;
    if (need_x) keep.push_back(wt.values);
    if (need_w) keep.push_back(xt.values);
    ctx->save_for_backward(keep);
    ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), x.size(1), w.size(0), need_x, need_w};
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("fp8_linear");
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> n = ctx->saved_data["sizes"].toIntVector();       // rows, in, out, and what was kept
    const int64_t rows = n[0], in = n[1], out = n[2];
    const bool need_x = n[3] && ctx->needs_input_grad(0), need_w = n[4] && ctx->needs_input_grad(1);
    const at::Tensor dy = apart(grads[0]);
    const c10::cuda::CUDAGuard guard(dy.device());
    auto kept = [&](int64_t i, int64_t cols) {           // (hooks may have moved it)
      const at::Tensor& t = saved[i];
      HM_CHECK(t.device() == dy.device() && t.scalar_type() == at::kByte && t.is_contiguous() && t.numel() == fp8_scales_at(in, cols) + 4 * fp8_scale_count(in, cols, 128) &&
                   aligned16(t), "fp8_linear: what was kept has changed");
      return fp8_in(t, in, cols, 128);
    };
    Fp8 q, qt;
    if (need_x) q = fp8_piece(dy, rows, out, 1);
    if (need_w) qt = fp8_piece(dy, out, rows, 1);
    quantize(dy, need_x ? &q : nullptr, need_w ? &qt : nullptr);
    variable_list result(2);
    if (need_x) result[0] = product("fp8_linear", q, kept(0, out), false);
    if (need_w) result[1] = product("fp8_linear", qt, kept(n[3] ? 1 : 0, rows), false);
    return result;
  }
};

std::vector<int64_t> shape_of(const at::Tensor& x, const at::Tensor& w) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = w.size(0);
  return shape;
}

}  // namespace

void bind_layer_ops(pybind11::module& m) {
  m.def("rotary", [](const at::Tensor& x, const c10::optional<at::Tensor>& positions, const at::Tensor& turns, int64_t seq_len, int64_t heads, int64_t rotary_dim,
                     bool interleaved, double factor) {
    if (any_grad({&x})) return Rotary::apply(x, positions, turns, seq_len, heads, rotary_dim, interleaved, factor, factor);
    return rotate(x, positions, turns, seq_len, heads, rotary_dim, interleaved, factor, factor);
  });
  m.def("gated_mlp", [](const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t activation) {
    HM_CHECK(x.dim() >= 1 && wg.dim() == 2 && wu.dim() == 2 && wd.dim() == 2 && x.size(-1) == wg.size(1), "gated_mlp: (..., hidden) and (inter, hidden) expected");
    const bool flat = x.dim() == 2;
    const at::Tensor x2 = with_rows(flat ? x : x.reshape({flat_rows(x), x.size(-1)})), g = with_rows(wg), u = with_rows(wu), d = with_rows(wd);
    at::Tensor y = any_grad({&x2, &g, &u, &d}) ? GatedMlp::apply(x2, g, u, d, activation) : gated_forward(x2, g, u, d, activation, nullptr);
    return flat ? y : y.view(x.sizes());
  });
  m.def("quantize_fp8", &quantize_fp8);
  m.def("fp8_dequantize", &fp8_dequantize);
  m.def("fp8_matmul", &fp8_matmul);
  m.def("fp8_linear_kept", [](const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scales, int64_t w_block, bool w_powers) {
    HM_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "fp8_linear: (..., in) inputs and an (out, in) weight expected");
    if (x.dim() == 2) return fp8_linear_kept(apart(x), w, w_scales, w_block, w_powers);
    return fp8_linear_kept(apart(x.reshape({flat_rows(x), x.size(-1)})), w, w_scales, w_block, w_powers).view(shape_of(x, w));
  });
  m.def("fp8_linear", [](const at::Tensor& x, const at::Tensor& w) {
    HM_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && x.is_cuda() && x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16 && x.device() == w.device(),
             "fp8_linear: (..., in) and (out, in) of bf16 on one device expected");
    const bool flat = x.dim() == 2;
    const at::Tensor x2 = apart(flat ? x : x.reshape({flat_rows(x), x.size(-1)})), w2 = apart(w);
    at::Tensor y = any_grad({&x2, &w2}) ? Fp8Linear::apply(x2, w2) : fp8_linear_forward(x2, w2, nullptr, nullptr);
    return flat ? y : y.view(shape_of(x, w));
  });
}
