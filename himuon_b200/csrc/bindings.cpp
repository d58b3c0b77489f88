// PyTorch bindings: tensors in, raw pointers + current stream out.  All checks that would
// otherwise become device faults (dtype, contiguity, alignment, shape agreement) happen here.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>

#include "himuon.h"
#include "symm.h"

namespace py = pybind11;
using himuon::GemmArgs;

#define HM_CHECK(cond, msg) TORCH_CHECK(cond, "himuon: ", msg)

static cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
static bool is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }
static bool is_f32(const at::Tensor& t) { return t.scalar_type() == at::kFloat; }

// out = alpha * op(a) @ op(b) + beta * aux.   a: (.., M, K) or (.., K, M) when trans_a; b: (.., K, N) or (.., N, K) when trans_b.
static GemmArgs gemm_args(const at::Tensor& a, const at::Tensor& b, const at::Tensor& out, const c10::optional<at::Tensor>& aux,
                          bool trans_a, bool trans_b, double alpha, double beta, bool round_acc, int64_t max_ctas,
                          bool symmetric) {
  HM_CHECK(a.is_cuda() && b.is_cuda() && out.is_cuda(), "gemm operands must be CUDA tensors");
  HM_CHECK(is_bf16(a) && is_bf16(b), "gemm operands must be bf16");
  HM_CHECK(is_bf16(out) || is_f32(out), "gemm output must be bf16 or fp32");
  HM_CHECK(a.dim() == b.dim() && a.dim() == out.dim() && (a.dim() == 2 || a.dim() == 3), "gemm takes 2-D or 3-D operands");
  const int nd = a.dim();
  GemmArgs g;
  g.batch = nd == 3 ? static_cast<int>(a.size(0)) : 1;
  const int64_t a_rows = a.size(nd - 2), a_cols = a.size(nd - 1);
  const int64_t b_rows = b.size(nd - 2), b_cols = b.size(nd - 1);
  g.M = static_cast<int>(trans_a ? a_cols : a_rows);
  g.K = static_cast<int>(trans_a ? a_rows : a_cols);
  g.N = static_cast<int>(trans_b ? b_rows : b_cols);
  HM_CHECK((trans_b ? b_cols : b_rows) == g.K, "gemm inner dimensions disagree");
  HM_CHECK(out.size(nd - 2) == g.M && out.size(nd - 1) == g.N, "gemm output has the wrong shape");
  HM_CHECK(a.stride(nd - 1) == 1 && b.stride(nd - 1) == 1 && out.stride(nd - 1) == 1, "gemm needs unit inner strides");
  if (nd == 3) HM_CHECK(b.size(0) == g.batch && out.size(0) == g.batch, "gemm batch sizes disagree");
  g.A = a.data_ptr(); g.B = b.data_ptr(); g.C = out.data_ptr();
  g.lda = a.stride(nd - 2); g.ldb = b.stride(nd - 2); g.ldc = out.stride(nd - 2);
  g.strideA = nd == 3 ? a.stride(0) : 0; g.strideB = nd == 3 ? b.stride(0) : 0; g.strideC = nd == 3 ? out.stride(0) : 0;
  HM_CHECK(g.lda % 8 == 0 && g.ldb % 8 == 0 && g.strideA % 8 == 0 && g.strideB % 8 == 0,
           "gemm operand strides must be multiples of 8 elements (16 bytes)");
  HM_CHECK(reinterpret_cast<uintptr_t>(g.A) % 16 == 0 && reinterpret_cast<uintptr_t>(g.B) % 16 == 0,
           "gemm operand base addresses must be 16-byte aligned");
  g.a_mn = trans_a;     // stored (K, M): M contiguous
  g.b_mn = !trans_b;    // stored (K, N): N contiguous
  g.alpha = static_cast<float>(alpha); g.beta = static_cast<float>(beta);
  g.out_fp32 = is_f32(out) ? 1 : 0;
  g.round_acc = round_acc ? 1 : 0;
  g.max_ctas = static_cast<int>(max_ctas);
  g.symmetric = symmetric ? 1 : 0;
  if (symmetric) HM_CHECK(g.M == g.N, "gemm: a symmetric output must be square");
  if (aux.has_value() && beta != 0.0) {
    const at::Tensor& x = aux.value();
    HM_CHECK(x.scalar_type() == out.scalar_type() && x.dim() == nd && x.stride(nd - 1) == 1, "gemm aux must match the output dtype/rank");
    HM_CHECK(x.size(nd - 2) == g.M && x.size(nd - 1) == g.N && (nd == 2 || x.size(0) >= g.batch), "gemm aux has the wrong shape");
    g.aux = x.data_ptr(); g.ldaux = x.stride(nd - 2); g.strideAux = nd == 3 ? x.stride(0) : 0;
  }
  return g;
}
static void gemm(const at::Tensor& a, const at::Tensor& b, at::Tensor& out, const c10::optional<at::Tensor>& aux,
                 bool trans_a, bool trans_b, double alpha, double beta, bool round_acc, int64_t max_ctas,
                 bool symmetric, bool ordered = false) {
  GemmArgs g = gemm_args(a, b, out, aux, trans_a, trans_b, alpha, beta, round_acc, max_ctas, symmetric);
  const c10::cuda::CUDAGuard guard(a.device());
  g.ordered = ordered ? 1 : 0;
  // (of this call's stream: calls on different streams share nothing)
  at::Tensor parts;
  if (const int64_t floats = himuon::gemm_parts_floats(g)) {
    parts = at::empty({floats}, a.options().dtype(at::kFloat));
    g.parts = parts.data_ptr<float>();
  }
  himuon::gemm_bf16(g, cur_stream());
}
// Whether gemm() with these arguments runs on CTA pairs.
static bool gemm_on_pairs(const at::Tensor& a, const at::Tensor& b, const at::Tensor& out, const c10::optional<at::Tensor>& aux,
                          bool trans_a, bool trans_b, double alpha, double beta, bool round_acc, int64_t max_ctas,
                          bool symmetric) {
  const GemmArgs g = gemm_args(a, b, out, aux, trans_a, trans_b, alpha, beta, round_acc, max_ctas, symmetric);
  const c10::cuda::CUDAGuard guard(a.device());
  return himuon::gemm2_supported(g);
}

static void momentum_tile(const at::Tensor& entries, int64_t n_entries, int64_t total_units, int64_t Th, int64_t Tw,
                          at::Tensor& tiles, double mu, bool nesterov, double gscale, int64_t n_src, bool grad_fp32) {
  HM_CHECK(entries.is_cuda() && tiles.is_cuda() && is_bf16(tiles), "momentum_tile: bad buffers");
  HM_CHECK(entries.numel() >= n_entries * (int64_t)sizeof(himuon::MomTileEntry), "momentum_tile: entry table too small");
  HM_CHECK(n_src >= 1 && n_src <= himuon::kMaxSrc, "momentum_tile: unsupported number of gradient replicas");
  const c10::cuda::CUDAGuard guard(tiles.device());
  himuon::momentum_tile(reinterpret_cast<const himuon::MomTileEntry*>(entries.data_ptr()), (int)n_entries, (int)total_units,
                        (int)Th, (int)Tw, tiles.data_ptr(), (float)mu, nesterov ? 1 : 0, (float)gscale, (int)n_src,
                        grad_fp32 ? 1 : 0, cur_stream());
}
static void untile_apply(const at::Tensor& entries, int64_t n_entries, int64_t total_units, int64_t Th, int64_t Tw,
                         const at::Tensor& tiles, const at::Tensor& hyper, bool param_fp32) {
  HM_CHECK(entries.is_cuda() && tiles.is_cuda() && is_bf16(tiles) && hyper.is_cuda() && is_f32(hyper), "untile_apply: bad buffers");
  HM_CHECK(entries.numel() >= n_entries * (int64_t)sizeof(himuon::ApplyEntry), "untile_apply: entry table too small");
  const c10::cuda::CUDAGuard guard(tiles.device());
  himuon::untile_apply(reinterpret_cast<const himuon::ApplyEntry*>(entries.data_ptr()), (int)n_entries, (int)total_units,
                       (int)Th, (int)Tw, tiles.data_ptr(), hyper.data_ptr<float>(), param_fp32 ? 1 : 0, cur_stream());
}
static void ns_repad(const at::Tensor& src, at::Tensor& dst, const c10::optional<at::Tensor>& norm, double eps) {
  HM_CHECK(src.is_cuda() && dst.is_cuda() && src.dim() == 3 && dst.dim() == 3 && src.size(0) == dst.size(0) && src.is_contiguous() && dst.is_contiguous(), "ns_repad: contiguous (B, m, n) tensors");
  HM_CHECK((is_bf16(src) || is_f32(src)) && (is_bf16(dst) || is_f32(dst)) && (is_bf16(src) || is_bf16(dst)), "ns_repad: bf16 on one side, bf16 or fp32 on the other");
  HM_CHECK(src.size(1) < (1LL << 30) && src.size(2) < (1LL << 30) && dst.size(1) < (1LL << 30) && dst.size(2) < (1LL << 30), "ns_repad: matrix too large");
  HM_CHECK(src.data_ptr() != dst.data_ptr() || (src.scalar_type() == dst.scalar_type() && src.sizes() == dst.sizes()), "ns_repad: in place needs one size and type");
  if (norm.has_value()) HM_CHECK(norm->is_cuda() && is_f32(*norm) && norm->is_contiguous() && norm->numel() == src.size(0), "ns_repad: one fp32 norm per matrix");
  const c10::cuda::CUDAGuard guard(src.device());
  himuon::ns_repad(src.data_ptr(), dst.data_ptr(), src.size(0), (int)src.size(1), (int)src.size(2), (int)dst.size(1), (int)dst.size(2),
                   is_f32(src) ? 1 : 0, is_f32(dst) ? 1 : 0, cur_stream(), norm.has_value() ? norm->data_ptr<float>() : nullptr, (float)eps);
}
static void ns_normalize(at::Tensor& tiles, int64_t n_tiles, int64_t tile_elems, double eps, const c10::optional<at::Tensor>& out) {
  HM_CHECK(tiles.is_cuda() && is_bf16(tiles) && tiles.is_contiguous(), "ns_normalize: tiles must be contiguous bf16");
  HM_CHECK(tiles.numel() >= n_tiles * tile_elems, "ns_normalize: buffer too small");
  if (out.has_value())
    HM_CHECK(out->is_cuda() && is_bf16(*out) && out->is_contiguous() && out->numel() >= n_tiles * tile_elems, "ns_normalize: bad out");
  const c10::cuda::CUDAGuard guard(tiles.device());
  himuon::ns_normalize(tiles.data_ptr(), n_tiles, tile_elems, (float)eps, cur_stream(), out.has_value() ? out->data_ptr() : nullptr);
}
static void adamw_multi(const at::Tensor& entries, int64_t n_entries, int64_t total_units, const at::Tensor& hyper,
                        at::Tensor& step, int64_t mode, bool param_fp32, bool state_fp32) {
  HM_CHECK(entries.is_cuda() && hyper.is_cuda() && is_f32(hyper) && step.is_cuda() && is_f32(step), "adamw_multi: bad buffers");
  HM_CHECK(entries.numel() >= n_entries * (int64_t)sizeof(himuon::AdamEntry), "adamw_multi: entry table too small");
  const c10::cuda::CUDAGuard guard(hyper.device());
  himuon::adamw_multi(reinterpret_cast<const himuon::AdamEntry*>(entries.data_ptr()), (int)n_entries, total_units,
                      hyper.data_ptr<float>(), step.data_ptr<float>(), (int)mode, param_fp32 ? 1 : 0, state_fp32 ? 1 : 0,
                      cur_stream());
}
static void adamw_step_advance(at::Tensor& step) {
  const c10::cuda::CUDAGuard guard(step.device());
  himuon::adamw_step_advance(step.data_ptr<float>(), cur_stream());
}

static void rmsnorm_fwd(const at::Tensor& x, const at::Tensor& w, at::Tensor& y, at::Tensor& rstd, double eps,
                        const c10::optional<at::Tensor>& delta, const c10::optional<at::Tensor>& h_out) {
  HM_CHECK(x.is_cuda() && is_bf16(x) && is_bf16(w) && is_bf16(y) && is_f32(rstd) && x.is_contiguous() && y.is_contiguous(), "rmsnorm_fwd: bad tensors");
  const int cols = (int)x.size(-1);
  const int rows = (int)(x.numel() / cols);
  HM_CHECK(rstd.numel() >= rows && w.numel() == cols, "rmsnorm_fwd: shape mismatch");
  HM_CHECK(delta.has_value() == h_out.has_value(), "rmsnorm_fwd: delta and h_out go together");
  if (delta.has_value())
    HM_CHECK(is_bf16(*delta) && is_bf16(*h_out) && delta->is_contiguous() && h_out->is_contiguous() &&
                 delta->numel() == x.numel() && h_out->numel() == x.numel(), "rmsnorm_fwd: bad delta / h_out");
  const c10::cuda::CUDAGuard guard(x.device());
  himuon::rmsnorm_fwd(x.data_ptr(), w.data_ptr(), y.data_ptr(), rstd.data_ptr<float>(), rows, cols, (float)eps, cur_stream(),
                      delta.has_value() ? delta->data_ptr() : nullptr, h_out.has_value() ? h_out->data_ptr() : nullptr);
}
static void rmsnorm_bwd(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const at::Tensor& rstd,
                        at::Tensor& dx, at::Tensor& dw_accum, const c10::optional<at::Tensor>& dres) {
  if (dres.has_value())
    HM_CHECK(is_bf16(*dres) && dres->is_contiguous() && dres->numel() == x.numel(), "rmsnorm_bwd: bad residual gradient");
  HM_CHECK(dy.is_cuda() && is_bf16(dy) && is_bf16(x) && is_bf16(w) && is_bf16(dx) && is_f32(dw_accum) && dy.is_contiguous() && x.is_contiguous() && dx.is_contiguous(), "rmsnorm_bwd: bad tensors");
  const int cols = (int)x.size(-1);
  const int rows = (int)(x.numel() / cols);
  HM_CHECK(dw_accum.numel() == cols, "rmsnorm_bwd: dw_accum must have one fp32 per column");
  const c10::cuda::CUDAGuard guard(x.device());
  himuon::rmsnorm_bwd(dy.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dx.data_ptr(), dw_accum.data_ptr<float>(), rows, cols, cur_stream(),
                      dres.has_value() ? dres->data_ptr() : nullptr);
}
// x, y: (tokens, heads*128) views with unit inner stride and row stride ld
static void headnorm_rope_fwd(const at::Tensor& x, const c10::optional<at::Tensor>& w, at::Tensor& y,
                              const c10::optional<at::Tensor>& rstd, const at::Tensor& cos_sin, int64_t heads,
                              int64_t seq_len, double eps) {
  HM_CHECK(x.is_cuda() && is_bf16(x) && is_bf16(y) && x.dim() == 2 && y.dim() == 2 && x.stride(1) == 1 && y.stride(1) == 1, "headnorm_rope_fwd: bad tensors");
  HM_CHECK(heads > 0 && (x.size(1) == heads * 128 || x.size(1) == heads * 64) && y.sizes() == x.sizes(), "headnorm_rope_fwd: head_dim must be 64 or 128");
  const int64_t hd = x.size(1) / heads;
  HM_CHECK(is_f32(cos_sin) && cos_sin.is_contiguous() && cos_sin.numel() >= seq_len * hd, "headnorm_rope_fwd: bad rope table");
  HM_CHECK(x.stride(0) % 8 == 0 && y.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0,
           "headnorm_rope_fwd: rows must start on 16-byte boundaries");
  const bool use_norm = w.has_value();
  if (use_norm) HM_CHECK(rstd.has_value() && rstd->numel() >= x.size(0) * heads && is_bf16(*w) && w->numel() == hd, "headnorm_rope_fwd: norm needs weight[head_dim] and rstd");
  const c10::cuda::CUDAGuard guard(x.device());
  himuon::headnorm_rope_fwd(x.data_ptr(), use_norm ? w->data_ptr() : nullptr, y.data_ptr(), use_norm ? rstd->data_ptr<float>() : nullptr,
                            cos_sin.data_ptr<float>(), (int)x.size(0), (int)heads, (int)hd, (int)seq_len, x.stride(0), y.stride(0), (float)eps,
                            use_norm ? 1 : 0, cur_stream());
}
static void headnorm_rope_bwd(const at::Tensor& dy, const c10::optional<at::Tensor>& x, const c10::optional<at::Tensor>& w,
                              const c10::optional<at::Tensor>& rstd, at::Tensor& dx, const c10::optional<at::Tensor>& dw_accum,
                              const at::Tensor& cos_sin, int64_t heads, int64_t seq_len) {
  HM_CHECK(dy.is_cuda() && is_bf16(dy) && is_bf16(dx) && dy.dim() == 2 && dx.dim() == 2 && dy.stride(1) == 1 && dx.stride(1) == 1, "headnorm_rope_bwd: bad tensors");
  HM_CHECK(heads > 0 && (dy.size(1) == heads * 128 || dy.size(1) == heads * 64) && dx.sizes() == dy.sizes() &&
               (!x.has_value() || x->sizes() == dy.sizes()), "headnorm_rope_bwd: head_dim must be 64 or 128");
  const int64_t hd = dy.size(1) / heads;
  HM_CHECK(is_f32(cos_sin) && cos_sin.is_contiguous() && cos_sin.numel() >= seq_len * hd, "headnorm_rope_bwd: bad rope table");
  HM_CHECK(dy.stride(0) % 8 == 0 && dx.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(dx.data_ptr()) % 16 == 0 &&
               (!x.has_value() || (x->stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0)),
           "headnorm_rope_bwd: rows must start on 16-byte boundaries");
  const bool use_norm = w.has_value();
  if (use_norm) HM_CHECK(x.has_value() && rstd.has_value() && dw_accum.has_value() && is_f32(*dw_accum) && dw_accum->numel() == hd && w->numel() == hd && x->stride(1) == 1, "headnorm_rope_bwd: norm needs x, rstd, dw_accum");
  const c10::cuda::CUDAGuard guard(dy.device());
  himuon::headnorm_rope_bwd(dy.data_ptr(), use_norm ? x->data_ptr() : nullptr, use_norm ? w->data_ptr() : nullptr,
                            use_norm ? rstd->data_ptr<float>() : nullptr, dx.data_ptr(), use_norm ? dw_accum->data_ptr<float>() : nullptr,
                            cos_sin.data_ptr<float>(), (int)dy.size(0), (int)heads, (int)hd, (int)seq_len, dy.stride(0),
                            use_norm ? x->stride(0) : 0, dx.stride(0), use_norm ? 1 : 0, cur_stream());
}
static void swiglu_fwd(const at::Tensor& gate, const at::Tensor& up, at::Tensor& out) {
  HM_CHECK(gate.is_cuda() && is_bf16(gate) && is_bf16(up) && is_bf16(out) && gate.dim() == 2 && up.dim() == 2 && out.dim() == 2, "swiglu_fwd: 2-D bf16 tensors");
  HM_CHECK(gate.stride(1) == 1 && up.stride(1) == 1 && out.stride(1) == 1 && gate.sizes() == up.sizes() && gate.sizes() == out.sizes(), "swiglu_fwd: shape/stride mismatch");
  const c10::cuda::CUDAGuard guard(gate.device());
  himuon::swiglu_fwd(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.size(0), (int)gate.size(1), gate.stride(0), up.stride(0), out.stride(0), cur_stream());
}
static void swiglu_bwd(const at::Tensor& dout, const at::Tensor& gate, const at::Tensor& up, at::Tensor& dgate, at::Tensor& dup) {
  HM_CHECK(dout.is_cuda() && is_bf16(dout) && is_bf16(gate) && is_bf16(up) && is_bf16(dgate) && is_bf16(dup), "swiglu_bwd: bf16 tensors");
  HM_CHECK(dout.stride(1) == 1 && gate.stride(1) == 1 && up.stride(1) == 1 && dgate.stride(1) == 1 && dup.stride(1) == 1, "swiglu_bwd: unit inner strides");
  HM_CHECK(dout.sizes() == gate.sizes() && gate.sizes() == up.sizes() && dgate.sizes() == gate.sizes() && dup.sizes() == gate.sizes(), "swiglu_bwd: shape mismatch");
  const c10::cuda::CUDAGuard guard(gate.device());
  himuon::swiglu_bwd(dout.data_ptr(), gate.data_ptr(), up.data_ptr(), dgate.data_ptr(), dup.data_ptr(), gate.size(0), (int)gate.size(1),
                     dout.stride(0), gate.stride(0), up.stride(0), dgate.stride(0), dup.stride(0), cur_stream());
}
static void embedding_fwd(const at::Tensor& ids, const at::Tensor& table, at::Tensor& out) {
  HM_CHECK(ids.is_cuda() && ids.scalar_type() == at::kLong && ids.is_contiguous() && is_bf16(table) && table.is_contiguous() && is_bf16(out) && out.is_contiguous(), "embedding_fwd: bad tensors");
  HM_CHECK(out.numel() == ids.numel() * table.size(1), "embedding_fwd: output shape");
  const c10::cuda::CUDAGuard guard(ids.device());
  himuon::embedding_fwd(ids.data_ptr<int64_t>() ? reinterpret_cast<const long long*>(ids.data_ptr<int64_t>()) : nullptr, table.data_ptr(), out.data_ptr(), ids.numel(), (int)table.size(1), cur_stream());
}
static void embedding_bwd(const at::Tensor& ids, const at::Tensor& dout, at::Tensor& dtable) {
  HM_CHECK(ids.is_cuda() && ids.scalar_type() == at::kLong && ids.is_contiguous() && is_bf16(dout) && dout.is_contiguous() && dtable.is_contiguous() && (is_bf16(dtable) || is_f32(dtable)), "embedding_bwd: bad tensors");
  HM_CHECK(dtable.size(1) % 2 == 0 && dout.numel() == ids.numel() * dtable.size(1), "embedding_bwd: shapes");
  const c10::cuda::CUDAGuard guard(ids.device());
  himuon::embedding_bwd(reinterpret_cast<const long long*>(ids.data_ptr<int64_t>()), dout.data_ptr(), dtable.data_ptr(), ids.numel(), (int)dtable.size(1), is_f32(dtable) ? 1 : 0, cur_stream());
}
static void cross_entropy(at::Tensor& logits, const at::Tensor& labels, at::Tensor& loss_sum, at::Tensor& count,
                          const c10::optional<at::Tensor>& lse, double grad_scale,
                          const c10::optional<at::Tensor>& scale_dev, int64_t ignore_index) {
  HM_CHECK(logits.is_cuda() && is_bf16(logits) && logits.dim() == 2 && logits.stride(1) == 1, "cross_entropy: logits must be 2-D bf16");
  HM_CHECK(labels.scalar_type() == at::kLong && labels.is_contiguous() && labels.numel() == logits.size(0), "cross_entropy: labels");
  HM_CHECK(is_f32(loss_sum) && is_f32(count), "cross_entropy: accumulators must be fp32");
  if (scale_dev.has_value()) HM_CHECK(scale_dev->is_cuda() && is_f32(*scale_dev) && scale_dev->numel() == 1, "cross_entropy: scale_dev must be one fp32 on the device");
  const c10::cuda::CUDAGuard guard(logits.device());
  himuon::cross_entropy_fwd_bwd(logits.data_ptr(), reinterpret_cast<const long long*>(labels.data_ptr<int64_t>()), loss_sum.data_ptr<float>(),
                                count.data_ptr<float>(), lse.has_value() ? lse->data_ptr<float>() : nullptr, logits.size(0),
                                (int)logits.size(1), logits.stride(0), (float)grad_scale,
                                scale_dev.has_value() ? scale_dev->data_ptr<float>() : nullptr, ignore_index, cur_stream());
}

static void flash_attn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& o, at::Tensor& lse,
                           int64_t B, int64_t S, int64_t Hq, int64_t Hkv, double scale) {
  HM_CHECK(q.is_cuda() && is_bf16(q) && is_bf16(k) && is_bf16(v) && is_bf16(o) && is_f32(lse), "flash_attn_fwd: dtypes");
  HM_CHECK(q.dim() == 2 && k.dim() == 2 && v.dim() == 2 && o.dim() == 2, "flash_attn_fwd: (tokens, heads*head_dim) views expected");
  HM_CHECK(Hq > 0 && Hkv > 0, "flash_attn_fwd: heads");
  const int64_t hd = q.size(1) / Hq;
  HM_CHECK(q.size(0) == B * S && q.size(1) == Hq * hd && k.size(1) == Hkv * hd && v.size(1) == Hkv * hd && o.size(1) == Hq * hd &&
               k.size(0) >= B * S && v.size(0) >= B * S && o.size(0) >= B * S, "flash_attn_fwd: shapes");
  HM_CHECK(q.stride(1) == 1 && k.stride(1) == 1 && v.stride(1) == 1 && o.stride(1) == 1, "flash_attn_fwd: unit inner strides");
  HM_CHECK(Hq % Hkv == 0 && lse.numel() >= B * Hq * S, "flash_attn_fwd: heads / lse size");
  const c10::cuda::CUDAGuard guard(q.device());
  himuon::AttnArgs a{};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.o = o.data_ptr(); a.lse = lse.data_ptr<float>();
  a.B = (int)B; a.S = (int)S; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.hd = (int)hd;
  a.ld_q = q.stride(0); a.ld_k = k.stride(0); a.ld_v = v.stride(0); a.ld_o = o.stride(0);
  a.scale = (float)scale;
  himuon::flash_attn_fwd(a, cur_stream());
}
static void flash_attn_bwd(const at::Tensor& d_o, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                           const at::Tensor& o, const at::Tensor& lse, at::Tensor& dq, at::Tensor& dk, at::Tensor& dv,
                           at::Tensor& delta, const c10::optional<at::Tensor>& dkv_part, int64_t B, int64_t S, int64_t Hq,
                           int64_t Hkv, double scale) {
  HM_CHECK(q.is_cuda() && is_bf16(q) && is_bf16(k) && is_bf16(v) && is_bf16(o) && is_bf16(d_o) && is_bf16(dq) && is_bf16(dk) && is_bf16(dv) && is_f32(lse) && is_f32(delta), "flash_attn_bwd: dtypes");
  HM_CHECK(q.stride(1) == 1 && k.stride(1) == 1 && v.stride(1) == 1 && o.stride(1) == 1 && d_o.stride(1) == 1 && dq.stride(1) == 1 && dk.stride(1) == 1 && dv.stride(1) == 1, "flash_attn_bwd: unit inner strides");
  HM_CHECK(Hq > 0 && Hkv > 0, "flash_attn_bwd: heads");
  const int64_t hd = q.size(1) / Hq;
  HM_CHECK(q.size(0) == B * S && q.size(1) == Hq * hd && k.size(1) == Hkv * hd && v.size(1) == Hkv * hd && delta.numel() >= B * Hq * S &&
               lse.numel() >= B * Hq * S && o.size(1) == Hq * hd && d_o.size(1) == Hq * hd && dq.size(1) == Hq * hd &&
               dk.size(1) == Hkv * hd && dv.size(1) == Hkv * hd, "flash_attn_bwd: shapes");
  for (const at::Tensor* t : {&k, &v, &o, &d_o, static_cast<const at::Tensor*>(&dq), static_cast<const at::Tensor*>(&dk), static_cast<const at::Tensor*>(&dv)})
    HM_CHECK(t->size(0) >= B * S, "flash_attn_bwd: too few tokens");
  const c10::cuda::CUDAGuard guard(q.device());
  himuon::AttnArgs a{};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.o = const_cast<void*>(o.data_ptr()); a.lse = lse.data_ptr<float>();
  a.d_o = d_o.data_ptr(); a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr(); a.delta = delta.data_ptr<float>();
  a.B = (int)B; a.S = (int)S; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.hd = (int)hd;
  a.ld_q = q.stride(0); a.ld_k = k.stride(0); a.ld_v = v.stride(0); a.ld_o = o.stride(0); a.ld_do = d_o.stride(0);
  a.ld_dq = dq.stride(0); a.ld_dk = dk.stride(0); a.ld_dv = dv.stride(0);
  if (dkv_part.has_value()) {
    const at::Tensor& t = dkv_part.value();     // (2, B*S, Hq*head_dim): per-query-head dK and dV
    HM_CHECK(t.is_cuda() && is_bf16(t) && t.is_contiguous() && t.dim() == 3 && t.size(0) == 2 && t.size(1) == B * S && t.size(2) == Hq * hd,
             "flash_attn_bwd: dkv_part must be a contiguous (2, B*S, Hq*head_dim) bf16 tensor");
    a.dk_part = t.data_ptr();
    a.dv_part = static_cast<char*>(t.data_ptr()) + t.stride(0) * 2;
    a.ld_part = t.stride(1);
  }
  a.scale = (float)scale;
  himuon::flash_attn_bwd(a, cur_stream());
}

// `plan`: (2 * tiles + pairs, 4) int32, the batch's tiles in their three orders (himuon.h); its entries are bounded by the caller, which
// makes them from the lengths on the host (`tokens` of them).
static himuon::PackedAttnArgs packed_attn_args(const char* op, const at::Tensor& plan, int64_t tiles, int64_t tokens, const at::Tensor& q, const at::Tensor& k,
                                               const at::Tensor& v, const at::Tensor& o, const c10::optional<at::Tensor>& lse, int64_t Hq, int64_t Hkv, double scale) {
  const std::string at = std::string("himuon: ") + op;
  TORCH_CHECK(Hq > 0 && Hkv > 0 && Hq % Hkv == 0, at, ": heads");
  TORCH_CHECK(q.dim() == 2 && q.size(1) % Hq == 0, at, ": (tokens, heads*head_dim) views expected");
  const int64_t T = q.size(0), hd = q.size(1) / Hq;
  TORCH_CHECK(hd > 0 && hd % 8 == 0 && hd <= 128, at, ": head_dim must be a multiple of 8 up to 128");
  TORCH_CHECK(T > 0 && T < (1LL << 30) && tokens >= 0 && tokens <= T, at, ": fewer rows than the layout has tokens");
  TORCH_CHECK(plan.device() == q.device() && plan.scalar_type() == at::kInt && plan.is_contiguous() && plan.dim() == 2 && plan.size(1) == 4 && tiles >= 0 &&
                  tiles < (1LL << 28) && plan.size(0) >= 2 * tiles && plan.size(0) <= 3 * tiles && reinterpret_cast<uintptr_t>(plan.data_ptr()) % 16 == 0,
              at, ": the plan must be a contiguous (2 * tiles + pairs, 4) int32 tensor on the device of q");
  himuon::PackedAttnArgs a{};
  a.n_tiles = static_cast<int>(tiles);
  a.n_pairs = static_cast<int>(plan.size(0) - 2 * tiles);
  a.by_keys = reinterpret_cast<const himuon::PackedTile*>(plan.data_ptr<int>());
  a.by_queries = a.by_keys + a.n_tiles;
  a.pairs = a.by_queries + a.n_tiles;
  a.tokens = static_cast<int>(tokens);
  a.rows = static_cast<int>(T); a.Hq = static_cast<int>(Hq); a.Hkv = static_cast<int>(Hkv); a.hd = static_cast<int>(hd);
  a.scale = static_cast<float>(scale);
  if (lse.has_value()) {
    TORCH_CHECK(is_f32(*lse) && lse->is_contiguous() && lse->device() == q.device() && lse->numel() == Hq * a.n_tiles * 128 &&
                    reinterpret_cast<uintptr_t>(lse->data_ptr()) % 16 == 0, at, ": lse must be fp32, (heads, tiles * 128)");
    a.lse = lse->data_ptr<float>();
  }
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.o = o.data_ptr();
  a.ld_q = q.stride(0); a.ld_k = k.stride(0); a.ld_v = v.stride(0); a.ld_o = o.stride(0);
  return a;
}
static void packed_rows(const char* op, const at::Tensor& t, const at::Tensor& q, int64_t cols) {
  const std::string at = std::string("himuon: ") + op;
  TORCH_CHECK(t.is_cuda() && t.device() == q.device() && is_bf16(t) && t.dim() == 2 && t.size(0) == q.size(0) && t.size(1) == cols && t.stride(1) == 1 &&
                  t.stride(0) % 8 == 0 && (t.size(0) <= 1 || t.stride(0) >= cols) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              at, ": bf16 rows of heads * head_dim columns with unit inner stride, each on a 16-byte boundary, expected");
}
// Bytes of O's low bits: rows of a multiple of 16.
static int64_t packed_low_size(int64_t Hq, int64_t tiles, int64_t hd) { return Hq * tiles * 128 * ((hd + 15) / 16 * 16); }
static signed char* packed_low(const char* op, const at::Tensor& low, const at::Tensor& q, int64_t Hq, int64_t tiles) {
  TORCH_CHECK(low.device() == q.device() && low.scalar_type() == at::kChar && low.is_contiguous() && low.numel() == packed_low_size(Hq, tiles, q.size(1) / Hq) &&
                  reinterpret_cast<uintptr_t>(low.data_ptr()) % 16 == 0, std::string("himuon: ") + op, ": o_low must be int8, (heads, tiles * 128, head_dim rounded up to 16)");
  return reinterpret_cast<signed char*>(low.data_ptr<int8_t>());
}
static void packed_attn_fwd(const at::Tensor& plan, int64_t tiles, int64_t tokens, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            at::Tensor& o, const c10::optional<at::Tensor>& lse, const c10::optional<at::Tensor>& o_low, int64_t Hq, int64_t Hkv, double scale) {
  himuon::PackedAttnArgs a = packed_attn_args("packed_attn_fwd", plan, tiles, tokens, q, k, v, o, lse, Hq, Hkv, scale);
  packed_rows("packed_attn_fwd", q, q, Hq * a.hd); packed_rows("packed_attn_fwd", k, q, Hkv * a.hd);
  packed_rows("packed_attn_fwd", v, q, Hkv * a.hd); packed_rows("packed_attn_fwd", o, q, Hq * a.hd);
  if (o_low.has_value()) a.o_low = packed_low("packed_attn_fwd", *o_low, q, Hq, tiles);
  const c10::cuda::CUDAGuard guard(q.device());
  himuon::packed_attn_fwd(a, cur_stream());
}
static void packed_attn_bwd(const at::Tensor& plan, int64_t tiles, int64_t tokens, const at::Tensor& d_o, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& o, const at::Tensor& lse, const at::Tensor& o_low, at::Tensor& dq, at::Tensor& dk, at::Tensor& dv, at::Tensor& delta,
                            const c10::optional<at::Tensor>& dkv_part, int64_t Hq, int64_t Hkv, double scale) {
  himuon::PackedAttnArgs a = packed_attn_args("packed_attn_bwd", plan, tiles, tokens, q, k, v, o, lse, Hq, Hkv, scale);
  for (const at::Tensor* t : {&q, &o, &d_o, static_cast<const at::Tensor*>(&dq)}) packed_rows("packed_attn_bwd", *t, q, Hq * a.hd);
  for (const at::Tensor* t : {&k, &v, static_cast<const at::Tensor*>(&dk), static_cast<const at::Tensor*>(&dv)}) packed_rows("packed_attn_bwd", *t, q, Hkv * a.hd);
  HM_CHECK(is_f32(delta) && delta.is_contiguous() && delta.device() == q.device() && delta.numel() == lse.numel() &&
               reinterpret_cast<uintptr_t>(delta.data_ptr()) % 16 == 0, "packed_attn_bwd: delta must look like lse");
  a.o_low = packed_low("packed_attn_bwd", o_low, q, Hq, tiles);
  a.d_o = d_o.data_ptr(); a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr(); a.delta = delta.data_ptr<float>();
  a.ld_do = d_o.stride(0); a.ld_dq = dq.stride(0); a.ld_dk = dk.stride(0); a.ld_dv = dv.stride(0);
  if (dkv_part.has_value()) {
    HM_CHECK(is_f32(*dkv_part) && dkv_part->is_contiguous() && dkv_part->device() == q.device() && dkv_part->numel() == 2 * lse.numel() * a.hd &&
                 reinterpret_cast<uintptr_t>(dkv_part->data_ptr()) % 16 == 0, "packed_attn_bwd: dkv_part must be fp32, (2, heads, tiles * 128, head_dim)");
    a.dkv_part = dkv_part->data_ptr<float>();
  }
  const c10::cuda::CUDAGuard guard(q.device());
  himuon::packed_attn_bwd(a, cur_stream());
}

// Autograd functions of calls whose kernels take tens of microseconds are written here and not in Python: a backward pass then runs in
// the engine's thread without waiting for the interpreter.  (Forward and gradients of the packed attention:
// 119 us of host time as a Python function, 88 here, of which a function that does nothing takes 63 and 40.)
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
static std::atomic<int64_t> autograd_launched{0};       // kernels launched by them

static void check_once(const char* op) {
  TORCH_CHECK(!c10::GradMode::is_enabled(), "himuon_b200.ops.", op, ": its gradient cannot be differentiated again (create_graph=True)");
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& plan, int64_t tiles,
                            int64_t tokens, int64_t Hq, int64_t Hkv, double scale, bool split_heads) {
    at::Tensor o = at::empty(q.sizes(), q.options()), lse = at::empty({Hq * tiles * 128}, q.options().dtype(at::kFloat));
    const at::Tensor o_low = at::empty({packed_low_size(Hq, tiles, q.size(1) / Hq)}, q.options().dtype(at::kChar));
    if (tiles) {
      packed_attn_fwd(plan, tiles, tokens, q, k, v, o, lse, o_low, Hq, Hkv, scale);
      autograd_launched += 1;
    } else {
      o.zero_();
    }
    ctx->save_for_backward({q, k, v, o, lse, plan, o_low});
    ctx->saved_data["tiles"] = tiles;
    ctx->saved_data["tokens"] = tokens;
    ctx->saved_data["Hq"] = Hq;
    ctx->saved_data["Hkv"] = Hkv;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["split_heads"] = split_heads;
    return o;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("packed_attention");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4], &plan = saved[5];
    const int64_t tiles = ctx->saved_data["tiles"].toInt(), Hq = ctx->saved_data["Hq"].toInt(), Hkv = ctx->saved_data["Hkv"].toInt(), hd = q.size(1) / Hq;
    at::Tensor d_o = grads[0];
    if (d_o.stride(1) != 1 || d_o.stride(0) % 8 || d_o.stride(0) < d_o.size(1) || reinterpret_cast<uintptr_t>(d_o.data_ptr()) % 16)
      d_o = d_o.clone(at::MemoryFormat::Contiguous);
    // dq | dk | dv share one buffer, as in attention(): a fused projection sees a single contiguous gradient
    at::Tensor all = at::empty({q.size(0), (Hq + 2 * Hkv) * hd}, q.options());
    at::Tensor dq = all.narrow(1, 0, Hq * hd), dk = all.narrow(1, Hq * hd, Hkv * hd), dv = all.narrow(1, (Hq + Hkv) * hd, Hkv * hd);
    if (tiles) {
      at::Tensor delta = at::empty_like(lse);
      c10::optional<at::Tensor> part;
      if (ctx->saved_data["split_heads"].toBool()) part = at::empty({2 * lse.numel() * hd}, lse.options());
      packed_attn_bwd(plan, tiles, ctx->saved_data["tokens"].toInt(), d_o, q, k, v, o, lse, saved[6], dq, dk, dv, delta, part, Hq, Hkv, ctx->saved_data["scale"].toDouble());
      autograd_launched += part.has_value() ? 3 : 2;
    } else {
      all.zero_();
    }
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Checks what the forward and the gradient call share.
static himuon::TokenScoreArgs token_score_args(const char* op, const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& entropy,
                                               int64_t ignore_index) {
  const std::string at = std::string("himuon: ") + op;
  TORCH_CHECK(logits.is_cuda() && (is_bf16(logits) || is_f32(logits)) && logits.dim() == 2 && logits.stride(1) == 1 &&
                  (logits.size(0) <= 1 || logits.stride(0) >= logits.size(1)), at, ": (rows, vocab) bf16 or fp32 logits with unit inner stride");
  TORCH_CHECK(logits.size(1) > 0 && logits.size(1) < (1LL << 31), at, ": bad vocabulary");
  TORCH_CHECK(ids.device() == logits.device() && ids.scalar_type() == at::kLong && ids.is_contiguous() && ids.numel() == logits.size(0), at, ": one int64 id for each row");
  TORCH_CHECK(entropy.device() == logits.device() && is_f32(entropy) && entropy.is_contiguous() && entropy.numel() == logits.size(0), at, ": entropy must be fp32, one for each row");
  himuon::TokenScoreArgs a{};
  a.logits = logits.data_ptr(); a.logits_fp32 = is_f32(logits) ? 1 : 0;
  a.ids = reinterpret_cast<const long long*>(ids.data_ptr<int64_t>()); a.ignore = ignore_index;
  a.rows = logits.size(0); a.ld = logits.stride(0); a.vocab = static_cast<int>(logits.size(1));
  a.entropy = entropy.data_ptr<float>();
  return a;
}
static void token_scores_fwd(const at::Tensor& logits, const at::Tensor& ids, at::Tensor& log_probs, at::Tensor& entropy,
                             const c10::optional<at::Tensor>& stats, const c10::optional<at::Tensor>& top_log_probs,
                             const c10::optional<at::Tensor>& top_ids, int64_t ignore_index) {
  himuon::TokenScoreArgs a = token_score_args("token_scores_fwd", logits, ids, entropy, ignore_index);
  HM_CHECK(log_probs.device() == logits.device() && is_f32(log_probs) && log_probs.is_contiguous() && log_probs.numel() == a.rows, "token_scores_fwd: log_probs must be fp32, one for each row");
  a.log_probs = log_probs.data_ptr<float>();
  if (stats.has_value()) {
    HM_CHECK(stats->device() == logits.device() && is_f32(*stats) && stats->is_contiguous() && stats->numel() == 2 * a.rows, "token_scores_fwd: stats must be fp32, two for each row");
    a.stats = stats->data_ptr<float>();
  }
  HM_CHECK(top_log_probs.has_value() == top_ids.has_value(), "token_scores_fwd: alternatives need values and ids");
  if (top_ids.has_value()) {
    HM_CHECK(top_ids->device() == logits.device() && top_log_probs->device() == logits.device() && top_ids->scalar_type() == at::kLong &&
                 is_f32(*top_log_probs) && top_ids->is_contiguous() && top_log_probs->is_contiguous() && top_ids->dim() == 2 &&
                 top_ids->size(0) == a.rows && top_log_probs->sizes() == top_ids->sizes() && top_ids->size(1) > 0 &&
                 top_ids->size(1) <= himuon::kTopMax && top_ids->size(1) <= a.vocab,
             "token_scores_fwd: alternatives must be (rows, 1..32) fp32 values and int64 ids");
    a.top_k = static_cast<int>(top_ids->size(1));
    a.top_log_probs = top_log_probs->data_ptr<float>();
    a.top_ids = reinterpret_cast<long long*>(top_ids->data_ptr<int64_t>());
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  himuon::token_scores_fwd(a, cur_stream());
}
static void token_scores_bwd(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& entropy, const at::Tensor& stats,
                             const c10::optional<at::Tensor>& g_log_probs, const c10::optional<at::Tensor>& g_entropy, at::Tensor& grad,
                             int64_t ignore_index) {
  himuon::TokenScoreArgs a = token_score_args("token_scores_bwd", logits, ids, entropy, ignore_index);
  HM_CHECK(stats.device() == logits.device() && is_f32(stats) && stats.is_contiguous() && stats.numel() == 2 * a.rows, "token_scores_bwd: stats must be fp32, two for each row");
  HM_CHECK(grad.device() == logits.device() && grad.dim() == 2 && grad.sizes() == logits.sizes() && grad.stride(1) == 1 && (is_bf16(grad) || is_f32(grad)) &&
               (grad.size(0) <= 1 || grad.stride(0) >= grad.size(1)), "token_scores_bwd: the gradient has the shape of the logits");
  for (const auto* g : {&g_log_probs, &g_entropy})
    if (g->has_value()) HM_CHECK((*g)->device() == logits.device() && is_f32(**g) && (*g)->is_contiguous() && (*g)->numel() == a.rows, "token_scores_bwd: incoming gradients must be fp32, one for each row");
  a.stats = stats.data_ptr<float>();
  a.g_log_probs = g_log_probs.has_value() ? g_log_probs->data_ptr<float>() : nullptr;
  a.g_entropy = g_entropy.has_value() ? g_entropy->data_ptr<float>() : nullptr;
  a.grad = grad.data_ptr(); a.grad_fp32 = is_f32(grad) ? 1 : 0; a.ld_grad = grad.stride(0);
  const c10::cuda::CUDAGuard guard(logits.device());
  himuon::token_scores_bwd(a, cur_stream());
}

// Outputs of a call: log probabilities, entropy, and values and ids of alternatives where there are any.
static variable_list score_outputs(const at::Tensor& logits, const at::Tensor& ids, int64_t top_k, int64_t ignore_index, const c10::optional<at::Tensor>& stats) {
  const int64_t rows = logits.size(0);
  const auto fp32 = logits.options().dtype(at::kFloat);
  variable_list out = {at::empty({rows}, fp32), at::empty({rows}, fp32)};
  c10::optional<at::Tensor> top_log_probs, top_ids;
  if (top_k) {
    top_log_probs = at::empty({rows, top_k}, fp32);
    top_ids = at::empty({rows, top_k}, ids.options());
    out.push_back(*top_log_probs);
    out.push_back(*top_ids);
  }
  if (rows) {
    token_scores_fwd(logits, ids, out[0], out[1], stats, top_log_probs, top_ids, ignore_index);
    autograd_launched += 1;
  }
  return out;
}

struct TokenScores : torch::autograd::Function<TokenScores> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids, int64_t top_k, int64_t ignore_index) {
    ctx->set_materialize_grads(false);                   // the gradient of an unused output arrives undefined
    const at::Tensor stats = at::empty({logits.size(0), 2}, logits.options().dtype(at::kFloat));
    variable_list out = score_outputs(logits, ids, top_k, ignore_index, stats);
    ctx->save_for_backward({logits, ids, out[1], stats});
    ctx->saved_data["ignore_index"] = ignore_index;
    if (top_k) ctx->mark_non_differentiable({out[2], out[3]});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("token_log_probs");
    at::Tensor grad;
    if (grads[0].defined() || grads[1].defined()) {
      const variable_list saved = ctx->get_saved_variables();
      grad = at::empty(saved[0].sizes(), saved[0].options());
      c10::optional<at::Tensor> g[2];
      for (int i = 0; i < 2; ++i)
        if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).contiguous();
      if (grad.numel()) {
        token_scores_bwd(saved[0], saved[1], saved[2], saved[3], g[0], g[1], grad, ctx->saved_data["ignore_index"].toInt());
        autograd_launched += 1;
      }
    }
    return {grad, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

static himuon::LinearScoreArgs linear_score_args(const char* op, const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, const at::Tensor& entropy,
                                                 const c10::optional<at::Tensor>& stats, int64_t ignore_index) {
  const std::string at = std::string("himuon: ") + op;
  TORCH_CHECK(h.is_cuda() && w.device() == h.device() && is_bf16(h) && is_bf16(w) && h.dim() == 2 && w.dim() == 2 && h.size(1) == w.size(1), at, ": (rows, hidden) and (vocab, hidden) bf16 expected");
  TORCH_CHECK(h.size(0) > 0 && w.size(0) > 0 && h.size(1) > 0 && h.size(1) % 8 == 0 && h.size(0) < (1LL << 30) && w.size(0) < (1LL << 30) && h.size(1) < (1LL << 30),
              at, ": rows, vocabulary and a hidden size of a multiple of 8 expected");
  for (const at::Tensor* t : {&h, &w})
    TORCH_CHECK(t->stride(1) == 1 && t->stride(0) % 8 == 0 && (t->size(0) <= 1 || t->stride(0) >= t->size(1)) && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                at, ": rows must have unit inner stride and start on 16-byte boundaries");
  TORCH_CHECK(ids.device() == h.device() && ids.scalar_type() == at::kLong && ids.is_contiguous() && ids.numel() == h.size(0), at, ": one int64 id for each row");
  TORCH_CHECK(entropy.device() == h.device() && is_f32(entropy) && entropy.is_contiguous() && entropy.numel() == h.size(0), at, ": entropy must be fp32, one for each row");
  himuon::LinearScoreArgs a{};
  a.h = h.data_ptr(); a.w = w.data_ptr(); a.ld_h = h.stride(0); a.ld_w = w.stride(0);
  a.rows = static_cast<int>(h.size(0)); a.hidden = static_cast<int>(h.size(1)); a.vocab = static_cast<int>(w.size(0));
  a.ids = reinterpret_cast<const long long*>(ids.data_ptr<int64_t>()); a.ignore = ignore_index;
  a.entropy = entropy.data_ptr<float>();
  if (stats.has_value()) {
    TORCH_CHECK(stats->device() == h.device() && is_f32(*stats) && stats->is_contiguous() && stats->numel() == 2 * a.rows, at, ": stats must be fp32, two for each row");
    a.stats = stats->data_ptr<float>();
  }
  return a;
}
// Kept exponentials or the gradient of the logits, and the maxima that belong to the former: `slab_max` (rows, vocab / 64 rounded up).
static void linear_score_kept(const char* op, himuon::LinearScoreArgs& a, const at::Tensor& h, const at::Tensor& kept, const c10::optional<at::Tensor>& slab_max) {
  const std::string at = std::string("himuon: ") + op;
  // (whole 16-byte groups of columns are written: the row stride covers them)
  TORCH_CHECK(kept.device() == h.device() && is_bf16(kept) && kept.dim() == 2 && kept.size(0) == a.rows && kept.size(1) == (a.vocab + 7) / 8 * 8 && kept.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(kept.data_ptr()) % 16 == 0, at, ": the gradient must be contiguous bf16, its columns rounded up to a multiple of 8");
  a.grad = kept.data_ptr(); a.ld_grad = kept.stride(0);
  if (slab_max.has_value()) {
    TORCH_CHECK(slab_max->device() == h.device() && is_f32(*slab_max) && slab_max->dim() == 2 && slab_max->size(0) == a.rows && slab_max->size(1) == (a.vocab + 63) / 64 &&
                    slab_max->is_contiguous(), at, ": slab_max must be fp32, (rows, vocab / 64 rounded up)");
    a.slab_max = slab_max->data_ptr<float>();
  }
}
static void linear_scores_fwd(const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, at::Tensor& log_probs, at::Tensor& entropy,
                              const c10::optional<at::Tensor>& stats, at::Tensor& scratch, int64_t ignore_index, const c10::optional<at::Tensor>& kept,
                              const c10::optional<at::Tensor>& slab_max) {
  himuon::LinearScoreArgs a = linear_score_args("linear_scores_fwd", h, w, ids, entropy, stats, ignore_index);
  HM_CHECK(log_probs.device() == h.device() && is_f32(log_probs) && log_probs.is_contiguous() && log_probs.numel() == a.rows, "linear_scores_fwd: log_probs must be fp32, one for each row");
  HM_CHECK(scratch.device() == h.device() && is_f32(scratch) && scratch.is_contiguous() && scratch.numel() >= himuon::linear_scores_scratch(a.rows, a.vocab), "linear_scores_fwd: scratch too small");
  a.log_probs = log_probs.data_ptr<float>();
  a.scratch = scratch.data_ptr<float>();
  HM_CHECK(kept.has_value() == slab_max.has_value(), "linear_scores_fwd: kept exponentials need their maxima");
  if (kept.has_value()) linear_score_kept("linear_scores_fwd", a, h, *kept, slab_max);
  const c10::cuda::CUDAGuard guard(h.device());
  himuon::linear_scores_fwd(a, cur_stream());
}
static void linear_scores_dlogits(const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, const at::Tensor& entropy, const at::Tensor& stats,
                                  const c10::optional<at::Tensor>& g_log_probs, const c10::optional<at::Tensor>& g_entropy, at::Tensor& grad,
                                  const c10::optional<at::Tensor>& kept, const c10::optional<at::Tensor>& slab_max, int64_t ignore_index) {
  himuon::LinearScoreArgs a = linear_score_args("linear_scores_dlogits", h, w, ids, entropy, stats, ignore_index);
  for (const auto* g : {&g_log_probs, &g_entropy})
    if (g->has_value()) HM_CHECK((*g)->device() == h.device() && is_f32(**g) && (*g)->is_contiguous() && (*g)->numel() == a.rows, "linear_scores_dlogits: incoming gradients must be fp32, one for each row");
  if (kept.has_value()) {
    linear_score_kept("linear_scores_dlogits", a, h, *kept, slab_max);
    a.kept = a.grad;
  }
  linear_score_kept("linear_scores_dlogits", a, h, grad, slab_max);
  a.g_log_probs = g_log_probs.has_value() ? g_log_probs->data_ptr<float>() : nullptr;
  a.g_entropy = g_entropy.has_value() ? g_entropy->data_ptr<float>() : nullptr;
  const c10::cuda::CUDAGuard guard(h.device());
  himuon::linear_scores_dlogits(a, cur_stream());
}

static void sum_parts(const at::Tensor& parts, at::Tensor& out) {
  HM_CHECK(parts.is_cuda() && is_f32(parts) && parts.is_contiguous() && parts.dim() == out.dim() + 1 && out.device() == parts.device() && is_bf16(out) && out.is_contiguous() &&
               parts.numel() == parts.size(0) * out.numel() && out.numel() % 4 == 0 && reinterpret_cast<uintptr_t>(parts.data_ptr()) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(out.data_ptr()) % 8 == 0, "sum_parts: contiguous fp32 parts of a contiguous bf16 output expected");
  const c10::cuda::CUDAGuard guard(parts.device());
  himuon::sum_parts(parts.data_ptr<float>(), out.data_ptr(), out.numel(), (int)parts.size(0), cur_stream());
}

// out = a b, for a long inner dimension and few output tiles: cut along it into batches whose fp32 results are added up.
// A GEMM's time goes by its rounds of tiles over the SMs, and the cut fills them: 777 x 128256 x 640, 12 tiles of 256 x 256
// on 74 CTA pairs, 130 us in 6 cuts against 567 whole; the fp32 results are what a cut costs.
static void long_product(const at::Tensor& a, const at::Tensor& b, at::Tensor& out) {
  const int64_t rows = a.size(0), inner = a.size(1), cols = b.size(1);
  const bool pairs = rows > 128 && cols > 192;
  const int64_t slots = pairs ? himuon::num_sms() / 2 : himuon::num_sms(), tile = pairs ? 256 : 128;
  const int64_t tiles = (rows + tile - 1) / tile * ((cols + 255) / 256);
  int64_t cuts = 1;
  if (tiles < 4 * slots && inner >= 8192) {
    const double unit = tile * 256.0 * 2 * inner / (1.4e15 / slots);                 // seconds of one tile, whole
    double best = 0;
    for (int64_t c = 1; c <= std::min<int64_t>(16, inner / 4096); ++c) {
      double rounds = static_cast<double>((tiles * c + slots - 1) / slots) / c;
      if (c == 1 && pairs && tiles > slots / 2 && tiles % slots > 0 && tiles % slots <= slots / 2)
        rounds = static_cast<double>(tiles) / slots;                                 // (the GEMM cuts such a last round itself)
      const double cost = rounds * unit + (c > 1 ? 8.0 * c * rows * cols / 6e12 + 8e-6 : 0.0);
      if (c == 1 || cost < best) { best = cost; cuts = c; }
    }
  }
  if (cuts == 1) {
    gemm(a, b, out, c10::nullopt, false, false, 1.0, 0.0, false, 0, false);
    autograd_launched += 1;
    return;
  }
  const int64_t step = inner / cuts / 64 * 64, rest = inner - cuts * step;
  const at::Tensor parts = at::empty({cuts + (rest > 0), rows, cols}, a.options().dtype(at::kFloat));
  at::Tensor whole = parts.narrow(0, 0, cuts);
  gemm(a.as_strided({cuts, rows, step}, {step, a.stride(0), 1}), b.as_strided({cuts, step, cols}, {step * b.stride(0), b.stride(0), 1}), whole, c10::nullopt,
       false, false, 1.0, 0.0, false, 0, false);
  if (rest) {
    at::Tensor last = parts.select(0, cuts);
    gemm(a.narrow(1, cuts * step, rest), b.narrow(0, cuts * step, rest), last, c10::nullopt, false, false, 1.0, 0.0, false, 0, false);
  }
  sum_parts(parts, out);
  autograd_launched += 2 + (rest > 0);
}

// Log probabilities and entropy, `launch_rows` rows at a time: their hidden states stay in the L2 while the weight streams by.
static variable_list linear_score_outputs(const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, int64_t ignore_index, int64_t launch_rows,
                                          const c10::optional<at::Tensor>& stats, const c10::optional<at::Tensor>& kept, const c10::optional<at::Tensor>& slab_max) {
  const int64_t rows = h.size(0);
  const auto fp32 = h.options().dtype(at::kFloat);
  variable_list out = {at::empty({rows}, fp32), at::empty({rows}, fp32)};
  if (!rows) return out;
  // a rest that the kernel for a few rows would take goes along with the launch before: its order of sums is another, and no result may depend
  // on the launch that a row is in
  auto of_launch = [&](int64_t r) { return rows - r <= launch_rows + himuon::kFewRows ? rows - r : launch_rows; };
  const int64_t rest = rows % launch_rows, most = std::max(of_launch(0), rows > launch_rows && rest <= himuon::kFewRows ? launch_rows + rest : 0);
  at::Tensor scratch = at::empty({himuon::linear_scores_scratch(most, static_cast<int>(w.size(0)))}, fp32);
  int64_t n;
  for (int64_t r = 0; r < rows; r += n) {
    n = of_launch(r);
    auto chunk = [&](const at::Tensor& t) { return n == rows ? t : t.narrow(0, r, n); };
    auto maybe = [&](const c10::optional<at::Tensor>& t) { return t.has_value() ? c10::optional<at::Tensor>(chunk(*t)) : c10::nullopt; };
    at::Tensor log_probs = chunk(out[0]), entropy = chunk(out[1]);
    linear_scores_fwd(chunk(h), w, chunk(ids), log_probs, entropy, maybe(stats), scratch, ignore_index, maybe(kept), maybe(slab_max));
    autograd_launched += 2;
  }
  return out;
}

// The backward pass multiplies the logits' gradient with both operands.  It gets it from the exponentials that the forward pass kept, in
// their place (one that a graph captures, elsewhere); where there are none (more than `gradient_values`, a few rows, whose kernel keeps nothing, or used up by an earlier backward
// pass) it makes the logits again, for as many rows at a time as that allows.
struct LinearScores : torch::autograd::Function<LinearScores> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, int64_t ignore_index, int64_t launch_rows,
                               int64_t gradient_values) {
    ctx->set_materialize_grads(false);
    const int64_t rows = h.size(0), vocab = w.size(0), cols = (vocab + 7) / 8 * 8;
    const auto fp32 = h.options().dtype(at::kFloat);
    const at::Tensor stats = at::empty({rows, 2}, fp32);
    c10::optional<at::Tensor> kept, slab_max;
    if (rows > himuon::kFewRows && rows * cols <= gradient_values) {
      kept = at::empty({rows, cols}, h.options());
      slab_max = at::empty({rows, (vocab + 63) / 64}, fp32);
    }
    variable_list out = linear_score_outputs(h, w, ids, ignore_index, launch_rows, stats, kept, slab_max);
    if (kept.has_value()) ctx->save_for_backward({h, w, ids, out[1], stats, *kept, *slab_max});      // (a checkpoint drops what is saved this way)
    else ctx->save_for_backward({h, w, ids, out[1], stats});
    ctx->saved_data["used"] = false;
    ctx->saved_data["captured"] = false;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["launch_rows"] = launch_rows;
    ctx->saved_data["gradient_values"] = gradient_values;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("linear_token_log_probs");
    variable_list result(6);
    if (!grads[0].defined() && !grads[1].defined()) return result;
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &h = saved[0], &w = saved[1];
    const int64_t rows = h.size(0), vocab = w.size(0), cols = (vocab + 7) / 8 * 8, ignore_index = ctx->saved_data["ignore_index"].toInt();
    c10::optional<at::Tensor> g[2], kept, slab_max;
    for (int i = 0; i < 2; ++i)
      if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).contiguous();
    at::Tensor buf;
    int64_t step = rows;
    if (saved.size() == 7 && !ctx->saved_data["used"].toBool()) {
      slab_max = saved[6];
      const bool captured = c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
      if (captured) ctx->saved_data["captured"] = true;    // may be replayed, and again for one forward pass: what was kept stays
      if (ctx->saved_data["captured"].toBool()) {
        kept = saved[5];
        buf = at::empty_like(*kept);
      } else {
        buf = saved[5];
        ctx->saved_data["used"] = true;
      }
    } else {
      step = std::max<int64_t>(256, std::min(ctx->saved_data["launch_rows"].toInt(), ctx->saved_data["gradient_values"].toInt() / cols / 256 * 256));
      buf = at::empty({std::min(rows, step), cols}, h.options());
    }
    at::Tensor dh, dw;
    if (ctx->needs_input_grad(0)) dh = at::empty(h.sizes(), h.options());
    if (ctx->needs_input_grad(1)) {
      dw = at::empty(w.sizes(), rows <= step ? w.options() : w.options().dtype(at::kFloat));       // a sum over several chunks is held in fp32
      if (!rows) dw.zero_();
    }
    for (int64_t r = 0; r < rows; r += step) {
      const int64_t n = std::min(rows - r, step);
      auto chunk = [&](const at::Tensor& t) { return n == rows ? t : t.narrow(0, r, n); };
      auto maybe = [&](const c10::optional<at::Tensor>& t) { return t.has_value() ? c10::optional<at::Tensor>(chunk(*t)) : c10::nullopt; };
      at::Tensor dx = buf.size(0) == n ? buf : buf.narrow(0, 0, n);
      const at::Tensor hc = chunk(h);
      linear_scores_dlogits(hc, w, chunk(saved[2]), chunk(saved[3]), chunk(saved[4]), maybe(g[0]), maybe(g[1]), dx, kept, slab_max, ignore_index);
      autograd_launched += 1;
      if (cols != vocab) dx = dx.narrow(1, 0, vocab);
      if (dh.defined()) {
        at::Tensor to = chunk(dh);
        long_product(dx, w, to);
      }
      if (dw.defined()) {
        gemm(dx, hc, dw, r ? c10::optional<at::Tensor>(dw) : c10::nullopt, true, false, 1.0, r ? 1.0 : 0.0, false, 0, false, true);
        autograd_launched += 1;
      }
    }
    result[0] = dh;
    if (dw.defined()) result[1] = dw.to(w.scalar_type());
    return result;
  }
};

static bool ns5_fused_supported(int64_t m, int64_t n) { return himuon::ns5_fused_supported((int)m, (int)n); }
static void ns5_fused(const at::Tensor& x, at::Tensor& out, int64_t steps, double eps, bool normalize) {
  HM_CHECK(x.is_cuda() && is_bf16(x) && is_bf16(out) && x.is_contiguous() && out.is_contiguous() && x.dim() == 3 && x.sizes() == out.sizes(), "ns5_fused: contiguous (B, m, n) bf16 tensors");
  HM_CHECK(himuon::ns5_fused_supported((int)x.size(1), (int)x.size(2)), "ns5_fused: tile shape not supported");
  const c10::cuda::CUDAGuard guard(x.device());
  himuon::ns5_fused(x.data_ptr(), out.data_ptr(), x.size(0), (int)x.size(1), (int)x.size(2), (int)steps, (float)eps, cur_stream(), normalize ? 1 : 0);
}

// (pairs per matrix, matrices per cluster, scratch bytes) of ns_pair for this batch, or nothing where it is not the better path.
static c10::optional<std::vector<int64_t>> ns_pair_plan(const at::Tensor& x) {
  HM_CHECK(x.is_cuda() && x.dim() == 3, "ns_pair_plan: (B, m, n) CUDA tensor");
  if (x.size(1) >= (1LL << 30) || x.size(2) >= (1LL << 30)) return c10::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  int P = 1, W = 1;
  if (!himuon::ns_pair_plan(x.size(0), (int)x.size(1), (int)x.size(2), &P, &W)) return c10::nullopt;
  return std::vector<int64_t>{P, W, himuon::ns_pair_scratch_bytes(x.size(0), (int)x.size(1), (int)x.size(2), P, W)};
}
static void ns_pair(const at::Tensor& x, at::Tensor& out, at::Tensor& scratch, int64_t steps, int64_t P, int64_t W) {
  HM_CHECK(x.is_cuda() && is_bf16(x) && is_bf16(out) && x.is_contiguous() && out.is_contiguous() && x.dim() == 3 && x.sizes() == out.sizes(), "ns_pair: contiguous (B, m, n) bf16 tensors");
  HM_CHECK(x.size(1) <= 2048 && x.size(2) <= 2048 && x.size(1) % 8 == 0 && x.size(2) % 8 == 0, "ns_pair: sides are multiples of 8, at most 2048");
  HM_CHECK(steps >= 1 && (steps >= 2 || x.data_ptr() != out.data_ptr()), "ns_pair: in place needs two steps");
  HM_CHECK((P == 1 || P == 2 || P == 4) && W >= 1 && W <= 8, "ns_pair: bad plan");
  const c10::cuda::CUDAGuard guard(x.device());
  HM_CHECK(scratch.is_cuda() && scratch.device() == x.device() && scratch.is_contiguous() && reinterpret_cast<uintptr_t>(scratch.data_ptr()) % 128 == 0 &&
           scratch.numel() * scratch.element_size() >= himuon::ns_pair_scratch_bytes(x.size(0), (int)x.size(1), (int)x.size(2), (int)P, (int)W), "ns_pair: scratch too small");
  himuon::ns_pair(x.data_ptr(), out.data_ptr(), scratch.data_ptr(), x.size(0), (int)x.size(1), (int)x.size(2), (int)steps, (int)P, (int)W, cur_stream());
}

static int64_t status(bool reset) { return himuon::read_status_word(reset); }

static void soap_moments(const at::Tensor& g, const at::Tensor& g_rot, at::Tensor& m, at::Tensor& v, double b1, double b2) {
  HM_CHECK(g.is_cuda() && is_bf16(g) && is_bf16(g_rot) && is_bf16(m) && is_bf16(v), "soap_moments: bf16 CUDA tensors");
  HM_CHECK(g.is_contiguous() && g_rot.is_contiguous() && m.is_contiguous() && v.is_contiguous(), "soap_moments: contiguous tensors");
  HM_CHECK(g.numel() == g_rot.numel() && g.numel() == m.numel() && g.numel() == v.numel() && g.numel() % 8 == 0,
           "soap_moments: equal element counts, multiples of 8");
  const at::Tensor* all4[4] = {&g, &g_rot, &m, &v};
  for (const at::Tensor* t : all4)
    HM_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "soap_moments: 16-byte aligned tensors");
  const c10::cuda::CUDAGuard guard(g.device());
  himuon::soap_moments(g.data_ptr(), g_rot.data_ptr(), m.data_ptr(), v.data_ptr(), g.numel(), (float)b1, (float)b2, cur_stream());
}
static void soap_ratio(const at::Tensor& m_rot, const at::Tensor& v, at::Tensor& out, double eps) {
  HM_CHECK(m_rot.is_cuda() && is_bf16(m_rot) && is_bf16(v) && is_bf16(out), "soap_ratio: bf16 CUDA tensors");
  HM_CHECK(m_rot.is_contiguous() && v.is_contiguous() && out.is_contiguous(), "soap_ratio: contiguous tensors");
  HM_CHECK(m_rot.numel() == v.numel() && m_rot.numel() == out.numel() && m_rot.numel() % 8 == 0,
           "soap_ratio: equal element counts, multiples of 8");
  const at::Tensor* all3[3] = {&m_rot, &v, &out};
  for (const at::Tensor* t : all3)
    HM_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "soap_ratio: 16-byte aligned tensors");
  const c10::cuda::CUDAGuard guard(m_rot.device());
  himuon::soap_ratio(m_rot.data_ptr(), v.data_ptr(), out.data_ptr(), m_rot.numel(), (float)eps, cur_stream());
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("soap_moments", &soap_moments);
  m.def("soap_ratio", &soap_ratio);
  m.def("gemm", &gemm, py::arg("a"), py::arg("b"), py::arg("out"), py::arg("aux") = py::none(), py::arg("trans_a") = false,
        py::arg("trans_b") = false, py::arg("alpha") = 1.0, py::arg("beta") = 0.0, py::arg("round_acc") = false,
        py::arg("max_ctas") = 0, py::arg("symmetric") = false, py::arg("ordered") = false);
  m.def("gemm_on_pairs", &gemm_on_pairs, py::arg("a"), py::arg("b"), py::arg("out"), py::arg("aux") = py::none(), py::arg("trans_a") = false,
        py::arg("trans_b") = false, py::arg("alpha") = 1.0, py::arg("beta") = 0.0, py::arg("round_acc") = false,
        py::arg("max_ctas") = 0, py::arg("symmetric") = false);
  m.def("momentum_tile", &momentum_tile);
  m.def("untile_apply", &untile_apply);
  m.def("ns_repad", &ns_repad, py::arg("src"), py::arg("dst"), py::arg("norm") = py::none(), py::arg("eps") = 0.0);
  m.def("ns_normalize", &ns_normalize, py::arg("tiles"), py::arg("n_tiles"), py::arg("tile_elems"), py::arg("eps"),
        py::arg("out") = py::none());
  m.def("adamw_multi", &adamw_multi);
  m.def("adamw_step_advance", &adamw_step_advance);
  m.def("rmsnorm_fwd", &rmsnorm_fwd, py::arg("x"), py::arg("w"), py::arg("y"), py::arg("rstd"), py::arg("eps"),
        py::arg("delta") = py::none(), py::arg("h_out") = py::none());
  m.def("rmsnorm_bwd", &rmsnorm_bwd, py::arg("dy"), py::arg("x"), py::arg("w"), py::arg("rstd"), py::arg("dx"),
        py::arg("dw_accum"), py::arg("dres") = py::none());
  m.def("headnorm_rope_fwd", &headnorm_rope_fwd);
  m.def("headnorm_rope_bwd", &headnorm_rope_bwd);
  m.def("headnorm_heads_per_pass", [](int64_t tokens, int64_t heads, int64_t head_dim, bool backward) {
    return himuon::headnorm_heads_per_pass(tokens * heads, (int)heads, (int)head_dim, backward);
  });
  m.def("swiglu_fwd", &swiglu_fwd);
  m.def("swiglu_bwd", &swiglu_bwd);
  m.def("embedding_fwd", &embedding_fwd);
  m.def("embedding_bwd", &embedding_bwd);
  m.def("cross_entropy", &cross_entropy);
  m.def("packed_attn_fwd", &packed_attn_fwd);
  m.def("packed_attention", [](const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& plan, int64_t tiles, int64_t tokens, int64_t Hq,
                               int64_t Hkv, double scale, bool split_heads) {
    return PackedAttention::apply(q, k, v, plan, tiles, tokens, Hq, Hkv, scale, split_heads);
  });
  m.def("token_scores", [](const at::Tensor& logits, const at::Tensor& ids, int64_t top_k, int64_t ignore_index) {
    if (c10::GradMode::is_enabled() && logits.requires_grad()) return TokenScores::apply(logits, ids, top_k, ignore_index);
    return score_outputs(logits, ids, top_k, ignore_index, c10::nullopt);
  });
  m.def("autograd_launched", [] { return autograd_launched.load(); });
  m.def("token_scores_fwd", &token_scores_fwd);
  m.def("token_scores_bwd", &token_scores_bwd);
  m.def("long_product", &long_product);
  m.def("linear_scores", [](const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, int64_t ignore_index, int64_t launch_rows, int64_t gradient_values) {
    if (c10::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad())) return LinearScores::apply(h, w, ids, ignore_index, launch_rows, gradient_values);
    return linear_score_outputs(h, w, ids, ignore_index, launch_rows, c10::nullopt, c10::nullopt, c10::nullopt);
  });
  m.def("flash_attn_fwd", &flash_attn_fwd);
  m.def("flash_attn_bwd", &flash_attn_bwd);
  m.def("ns5_fused_supported", &ns5_fused_supported);
  m.def("ns5_fused", &ns5_fused, py::arg("x"), py::arg("out"), py::arg("steps"), py::arg("eps"), py::arg("normalize") = true);
  m.def("ns_pair_plan", &ns_pair_plan);
  m.def("ns_pair", &ns_pair);
  m.def("status", &status, py::arg("reset") = true);
  m.def("num_sms", [] { return himuon::num_sms(); });
  m.def("momentum_tile_units", [](int64_t R, int64_t C, int64_t Th) { return himuon::momentum_tile_units((int)R, (int)C, (int)Th); });
  m.def("sizeof_entries", [] {
    return std::vector<int64_t>{(int64_t)sizeof(himuon::MomTileEntry), (int64_t)sizeof(himuon::ApplyEntry), (int64_t)sizeof(himuon::AdamEntry)};
  });
  himuon::bind_symm(m);
}
