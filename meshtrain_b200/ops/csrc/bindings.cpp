// bindings.cpp -- torch adapters for the meshtrain_b200 sm_100a kernels.
//
// Each function validates dtypes/shapes/alignment, launches on the current
// CUDA stream of the tensor's device and raises a Python error if the launch
// fails.  No function here falls back to a library implementation.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "mt_api.h"

namespace {

using torch::Tensor;

#define MT_CHECK_LAUNCH(expr, what)                                              \
  do {                                                                           \
    int _rc = (expr);                                                            \
    TORCH_CHECK(_rc == 0, "meshtrain_b200 ", what, " failed (code ", _rc, ")"); \
  } while (0)

void check_cuda(const Tensor& t, const char* name, at::ScalarType dt) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == dt, name, " has dtype ", t.scalar_type(), ", expected ", dt);
}
void check_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name, " must be 16-byte aligned");
}
cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()); }

void check_matrix(const Tensor& t, const char* name) {
  check_cuda(t, name, at::kBFloat16);
  TORCH_CHECK(t.dim() == 2 && t.stride(1) == 1, name, " must be a 2-D row-major matrix");
  TORCH_CHECK(t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1), name,
              " leading dimension must be a multiple of 8 elements and cover a row");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name, " must be 16-byte aligned");
}

// D = epi(A x B^T).  a: [M,K] (a_mn=false) or [K,M]; b: [N,K] (b_mn=false) or [K,N].
void gemm(Tensor a, bool a_mn, Tensor b, bool b_mn, Tensor d, int64_t epi, c10::optional<Tensor> bias,
          c10::optional<Tensor> aux, c10::optional<Tensor> d2, double beta) {
  check_matrix(a, "A");
  check_matrix(b, "B");
  const int64_t M = a_mn ? a.size(1) : a.size(0);
  const int64_t K = a_mn ? a.size(0) : a.size(1);
  const int64_t N = b_mn ? b.size(1) : b.size(0);
  TORCH_CHECK((b_mn ? b.size(0) : b.size(1)) == K, "gemm: K mismatch");
  TORCH_CHECK(d.is_cuda() && d.dim() == 2 && d.stride(1) == 1 && d.size(0) == M, "gemm: D must be [M, *] row-major");
  TORCH_CHECK(a.get_device() == b.get_device() && a.get_device() == d.get_device(), "gemm: device mismatch");
  const bool f32 = epi == 4;
  TORCH_CHECK(d.scalar_type() == (f32 ? at::kFloat : at::kBFloat16), "gemm: D dtype does not match the epilogue");
  if (epi == 5) {
    TORCH_CHECK(d.size(1) >= N / 2, "gemm: SwiGLU output too narrow");
  } else {
    TORCH_CHECK(d.size(1) >= N, "gemm: D too narrow");
  }
  c10::cuda::CUDAGuard guard(a.get_device());
  mt::GemmArgs g{};
  g.a = a.data_ptr();
  g.lda = a.stride(0);
  g.a_mn = a_mn;
  g.b = b.data_ptr();
  g.ldb = b.stride(0);
  g.b_mn = b_mn;
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.epi = (int)epi;
  g.d = d.data_ptr();
  g.ldd = d.stride(0);
  g.beta = (float)beta;
  if (bias) {
    check_cuda(*bias, "bias", at::kBFloat16);
    TORCH_CHECK(bias->is_contiguous() && bias->numel() >= N, "gemm: bias must be contiguous [N]");
    g.bias = bias->data_ptr();
  }
  if (aux) {
    check_cuda(*aux, "aux", at::kBFloat16);
    TORCH_CHECK(aux->dim() == 2 && aux->stride(1) == 1 && aux->size(0) == M && aux->size(1) >= N, "gemm: bad aux");
    g.aux = aux->data_ptr();
    g.ldaux = aux->stride(0);
  }
  if (d2) {
    check_cuda(*d2, "d2", at::kBFloat16);
    TORCH_CHECK(d2->dim() == 2 && d2->stride(1) == 1 && d2->size(0) == M && d2->size(1) >= N, "gemm: bad d2");
    g.d2 = d2->data_ptr();
    g.ldd2 = d2->stride(0);
  }
  if (epi == 1 || epi == 5) TORCH_CHECK(g.d2 != nullptr, "gemm: epilogue needs d2");
  if (epi == 2 || epi == 3) TORCH_CHECK(g.aux != nullptr, "gemm: epilogue needs aux");
  if (epi == 5) TORCH_CHECK(N % 32 == 0, "gemm: SwiGLU needs N % 32 == 0");
  if (M == 0 || N == 0) return;
  if (K == 0) {
    if (f32) {
      if (beta == 0.0) d.narrow(1, 0, N).zero_();
      else if (beta != 1.0) d.narrow(1, 0, N).mul_(beta);
    } else {
      d.narrow(1, 0, epi == 5 ? N / 2 : N).zero_();
    }
    return;
  }
  char err[256] = {0};
  int rc = mt::gemm_launch(g, a.get_device(), stream_of(a), err, sizeof(err));
  TORCH_CHECK(rc == 0, "meshtrain_b200 gemm: ", err);
}

std::vector<Tensor> layernorm_fwd(Tensor x, Tensor gamma, Tensor beta, double eps) {
  check_cuda(x, "x", at::kBFloat16);
  check_rows(x, "x");
  const int64_t d = x.size(-1), T = x.numel() / std::max<int64_t>(d, 1);
  c10::cuda::CUDAGuard guard(x.get_device());
  auto y = torch::empty_like(x);
  auto opts = x.options().dtype(at::kFloat);
  auto mean = torch::empty({T}, opts), rstd = torch::empty({T}, opts);
  MT_CHECK_LAUNCH(mt::layernorm_fwd(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(),
                                    mean.data_ptr<float>(), rstd.data_ptr<float>(), (int)T, (int)d, (float)eps,
                                    stream_of(x)),
                  "layernorm_fwd");
  return {y, mean, rstd};
}

Tensor layernorm_bwd(Tensor dy, Tensor x, Tensor gamma, Tensor mean, Tensor rstd, c10::optional<Tensor> dres,
                     Tensor dgamma, Tensor dbeta) {
  check_cuda(dy, "dy", at::kBFloat16);
  check_rows(dy, "dy");
  check_rows(x, "x");
  check_cuda(dgamma, "dgamma", at::kFloat);
  check_cuda(dbeta, "dbeta", at::kFloat);
  const int64_t d = x.size(-1), T = x.numel() / std::max<int64_t>(d, 1);
  c10::cuda::CUDAGuard guard(x.get_device());
  auto dx = torch::empty_like(x);
  MT_CHECK_LAUNCH(mt::layernorm_bwd(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr<float>(),
                                    rstd.data_ptr<float>(), dres ? dres->data_ptr() : nullptr, dx.data_ptr(),
                                    dgamma.data_ptr<float>(), dbeta.data_ptr<float>(), (int)T, (int)d, stream_of(x)),
                  "layernorm_bwd");
  return dx;
}

std::vector<Tensor> rmsnorm_fwd(Tensor x, Tensor gamma, double eps) {
  check_cuda(x, "x", at::kBFloat16);
  check_rows(x, "x");
  const int64_t d = x.size(-1), T = x.numel() / std::max<int64_t>(d, 1);
  c10::cuda::CUDAGuard guard(x.get_device());
  auto y = torch::empty_like(x);
  auto rstd = torch::empty({T}, x.options().dtype(at::kFloat));
  MT_CHECK_LAUNCH(mt::rmsnorm_fwd(x.data_ptr(), gamma.data_ptr(), y.data_ptr(), rstd.data_ptr<float>(), (int)T,
                                  (int)d, (float)eps, stream_of(x)),
                  "rmsnorm_fwd");
  return {y, rstd};
}

Tensor rmsnorm_bwd(Tensor dy, Tensor x, Tensor gamma, Tensor rstd, c10::optional<Tensor> dres, Tensor dgamma) {
  check_cuda(dy, "dy", at::kBFloat16);
  check_rows(dy, "dy");
  check_rows(x, "x");
  check_cuda(dgamma, "dgamma", at::kFloat);
  const int64_t d = x.size(-1), T = x.numel() / std::max<int64_t>(d, 1);
  c10::cuda::CUDAGuard guard(x.get_device());
  auto dx = torch::empty_like(x);
  MT_CHECK_LAUNCH(mt::rmsnorm_bwd(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), rstd.data_ptr<float>(),
                                  dres ? dres->data_ptr() : nullptr, dx.data_ptr(), dgamma.data_ptr<float>(), (int)T,
                                  (int)d, stream_of(x)),
                  "rmsnorm_bwd");
  return dx;
}

Tensor embedding_fwd(Tensor ids, Tensor tok, c10::optional<Tensor> pos, int64_t S) {
  check_cuda(ids, "ids", at::kLong);
  check_cuda(tok, "tok", at::kBFloat16);
  const int64_t T = ids.numel(), d = tok.size(1), V = tok.size(0);
  c10::cuda::CUDAGuard guard(tok.get_device());
  auto out = torch::empty({T, d}, tok.options());
  MT_CHECK_LAUNCH(mt::embedding_fwd(ids.contiguous().data_ptr<int64_t>(), tok.data_ptr(),
                                    pos ? pos->data_ptr() : nullptr, out.data_ptr(), (int)T, (int)S, (int)d, (int)V,
                                    stream_of(tok)),
                  "embedding_fwd");
  return out;
}

void embedding_bwd(Tensor ids, Tensor dy, Tensor tok_grad, c10::optional<Tensor> pos_grad, int64_t S) {
  check_cuda(ids, "ids", at::kLong);
  check_cuda(dy, "dy", at::kBFloat16);
  check_rows(dy, "dy");
  check_cuda(tok_grad, "tok_grad", at::kFloat);
  const int64_t T = ids.numel(), d = tok_grad.size(1), V = tok_grad.size(0);
  c10::cuda::CUDAGuard guard(dy.get_device());
  Tensor flat_ids = ids.contiguous();
  if (T <= 32768 && V <= 131072) {  // deterministic: sorted by token id, one writer per row
    Tensor scratch = torch::empty({mt::embedding_bwd_sorted_scratch_ints((int)T)},
                                  torch::dtype(torch::kInt32).device(dy.device()));
    MT_CHECK_LAUNCH(mt::embedding_bwd_sorted(flat_ids.data_ptr<int64_t>(), dy.data_ptr(), tok_grad.data_ptr<float>(),
                                             pos_grad ? pos_grad->data_ptr<float>() : nullptr, (int)T, (int)S, (int)d,
                                             (int)V, scratch.data_ptr<int>(), stream_of(dy)),
                    "embedding_bwd_sorted");
    return;
  }
  MT_CHECK_LAUNCH(mt::embedding_bwd(flat_ids.data_ptr<int64_t>(), dy.data_ptr(), tok_grad.data_ptr<float>(),
                                    pos_grad ? pos_grad->data_ptr<float>() : nullptr, (int)T, (int)S, (int)d, (int)V,
                                    stream_of(dy)),
                  "embedding_bwd");
}

void colsum_(Tensor dy, Tensor out) {
  check_cuda(dy, "dy", at::kBFloat16);
  check_cuda(out, "out", at::kFloat);
  TORCH_CHECK(dy.dim() == 2 && dy.stride(1) == 1, "colsum: dy must be 2-D row-major");
  c10::cuda::CUDAGuard guard(dy.get_device());
  MT_CHECK_LAUNCH(mt::colsum_accumulate(dy.data_ptr(), dy.stride(0), out.data_ptr<float>(), (int)dy.size(0),
                                        (int)dy.size(1), stream_of(dy)),
                  "colsum");
}

Tensor swiglu_bwd(Tensor dout, Tensor raw) {
  check_cuda(dout, "dout", at::kBFloat16);
  check_cuda(raw, "raw", at::kBFloat16);
  check_rows(dout, "dout");
  check_rows(raw, "raw");
  const int64_t F = dout.size(-1), T = dout.numel() / std::max<int64_t>(F, 1);
  c10::cuda::CUDAGuard guard(dout.get_device());
  auto draw = torch::empty_like(raw);
  MT_CHECK_LAUNCH(mt::swiglu_bwd(dout.data_ptr(), raw.data_ptr(), draw.data_ptr(), (int)T, (int)F, stream_of(dout)),
                  "swiglu_bwd");
  return draw;
}

void rope_(Tensor qk, int64_t S, int64_t H, int64_t hd, double theta, bool inverse) {
  check_cuda(qk, "qk", at::kBFloat16);
  TORCH_CHECK(qk.dim() == 2 && qk.stride(1) == 1 && qk.size(1) >= H * hd, "rope: qk must be [T, >=H*hd]");
  c10::cuda::CUDAGuard guard(qk.get_device());
  MT_CHECK_LAUNCH(mt::rope_apply(qk.data_ptr(), qk.stride(0), (int)qk.size(0), (int)S, (int)H, (int)hd, (float)theta,
                                 inverse, stream_of(qk)),
                  "rope");
}

void cross_entropy_(Tensor logits, int64_t V, Tensor targets, Tensor loss_sum, double loss_scale, double grad_scale) {
  check_cuda(logits, "logits", at::kBFloat16);
  check_cuda(targets, "targets", at::kLong);
  check_cuda(loss_sum, "loss_sum", at::kFloat);
  TORCH_CHECK(logits.dim() == 2 && logits.stride(1) == 1 && logits.stride(0) % 8 == 0 && logits.size(1) >= V,
              "cross_entropy: logits must be [T, >=V] with a leading dim multiple of 8");
  TORCH_CHECK(targets.numel() == logits.size(0), "cross_entropy: one target per row");
  c10::cuda::CUDAGuard guard(logits.get_device());
  MT_CHECK_LAUNCH(mt::cross_entropy_fwd_bwd(logits.data_ptr(), logits.stride(0), targets.contiguous().data_ptr<int64_t>(),
                                            loss_sum.data_ptr<float>(), (int)logits.size(0), (int)V, (float)loss_scale,
                                            (float)grad_scale, stream_of(logits)),
                  "cross_entropy");
}

// The functions below refuse bad arguments with a ValueError and take any layout: what the kernels
// cannot read in place is copied first.

// Element type code of mt_api.h.
int dtype_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK_VALUE(false, name, " has dtype ", t.scalar_type(), ", expected bfloat16, float16 or float32");
  }
  return -1;
}
constexpr int64_t kMostRows = int64_t(1) << 30;  // the kernels' row and column indexes are 32-bit
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// Rows the kernels read and write in place: unit column stride, 16-byte aligned, a leading dimension
// that is a multiple of 8.
bool is_rows(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && aligned16(t);
}
Tensor padded_rows(const Tensor& like, int64_t rows, int64_t cols) {
  const int64_t ld = (cols + 7) / 8 * 8;
  Tensor t = torch::empty({rows, ld}, like.options());
  return ld == cols ? t : t.narrow(1, 0, cols);
}
// The first `cols` columns of a matrix of at least that many, on `like`'s device and of its type, as rows.
Tensor as_rows(const Tensor& t, const char* name, const Tensor& like, int64_t rows, int64_t cols) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) >= cols && t.scalar_type() == like.scalar_type() &&
                        t.device() == like.device(),
                    name, " must be [", rows, ", >= ", cols, "] ", like.scalar_type(), " on ", like.device());
  TORCH_CHECK_VALUE(rows <= kMostRows && cols <= kMostRows, name, " is larger than 2^30 rows or columns");
  if (is_rows(t)) return t;
  Tensor copy = padded_rows(like, rows, cols);
  copy.copy_(t.narrow(1, 0, cols));
  return copy;
}
// `out` checked for in-place writing, or new rows.
Tensor out_rows(const c10::optional<Tensor>& out, const char* name, const Tensor& like, int64_t rows, int64_t cols) {
  if (!out) return padded_rows(like, rows, cols);
  TORCH_CHECK_VALUE(out->dim() == 2 && out->size(0) == rows && out->size(1) >= cols &&
                        out->scalar_type() == like.scalar_type() && out->device() == like.device() &&
                        out->stride(1) == 1 && out->stride(0) % 8 == 0 && (rows < 2 || out->stride(0) >= cols) &&
                        aligned16(*out),
                    name, ": out must be [rows, >= ", cols, "] row-major of the input's dtype and device, its rows on ",
                    "16-byte boundaries with a leading dimension that is a multiple of 8");
  return out->size(1) == cols ? *out : out->narrow(1, 0, cols);
}
// A contiguous vector of n values on `like`'s device.
Tensor as_vector(const Tensor& t, const char* name, at::ScalarType dt, const Tensor& like, int64_t n) {
  TORCH_CHECK_VALUE(t.numel() == n && t.scalar_type() == dt && t.device() == like.device(), name, " must have ", n,
                    " values of ", dt, " on ", like.device(), ", got ", t.sizes(), " of ", t.scalar_type(), " on ",
                    t.device());
  return t.contiguous();
}
Tensor as_aligned(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone();
}

struct QkInputs {
  mt::QkNormRopeArgs a{};
  Tensor x, gq, gk, out;  // keep copies alive
};
void qk_inputs(QkInputs& in, const char* name, const Tensor& qkv, const Tensor& gq, const Tensor& gk,
                   const c10::optional<Tensor>& out, int64_t S, int64_t H, int64_t HK, int64_t hd, double theta,
                   double eps) {
  TORCH_CHECK_VALUE(qkv.is_cuda() && qkv.dim() == 2 && H >= 0 && HK >= 0 && H + HK >= 1 && H + HK <= 65536 && hd >= 2,
                    name, ": qkv must be [rows, >= (heads + kv_heads) * head_dim]");
  TORCH_CHECK_VALUE(hd % 16 == 0 && hd <= 256, name, ": head_dim ", hd,
                    " unsupported by the kernel (multiples of 16 up to 256)");
  TORCH_CHECK_VALUE(S >= 1 && S < INT32_MAX && theta > 0 && eps >= 0, name,
                    ": needs seq_len >= 1, theta > 0 and eps >= 0");
  in.a.dtype = dtype_code(qkv, name);
  const int64_t rows = qkv.size(0), cols = (H + HK) * hd;
  for (auto* g : {&gq, &gk})
    TORCH_CHECK_VALUE(g->dim() == 1 && g->size(0) == hd && g->scalar_type() == qkv.scalar_type() &&
                          g->device() == qkv.device(),
                      name, ": gains must be [head_dim] of qkv's dtype and device");
  in.x = as_rows(qkv, name, qkv, rows, cols);
  in.out = out_rows(out, name, qkv, rows, cols);
  in.gq = as_aligned(gq);
  in.gk = as_aligned(gk);
  in.a.x = in.x.data_ptr();
  in.a.ldx = in.x.stride(0);
  in.a.gq = in.gq.data_ptr();
  in.a.gk = in.gk.data_ptr();
  in.a.out = in.out.data_ptr();
  in.a.ldo = in.out.stride(0);
  in.a.rows = (int)rows;
  in.a.S = (int)S;
  in.a.H = (int)H;
  in.a.HK = (int)HK;
  in.a.hd = (int)hd;
  in.a.eps = (float)eps;
  in.a.theta = theta;
}

Tensor qk_norm_rope_fwd(const Tensor& qkv, const Tensor& gq, const Tensor& gk, int64_t S, int64_t H, int64_t HK,
                        int64_t hd, double theta, double eps, const c10::optional<Tensor>& out) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(qkv));
  QkInputs in;
  qk_inputs(in, "qk_norm_rope", qkv, gq, gk, out, S, H, HK, hd, theta, eps);
  MT_CHECK_LAUNCH(mt::qk_norm_rope_fwd(in.a, stream_of(qkv)), "qk_norm_rope");
  return in.out;
}

Tensor qk_norm_rope_bwd(const Tensor& dqk, const Tensor& qkv, const Tensor& gq, const Tensor& gk, int64_t S, int64_t H,
                        int64_t HK, int64_t hd, double theta, Tensor dgq, Tensor dgk, double eps,
                        const c10::optional<Tensor>& out) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(qkv));
  QkInputs in;
  qk_inputs(in, "qk_norm_rope_bwd", qkv, gq, gk, out, S, H, HK, hd, theta, eps);
  const Tensor dy = as_rows(dqk, "qk_norm_rope_bwd: dqk", qkv, qkv.size(0), (H + HK) * hd);
  for (auto* g : {&dgq, &dgk})
    TORCH_CHECK_VALUE(g->dim() == 1 && g->size(0) == hd && g->scalar_type() == at::kFloat &&
                          g->device() == qkv.device() && g->is_contiguous(),
                      "qk_norm_rope_bwd: dq_gain and dk_gain must be contiguous float32 [head_dim]");
  if (in.a.rows == 0) return in.out;
  // One gradient for both gains (or two that share memory): the kernel adds to either without order, so the
  // key gain's sum is formed beside it and added after.
  const auto *q0 = dgq.data_ptr<float>(), *k0 = dgk.data_ptr<float>();
  const bool shared = q0 < k0 + hd && k0 < q0 + hd;
  Tensor dk = shared ? torch::zeros({hd}, dgk.options()) : dgk;
  auto partial = torch::empty({mt::qk_norm_rope_blocks(in.a.rows, in.a.H + in.a.HK, in.a.hd), 2 * hd}, dgq.options());
  MT_CHECK_LAUNCH(mt::qk_norm_rope_bwd(in.a, dy.data_ptr(), dy.stride(0), partial.data_ptr<float>(),
                                       dgq.data_ptr<float>(), dk.data_ptr<float>(), stream_of(qkv)),
                  "qk_norm_rope_bwd");
  if (shared) dgk.add_(dk);
  return in.out;
}

// seed carries 64 unsigned bits in int64, and so does an offset that is no tensor.
Tensor dropout(const Tensor& x, int64_t cut, int64_t seed, int64_t offset, const c10::optional<Tensor>& offset_tensor,
               const c10::optional<Tensor>& residual, const c10::optional<Tensor>& out) {
  TORCH_CHECK_VALUE(x.is_cuda(), "dropout: x must be a CUDA tensor");
  TORCH_CHECK_VALUE(cut >= 0 && cut < 65536, "dropout: p must be in [0, 1) and round below 1");
  c10::cuda::OptionalCUDAGuard guard(at::device_of(x));
  mt::DropoutArgs a{};
  a.dtype = dtype_code(x, "x");
  for (auto* t : {&residual, &out})
    TORCH_CHECK_VALUE(!*t || ((*t)->sizes() == x.sizes() && (*t)->scalar_type() == x.scalar_type() &&
                              (*t)->device() == x.device()),
                      "dropout: residual and out must have x's shape, dtype and device");
  TORCH_CHECK_VALUE(!out || (out->is_contiguous() && aligned16(*out)),
                    "dropout: out must be contiguous and start on a 16-byte boundary");
  const Tensor xc = as_aligned(x);
  Tensor rc, res = out ? *out : torch::empty(x.sizes(), x.options());
  a.x = xc.data_ptr();
  a.n = x.numel();
  if (residual) {
    rc = as_aligned(*residual);
    a.residual = rc.data_ptr();
  }
  a.out = res.data_ptr();
  a.cut = (uint32_t)cut;
  a.seed = (uint64_t)seed;
  a.offset = (uint64_t)offset;
  if (offset_tensor) {
    TORCH_CHECK_VALUE(offset_tensor->numel() == 1 && offset_tensor->scalar_type() == at::kLong &&
                          offset_tensor->device() == x.device(),
                      "dropout: an offset tensor must be one int64 on x's device");
    a.offset_ptr = offset_tensor->data_ptr<int64_t>();
  }
  MT_CHECK_LAUNCH(mt::dropout_apply(a, stream_of(x)), "dropout");
  return res;
}

Tensor as_logits(const char* name, const Tensor& logits, int64_t V) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && V >= 1 && logits.size(1) >= V, name,
                    ": logits must be [rows, >= vocab]");
  return as_rows(logits, name, logits, logits.size(0), V);
}

std::tuple<Tensor, Tensor> token_logprobs(const Tensor& logits, int64_t V, const Tensor& targets) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(logits));
  const Tensor x = as_logits("token_logprobs", logits, V);
  const int64_t rows = logits.size(0);
  const Tensor t = as_vector(targets, "token_logprobs: targets", at::kLong, logits, rows);
  auto fopts = logits.options().dtype(at::kFloat);
  auto logps = torch::empty({rows}, fopts), stats = torch::empty({rows, 2}, fopts);
  MT_CHECK_LAUNCH(mt::token_logprobs(x.data_ptr(), x.stride(0), dtype_code(logits, "logits"), t.data_ptr<int64_t>(),
                                     logps.data_ptr<float>(), stats.data_ptr<float>(), (int)rows, (int)V,
                                     stream_of(logits)),
                  "token_logprobs");
  return {logps, stats};
}

Tensor token_logprobs_bwd(const Tensor& logits, int64_t V, const Tensor& targets, const Tensor& stats,
                          const Tensor& dlogps, const c10::optional<Tensor>& out) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(logits));
  const Tensor x = as_logits("token_logprobs_bwd", logits, V);
  const int64_t rows = logits.size(0);
  const Tensor t = as_vector(targets, "token_logprobs_bwd: targets", at::kLong, logits, rows);
  const Tensor st = as_aligned(as_vector(stats, "token_logprobs_bwd: stats", at::kFloat, logits, 2 * rows));
  const Tensor up = as_vector(dlogps, "token_logprobs_bwd: dlogps", at::kFloat, logits, rows);
  Tensor res = out_rows(out, "token_logprobs_bwd", logits, rows, V);
  MT_CHECK_LAUNCH(mt::token_logprobs_bwd(x.data_ptr(), x.stride(0), dtype_code(logits, "logits"), t.data_ptr<int64_t>(),
                                         st.data_ptr<float>(), up.data_ptr<float>(), res.data_ptr(), res.stride(0),
                                         (int)rows, (int)V, stream_of(logits)),
                  "token_logprobs_bwd");
  return res;
}

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, int64_t V, const Tensor& targets,
                                               const Tensor& old_logps, const Tensor& advantages,
                                               const c10::optional<Tensor>& weights,
                                               const c10::optional<Tensor>& ref_logps, double clip_low,
                                               double clip_high, double kl_coef, double grad_scale,
                                               const c10::optional<Tensor>& out) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(logits));
  const Tensor x = as_logits("policy_loss_chunk", logits, V);
  const int64_t rows = logits.size(0);
  TORCH_CHECK_VALUE(clip_low >= 0 && clip_low <= 1 && clip_high >= 0,
                    "policy_loss_chunk: needs 0 <= clip_low <= 1 and clip_high >= 0");
  TORCH_CHECK_VALUE(kl_coef == 0 || ref_logps, "policy_loss_chunk: a KL term needs ref_logps");
  const Tensor t = as_vector(targets, "policy_loss_chunk: targets", at::kLong, logits, rows);
  const Tensor old = as_vector(old_logps, "policy_loss_chunk: old_logps", at::kFloat, logits, rows);
  const Tensor adv = as_vector(advantages, "policy_loss_chunk: advantages", at::kFloat, logits, rows);
  Tensor w, ref;
  if (weights) w = as_vector(*weights, "policy_loss_chunk: weights", at::kFloat, logits, rows);
  if (ref_logps) ref = as_vector(*ref_logps, "policy_loss_chunk: ref_logps", at::kFloat, logits, rows);
  Tensor res = out_rows(out, "policy_loss_chunk", logits, rows, V);
  auto losses = torch::empty({rows}, logits.options().dtype(at::kFloat)), logps = torch::empty_like(losses);
  mt::PolicyArgs a{};
  a.logits = x.data_ptr();
  a.ld = x.stride(0);
  a.out = res.data_ptr();
  a.ldo = res.stride(0);
  a.dtype = dtype_code(logits, "logits");
  a.targets = t.data_ptr<int64_t>();
  a.old_logps = old.data_ptr<float>();
  a.ref_logps = kl_coef != 0 ? ref.data_ptr<float>() : nullptr;
  a.advantages = adv.data_ptr<float>();
  a.weights = weights ? w.data_ptr<float>() : nullptr;
  a.losses = losses.data_ptr<float>();
  a.logps = logps.data_ptr<float>();
  a.rows = (int)rows;
  a.V = (int)V;
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  a.grad_scale = grad_scale;
  MT_CHECK_LAUNCH(mt::policy_loss(a, stream_of(logits)), "policy_loss_chunk");
  return {losses, logps, res};
}

std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor& logps, const Tensor& ref_logps, const Tensor& mask,
                                                   double beta, double label_smoothing, bool squared,
                                                   double grad_scale) {
  TORCH_CHECK_VALUE(logps.is_cuda() && logps.dim() == 2 && logps.size(0) % 2 == 0 &&
                        logps.scalar_type() == at::kFloat && logps.size(1) <= kMostRows && logps.size(0) <= kMostRows,
                    "preference_loss: logps must be fp32 [2 pairs, S]");
  TORCH_CHECK_VALUE(beta > 0 && label_smoothing >= 0 && label_smoothing <= 1,
                    "preference_loss: needs beta > 0 and 0 <= label_smoothing <= 1");
  TORCH_CHECK_VALUE(!squared || label_smoothing == 0, "preference_loss: label_smoothing is the sigmoid form's");
  TORCH_CHECK_VALUE(ref_logps.sizes() == logps.sizes() && mask.sizes() == logps.sizes(),
                    "preference_loss: ref_logps and mask must have logps's shape");
  c10::cuda::OptionalCUDAGuard guard(at::device_of(logps));
  const int64_t pairs = logps.size(0) / 2;
  const Tensor lp = logps.contiguous();
  const Tensor ref = as_vector(ref_logps, "preference_loss: ref_logps", at::kFloat, logps, logps.numel());
  const Tensor m = as_vector(mask, "preference_loss: mask", at::kBool, logps, logps.numel());
  auto losses = torch::empty({pairs}, logps.options()), rewards = torch::empty({2 * pairs}, logps.options());
  auto dlogps = torch::empty(logps.sizes(), logps.options());
  mt::PreferenceArgs a{};
  a.logps = lp.data_ptr<float>();
  a.ref_logps = ref.data_ptr<float>();
  a.mask = reinterpret_cast<const uint8_t*>(m.data_ptr<bool>());
  a.losses = losses.data_ptr<float>();
  a.rewards = rewards.data_ptr<float>();
  a.dlogps = dlogps.data_ptr<float>();
  a.pairs = (int)pairs;
  a.S = (int)logps.size(1);
  a.beta = beta;
  a.label_smoothing = label_smoothing;
  a.grad_scale = grad_scale;
  a.squared = squared;
  MT_CHECK_LAUNCH(mt::preference_loss(a, stream_of(logps)), "preference_loss");
  return {losses, rewards, dlogps};
}

void adam_(Tensor p, Tensor g, Tensor m, Tensor v, c10::optional<Tensor> pb, double lr, double beta1, double beta2,
           double eps, double wd, bool decoupled, double bc1, double bc2, double grad_scale) {
  for (auto* t : {&p, &g, &m, &v}) {
    check_cuda(*t, "adam buffer", at::kFloat);
    check_rows(*t, "adam buffer");
    TORCH_CHECK(t->numel() == p.numel(), "adam: buffer sizes differ");
  }
  if (pb) {
    check_cuda(*pb, "param_bf16", at::kBFloat16);
    TORCH_CHECK(pb->is_contiguous() && pb->numel() == p.numel(), "adam: bf16 copy size differs");
    TORCH_CHECK((reinterpret_cast<uintptr_t>(pb->data_ptr()) & 7) == 0, "adam: bf16 copy must be 8-byte aligned");
  }
  c10::cuda::CUDAGuard guard(p.get_device());
  MT_CHECK_LAUNCH(mt::adam_step(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(),
                                pb ? pb->data_ptr() : nullptr, p.numel(), (float)lr, (float)beta1, (float)beta2,
                                (float)eps, (float)wd, decoupled, (float)bc1, (float)bc2, (float)grad_scale,
                                stream_of(p)),
                  "adam");
}

void cast_bf16_(Tensor in, Tensor out) {
  check_cuda(in, "in", at::kFloat);
  check_cuda(out, "out", at::kBFloat16);
  check_rows(in, "in");
  check_rows(out, "out");
  TORCH_CHECK(in.numel() == out.numel(), "cast: size mismatch");
  c10::cuda::CUDAGuard guard(in.get_device());
  MT_CHECK_LAUNCH(mt::cast_f32_bf16(in.data_ptr<float>(), out.data_ptr(), in.numel(), stream_of(in)), "cast");
}

void check_bshd(const Tensor& t, const char* name) {
  check_cuda(t, name, at::kBFloat16);
  TORCH_CHECK(t.dim() == 4, name, " must be [B, S, H, hd]");
  TORCH_CHECK(t.stride(3) == 1 && t.stride(2) == t.size(3), name, " must have contiguous heads");
  TORCH_CHECK(t.size(0) == 1 || t.stride(0) == t.size(1) * t.stride(1), name, " batches must be back to back");
  TORCH_CHECK(t.stride(1) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name,
              " rows must be 16-byte aligned");
}

std::vector<Tensor> attention_fwd(Tensor q, Tensor k, Tensor v, bool causal, double scale) {
  check_bshd(q, "q");
  check_bshd(k, "k");
  check_bshd(v, "v");
  const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2), hd = q.size(3), Hk = k.size(2);
  TORCH_CHECK(k.size(0) == B && k.size(1) == S && k.size(3) == hd && v.sizes() == k.sizes(), "attention: k/v shape");
  c10::cuda::CUDAGuard guard(q.get_device());
  auto o = torch::empty({B, S, Hq, hd}, q.options());
  auto lse = torch::empty({B, Hq, S}, q.options().dtype(at::kFloat));
  mt::AttnArgs a{};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.ld_q = q.stride(1);
  a.ld_k = k.stride(1);
  a.ld_v = v.stride(1);
  a.o = o.data_ptr();
  a.ld_o = Hq * hd;
  a.lse = lse.data_ptr<float>();
  a.B = (int)B;
  a.S = (int)S;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.hd = (int)hd;
  a.scale = (float)scale;
  a.causal = causal;
  char err[256] = {0};
  int rc = mt::attention_fwd(a, q.get_device(), stream_of(q), err, sizeof(err));
  TORCH_CHECK(rc == 0, "meshtrain_b200 ", err);
  return {o, lse};
}

std::vector<Tensor> attention_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, bool causal,
                                  double scale, c10::optional<Tensor> dq_out, c10::optional<Tensor> dk_out,
                                  c10::optional<Tensor> dv_out) {
  check_bshd(dout, "dout");
  check_bshd(q, "q");
  check_bshd(k, "k");
  check_bshd(v, "v");
  check_bshd(o, "o");
  check_cuda(lse, "lse", at::kFloat);
  TORCH_CHECK(lse.is_contiguous(), "lse must be contiguous [B, Hq, S]");
  const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2), hd = q.size(3), Hk = k.size(2);
  c10::cuda::CUDAGuard guard(q.get_device());
  Tensor dq = dq_out ? *dq_out : torch::empty({B, S, Hq, hd}, q.options());
  Tensor dk = dk_out ? *dk_out : torch::empty({B, S, Hk, hd}, q.options());
  Tensor dv = dv_out ? *dv_out : torch::empty({B, S, Hk, hd}, q.options());
  check_bshd(dq, "dq");
  check_bshd(dk, "dk");
  check_bshd(dv, "dv");
  auto fopts = q.options().dtype(at::kFloat);
  auto dq_accum = torch::empty({B, S, Hq, hd}, fopts);
  auto delta = torch::empty({B, Hq, S}, fopts);
  mt::AttnBwdArgs a{};
  a.f.q = q.data_ptr();
  a.f.k = k.data_ptr();
  a.f.v = v.data_ptr();
  a.f.ld_q = q.stride(1);
  a.f.ld_k = k.stride(1);
  a.f.ld_v = v.stride(1);
  a.f.o = o.data_ptr();
  a.f.ld_o = o.stride(1);
  a.f.lse = lse.data_ptr<float>();
  a.f.B = (int)B;
  a.f.S = (int)S;
  a.f.Hq = (int)Hq;
  a.f.Hk = (int)Hk;
  a.f.hd = (int)hd;
  a.f.scale = (float)scale;
  a.f.causal = causal;
  a.dout = dout.data_ptr();
  a.ld_do = dout.stride(1);
  a.dq = dq.data_ptr();
  a.dk = dk.data_ptr();
  a.dv = dv.data_ptr();
  a.ld_dq = dq.stride(1);
  a.ld_dk = dk.stride(1);
  a.ld_dv = dv.stride(1);
  a.dq_accum = dq_accum.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  char err[256] = {0};
  int rc = mt::attention_bwd(a, q.get_device(), stream_of(q), err, sizeof(err));
  TORCH_CHECK(rc == 0, "meshtrain_b200 ", err);
  return {dq, dk, dv};
}

int64_t read_status(int64_t device) { return (int64_t)mt::read_and_clear_status((int)device); }
int64_t read_checks() { return (int64_t)mt::read_and_clear_checks(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "meshtrain_b200 hand-written sm_100a kernels";
  m.def("gemm", &gemm, "tcgen05 GEMM with fused epilogue");
  m.def("layernorm_fwd", &layernorm_fwd);
  m.def("layernorm_bwd", &layernorm_bwd);
  m.def("rmsnorm_fwd", &rmsnorm_fwd);
  m.def("rmsnorm_bwd", &rmsnorm_bwd);
  m.def("embedding_fwd", &embedding_fwd);
  m.def("embedding_bwd", &embedding_bwd);
  m.def("colsum_", &colsum_);
  m.def("swiglu_bwd", &swiglu_bwd);
  m.def("rope_", &rope_);
  m.def("cross_entropy_", &cross_entropy_);
  m.def("qk_norm_rope_fwd", &qk_norm_rope_fwd);
  m.def("qk_norm_rope_bwd", &qk_norm_rope_bwd);
  m.def("dropout", &dropout);
  m.def("token_logprobs", &token_logprobs);
  m.def("token_logprobs_bwd", &token_logprobs_bwd);
  m.def("policy_loss", &policy_loss);
  m.def("preference_loss", &preference_loss);
  m.def("adam_", &adam_);
  m.def("cast_bf16_", &cast_bf16_);
  m.def("attention_fwd", &attention_fwd);
  m.def("attention_bwd", &attention_bwd);
  m.def("read_status", &read_status);
  m.def("read_checks", &read_checks);
  m.def("debug_checks_built", &mt::debug_checks_built);
}
