// Log-probabilities and distillation over the vocabulary for torch tensors: argument checks, outputs and
// workspaces from torch's caching allocator (stream-ordered, so that calls on several streams and
// captured graphs share nothing), and the autograd nodes. The nodes are C++ because a small batch is
// bound by the host: a forward and backward pass of 4 x 8192 takes 59 us, with Python nodes it took 86.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <functional>
#include <limits>

#include "api.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// ---------------------------------------------------------------------------------------------
// Operands
// ---------------------------------------------------------------------------------------------
ob::LogitType logit_type(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return ob::LogitType::F32;
    case torch::kBFloat16: return ob::LogitType::BF16;
    case torch::kFloat16: return ob::LogitType::F16;
    default: TORCH_CHECK_TYPE(false, "logits must be float32, bfloat16 or float16");
  }
}

// Any strides over the leading dimensions that two of them can express (slices of a padded vocabulary,
// `logits[:, :-1]`, expanded batches); false where the rows have to be copied together first.
bool rows_view(const Tensor& t, ob::RowsView& view) {
  const int64_t vocab = t.size(-1);
  if (vocab > 1 && t.stride(-1) != 1) return false;
  int64_t sizes[2] = {1, 1}, strides[2] = {0, 0};  // innermost first
  int used = 0;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    const int64_t n = t.size(d), st = t.stride(d);
    if (n == 1) continue;
    if (used > 0 && st == strides[used - 1] * sizes[used - 1]) {
      sizes[used - 1] *= n;
    } else if (used < 2) {
      sizes[used] = n;
      strides[used] = st;
      ++used;
    } else {
      return false;
    }
  }
  view.base = t.data_ptr();
  view.inner = sizes[0];
  view.inner_stride = strides[0];
  view.outer_stride = strides[1];
  return true;
}

struct LogitRows {
  Tensor t;  // keeps a copy alive
  ob::RowsView view;
  ob::LogitType type;
  int64_t rows;
  int vocab;
};
LogitRows logit_rows(const Tensor& logits) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits need a vocabulary dimension");
  TORCH_CHECK_VALUE(logits.size(-1) < (1ll << 31) - 1024, "vocabulary too large");
  LogitRows r;
  r.t = logits;
  r.type = logit_type(logits);
  if (!rows_view(r.t, r.view)) {
    r.t = logits.contiguous();
    TORCH_CHECK(rows_view(r.t, r.view));
  }
  r.vocab = (int)logits.size(-1);
  r.rows = logits.numel() / r.vocab;
  return r;
}

ob::RowsView pitched(void* base, int64_t pitch, int64_t rows) { return ob::RowsView{base, 0, pitch, rows}; }

// A tensor for the gradient of `logits`, in their layout if that has no more than a few gaps: its rows
// then start at the same distance from a 16-byte boundary and whole vectors can be stored (a slice of
// a padded or odd vocabulary, `logits[:, :-1]`).
Tensor gradient_like(const Tensor& logits, const LogitRows& l, ob::RowsView& view) {
  const int64_t item = logits.element_size();
  const int64_t offset = reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16 / item;
  const ob::RowsView& v = l.view;
  const int64_t outer = l.rows > 0 ? l.rows / v.inner : 0;
  const int64_t span = (outer - 1) * v.outer_stride + (v.inner - 1) * v.inner_stride + l.vocab;
  const bool apart = (v.inner <= 1 || v.inner_stride >= l.vocab) &&
                     (outer <= 1 || v.outer_stride >= (v.inner - 1) * v.inner_stride + l.vocab);
  Tensor out;
  if (l.rows > 0 && l.t.is_same(logits) && apart && span <= 2 * logits.numel() &&
      (offset != 0 || !logits.is_contiguous()))
    out = torch::empty({offset + span}, logits.options()).as_strided(logits.sizes(), logits.strides(), offset);
  else
    out = torch::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  TORCH_CHECK(rows_view(out, view));
  return out;
}

template <typename S>
S* data(const Tensor& t) {
  return t.defined() ? t.data_ptr<S>() : nullptr;
}
float4* stats_of(const Tensor& t) { return reinterpret_cast<float4*>(data<float>(t)); }

// A contiguous operand with `numel` elements of type `type` on `device`; undefined stays undefined.
Tensor operand(const OptTensor& t, c10::Device device, torch::ScalarType type, int64_t numel,
               const char* name) {
  if (!t.has_value() || !t->defined()) return Tensor();
  TORCH_CHECK_VALUE(t->device() == device, name, " must be on the device of the logits");
  TORCH_CHECK_VALUE(t->numel() == numel, name, " must have ", numel, " elements, has ", t->numel());
  return t->to(type).contiguous();
}

Tensor f32(const Tensor& like, at::IntArrayRef sizes) {
  return torch::empty(sizes, like.options().dtype(torch::kFloat32));
}

int64_t check_top(int64_t top, int64_t vocab) {
  TORCH_CHECK_VALUE(top >= 0 && top <= std::min<int64_t>(ob::kMaxAlternatives, vocab),
                    "top must be between 0 and ", std::min<int64_t>(ob::kMaxAlternatives, vocab));
  return top;
}
int64_t check_list(const Tensor& tokens) {
  const int64_t k = tokens.dim() > 0 ? tokens.size(-1) : 0;
  TORCH_CHECK_VALUE(k >= 1 && k <= ob::kMaxAlternatives, "a teacher's list has 1 to ",
                    ob::kMaxAlternatives, " entries");
  return k;
}

// The gradients are formulas that autograd does not see: with create_graph they come with a node that
// raises when somebody differentiates them again.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads) {
    if (!g.defined()) continue;
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "the vocabulary operators are differentiable once", 1);
    Tensor d = g.detach();
    d.set_requires_grad(true);
    g = (*node)({d})[0];
  }
  return grads;
}

// The nodes take an absent tensor as an empty optional.
OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// ---------------------------------------------------------------------------------------------
// On given logits
// ---------------------------------------------------------------------------------------------
struct TokenResults {
  Tensor logprobs, entropy, top_logprobs, top_tokens, stats;
  // Those that were asked for, in this order.
  variable_list list() const {
    variable_list out;
    for (const Tensor* t : {&logprobs, &entropy, &top_logprobs, &top_tokens})
      if (t->defined()) out.push_back(*t);
    return out;
  }
};
TokenResults empty_results(const Tensor& like, at::IntArrayRef lead, int64_t rows, bool tokens,
                           bool entropy, int64_t top) {
  TokenResults r;
  if (tokens) r.logprobs = f32(like, lead);
  if (entropy) r.entropy = f32(like, lead);
  if (top > 0) {
    auto sizes = lead.vec();
    sizes.push_back(top);
    r.top_logprobs = f32(like, sizes);
    r.top_tokens = torch::empty(sizes, like.options().dtype(torch::kInt64));
  }
  r.stats = f32(like, {rows, 4});
  return r;
}

void run_logprobs(const LogitRows& l, const int64_t* tokens, double inv_temperature, int64_t ignore_index,
                  const TokenResults& out, int64_t first, int64_t top) {
  ob::TokenLogprobsArgs a = {};
  auto at_row = [&](auto* p, int64_t width) { return p == nullptr ? nullptr : p + first * width; };
  a.tokens = at_row(tokens, 1);
  a.logprobs = at_row(data<float>(out.logprobs), 1);
  a.entropy = at_row(data<float>(out.entropy), 1);
  a.top_logprobs = at_row(data<float>(out.top_logprobs), top);
  a.top_tokens = at_row(data<int64_t>(out.top_tokens), top);
  a.stats = stats_of(out.stats) + first;
  a.ignore_index = ignore_index;
  a.inv_temperature = (float)inv_temperature;
  a.vocab = l.vocab;
  a.top = (int)top;
  ob::token_logprobs(l.view, l.type, a, l.rows, current_stream());
}

// Arguments of the gradient of log-probabilities: whatever came in, fp32 and contiguous.
struct TokenGrads {
  Tensor logprobs, entropy, top;
  bool any() const { return logprobs.defined() || entropy.defined() || top.defined(); }
  TokenGrads(const variable_list& grads, bool tokens, bool entropies, bool tops) {
    size_t i = 0;
    auto next = [&](bool there) {
      if (!there) return Tensor();
      const Tensor& g = grads[i++];
      return g.defined() ? g.to(torch::kFloat32).contiguous() : Tensor();
    };
    logprobs = next(tokens);
    entropy = next(entropies);
    top = next(tops);
  }
};

void run_logprobs_grad(const LogitRows& l, const Tensor& stats, const Tensor& tokens,
                       const Tensor& top_tokens, const TokenGrads& g, double inv_temperature,
                       int64_t first, ob::LogitType out_type, const ob::RowsView& out) {
  ob::VocabGradArgs a = {};
  auto at_row = [&](auto* p, int64_t width) { return p == nullptr ? nullptr : p + first * width; };
  const int64_t top = g.top.defined() ? g.top.size(-1) : 0;
  a.stats = stats_of(stats) + first;
  a.out = out;
  a.grad = at_row(data<float>(g.logprobs), 1);
  a.grad_entropy = at_row(data<float>(g.entropy), 1);
  a.grad_top = at_row(data<float>(g.top), top);
  a.tokens = at_row(data<int64_t>(tokens), 1);
  a.top_tokens = top > 0 ? at_row(data<int64_t>(top_tokens), top) : nullptr;
  a.inv_temperature = (float)inv_temperature;
  a.vocab = l.vocab;
  a.top = (int)top;
  ob::vocab_grad(l.view, l.type, out_type, a, l.rows, false, current_stream());
}

struct TokenLogprobsFn : torch::autograd::Function<TokenLogprobsFn> {
  static TokenResults compute(const Tensor& logits, const Tensor& tokens, double inv_temperature,
                              bool entropy, int64_t top, int64_t ignore_index) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const LogitRows l = logit_rows(logits);
    TokenResults r = empty_results(logits, logits.sizes().slice(0, logits.dim() - 1), l.rows,
                                   tokens.defined(), entropy, top);
    run_logprobs(l, data<int64_t>(tokens), inv_temperature, ignore_index, r, 0, top);
    return r;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& given,
                               double inv_temperature, bool entropy, int64_t top, int64_t ignore_index) {
    const Tensor tokens = given.value_or(Tensor());
    TokenResults r = compute(logits, tokens, inv_temperature, entropy, top, ignore_index);
    ctx->set_materialize_grads(false);
    if (top > 0) ctx->mark_non_differentiable({r.top_tokens});
    ctx->save_for_backward({logits, tokens, r.top_tokens, r.stats});
    ctx->saved_data["inv"] = inv_temperature;
    ctx->saved_data["entropy"] = entropy;
    return r.list();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1], &top_tokens = saved[2], &stats = saved[3];
    const TokenGrads g(grads, tokens.defined(), ctx->saved_data["entropy"].toBool(), top_tokens.defined());
    variable_list out(6);
    if (!g.any()) return out;
    const c10::cuda::CUDAGuard guard(logits.device());
    const LogitRows l = logit_rows(logits);
    ob::RowsView to;
    out[0] = gradient_like(logits, l, to);
    run_logprobs_grad(l, stats, tokens, top_tokens, g, ctx->saved_data["inv"].toDouble(), 0, l.type, to);
    return once(std::move(out));
  }
};

variable_list token_logprobs(const Tensor& logits, const OptTensor& tokens, double inv_temperature,
                             bool entropy, int64_t top, int64_t ignore_index) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() >= 1, "logits must be a CUDA tensor");
  const int64_t vocab = logits.size(-1);
  check_top(top, vocab);
  const Tensor t = operand(tokens, logits.device(), torch::kInt64, vocab > 0 ? logits.numel() / vocab : 0,
                           "tokens");
  if (!wants_grad(logits))
    return TokenLogprobsFn::compute(logits, t, inv_temperature, entropy, top, ignore_index).list();
  return TokenLogprobsFn::apply(logits, optional_of(t), inv_temperature, entropy, top, ignore_index);
}

// `loss`, `stats`, `picked` of `rows` rows of lists from row `first` on.
ob::DistillationArgs distillation_args(const Tensor& teacher, const Tensor& tokens, double inv_temperature,
                                       bool tail, const Tensor& loss, const Tensor& stats, int vocab,
                                       int64_t first) {
  ob::DistillationArgs a = {};
  a.top = (int)tokens.size(-1);
  a.teacher = data<float>(teacher) + first * a.top;
  a.tokens = data<int64_t>(tokens) + first * a.top;
  a.loss = data<float>(loss) + first;
  a.stats = stats_of(stats) + first;
  a.inv_temperature = (float)inv_temperature;
  a.vocab = vocab;
  a.tail = tail ? 1 : 0;
  return a;
}
ob::VocabGradArgs distillation_grad_args(const Tensor& teacher, const Tensor& tokens, const Tensor& stats,
                                         const Tensor& grad, double inv_temperature, bool tail, int vocab,
                                         int64_t first) {
  ob::VocabGradArgs a = {};
  a.top = (int)tokens.size(-1);
  a.stats = stats_of(stats) + first;
  a.grad = data<float>(grad) + first;
  a.teacher = data<float>(teacher) + first * a.top;
  a.tokens = data<int64_t>(tokens) + first * a.top;
  a.inv_temperature = (float)inv_temperature;
  a.vocab = vocab;
  a.tail = tail ? 1 : 0;
  return a;
}

struct DistillationFn : torch::autograd::Function<DistillationFn> {
  static std::pair<Tensor, Tensor> compute(const Tensor& logits, const Tensor& teacher,
                                           const Tensor& tokens, double inv_temperature, bool tail) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const LogitRows l = logit_rows(logits);
    Tensor loss = f32(logits, logits.sizes().slice(0, logits.dim() - 1));
    Tensor stats = f32(logits, {l.rows, 4});
    if (l.rows > 0)
      ob::distillation_loss(l.view, l.type,
                            distillation_args(teacher, tokens, inv_temperature, tail, loss, stats, l.vocab, 0),
                            l.rows, current_stream());
    return {loss, stats};
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher,
                        const Tensor& tokens, double inv_temperature, bool tail) {
    auto [loss, stats] = compute(logits, teacher, tokens, inv_temperature, tail);
    ctx->save_for_backward({logits, teacher, tokens, stats});
    ctx->saved_data["inv"] = inv_temperature;
    ctx->saved_data["tail"] = tail;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& logits = saved[0];
    const c10::cuda::CUDAGuard guard(logits.device());
    const LogitRows l = logit_rows(logits);
    const Tensor g = grads[0].to(torch::kFloat32).contiguous();
    variable_list out(5);
    ob::RowsView to;
    out[0] = gradient_like(logits, l, to);
    if (l.rows > 0) {
      ob::VocabGradArgs a =
          distillation_grad_args(saved[1], saved[2], saved[3], g, ctx->saved_data["inv"].toDouble(),
                                 ctx->saved_data["tail"].toBool(), l.vocab, 0);
      a.out = to;
      ob::vocab_grad(l.view, l.type, l.type, a, l.rows, true, current_stream());
    }
    return once(std::move(out));
  }
};

Tensor distillation_loss(const Tensor& logits, const Tensor& teacher, const Tensor& tokens,
                         double inv_temperature, bool tail) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() >= 1, "logits must be a CUDA tensor");
  const int64_t entries = check_list(tokens) * (logits.size(-1) > 0 ? logits.numel() / logits.size(-1) : 0);
  const Tensor p = operand(teacher, logits.device(), torch::kFloat32, entries, "teacher_logprobs");
  const Tensor t = operand(tokens, logits.device(), torch::kInt64, entries, "teacher_tokens");
  if (!wants_grad(logits)) return DistillationFn::compute(logits, p, t, inv_temperature, tail).first;
  return DistillationFn::apply(logits, p, t, inv_temperature, tail);
}

// ---------------------------------------------------------------------------------------------
// From hidden states
// ---------------------------------------------------------------------------------------------
bool aligned_rows(const Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1))) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
Tensor bf16_rows(const Tensor& t) {  // (rows, width) bf16 as the TMA can read it
  Tensor r = t.detach().reshape({-1, t.size(-1)}).to(torch::kBFloat16);
  if (!aligned_rows(r)) r = r.clone(at::MemoryFormat::Contiguous);
  return r;
}
int64_t pitch_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct Head {
  Tensor hidden, weight;  // bf16 rows
  int64_t n, vocab, width;
  // Rows [first, first + rows) as the kernels take them.
  ob::LinearHead part(int64_t first, int64_t rows) const {
    ob::LinearHead h;
    h.ldh = pitch_of(hidden);
    h.ldw = pitch_of(weight);
    h.hidden = static_cast<const char*>(hidden.data_ptr()) + 2 * first * h.ldh;
    h.weight = weight.data_ptr();
    h.M = (int)rows;
    h.N = (int)vocab;
    h.K = (int)width;
    return h;
  }
};
Head make_head(const Tensor& hidden, const Tensor& weight16) {
  TORCH_CHECK_VALUE(hidden.size(-1) == weight16.size(1) && hidden.size(-1) % 8 == 0 && hidden.size(-1) > 0,
                    "the hidden width must be a positive multiple of 8");
  TORCH_CHECK_VALUE(weight16.size(0) >= 1 && weight16.size(0) < (1 << 30), "bad vocabulary size");
  Head h;
  h.hidden = bf16_rows(hidden);
  h.weight = bf16_rows(weight16);
  h.n = h.hidden.size(0);
  h.vocab = h.weight.size(0);
  h.width = h.weight.size(1);
  return h;
}

// Rows whose `bytes` each fill `chunk_bytes`, in whole row tiles of the product.
int64_t chunk_rows(const Head& h, int64_t bytes, int64_t chunk_bytes) {
  const int64_t rows = std::max<int64_t>(256, chunk_bytes / bytes / 256 * 256);
  return std::min<int64_t>(std::min<int64_t>(rows, 1 << 24), std::max<int64_t>(h.n, 1));
}

void gemm(const void* a, const void* b, void* c, int64_t m, int64_t n, int64_t k, int64_t batches, bool a_mn,
          int64_t lda, int64_t ldb, int64_t ldc, int64_t stride_a, int64_t stride_b, int64_t stride_c,
          bool out_f32, bool add) {
  // a: (m, k) or, with a_mn, (k, m); b: (k, n); c: (m, n)
  ob::gemm_bf16(a, b, c, (int)m, (int)n, (int)k, (int)batches, a_mn, true, lda, ldb, ldc, stride_a,
                stride_b, stride_c, batches > 1, batches > 1, (int)batches, out_f32, 1, add, 1.f, nullptr,
                nullptr, a_mn ? k : m, k, ob::device_sm_count(), nullptr, 0, 0, 0.f, current_stream());
}

// Pieces to cut the sum over the vocabulary into for d (rows x vocab) W (vocab x width), which has few
// output tiles: the count with the least estimated time, from whole waves of tiles (pairs of SMs take
// 256 x 256 above 128 rows, single ones 128 x 256) at the measured product rate, and a write and a read
// of every piece. 8188 x 768 over 50304: one piece 590 us, three 465; 100 x 1024 over 131072: 741, 74.
int64_t reduction_cuts(int64_t rows, int64_t width, int64_t vocab) {
  const bool pairs = rows > 128;
  const int64_t tile = pairs ? 256 : 128, units = ob::device_sm_count() / (pairs ? 2 : 1);
  const int64_t tiles = ((rows + tile - 1) / tile) * ((width + 255) / 256);
  const double whole = 2.0 * tile * 256 * vocab / (pairs ? 22e12 : 9e12);
  int64_t best = 1;
  double best_time = std::numeric_limits<double>::infinity();
  for (int64_t cuts = 1; cuts <= std::max<int64_t>(1, std::min<int64_t>(64, vocab / 512)); ++cuts) {
    double time = (double)((tiles * cuts + units - 1) / units) * whole / cuts;
    if (cuts > 1) time += 4e-6 + 8.0 * cuts * rows * width / 5e12;
    if (time < best_time) {
      best_time = time;
      best = cuts;
    }
  }
  return best;
}

// Up to this many rows the gradient with respect to the logits is held as the sum of two bf16 matrices:
// the products are bound by the weight then, and with few rows the rounding of single elements (the
// target's, near 1) shows in the results: error 2.7e-3 against 1.7e-3 of the results' own rounding at
// 4 x 1256, 1.7e-3 with the pair.
constexpr int64_t kPairRows = 256;

// dh (n x width) = sum over the `copies` blocks of n rows in d of d W, the pieces added in a fixed order.
void hidden_gradient(const Head& h, const Tensor& d, int64_t n, int64_t copies, int64_t pitch,
                     const Tensor& dh, int64_t first) {
  char* out = static_cast<char*>(dh.data_ptr()) + 2 * first * h.width;
  const int64_t ldw = pitch_of(h.weight), rows = n * copies;
  const int64_t cuts = reduction_cuts(rows, h.width, h.vocab);
  if (cuts * copies == 1) {
    gemm(d.data_ptr(), h.weight.data_ptr(), out, rows, h.width, h.vocab, 1, false, pitch, ldw, h.width, 0, 0,
         0, false, false);
    return;
  }
  const int64_t piece = (h.vocab + cuts * 64 - 1) / (cuts * 64) * 64;
  const int64_t whole = h.vocab / piece, rest = h.vocab - whole * piece;
  const int64_t count = whole + (rest > 0 ? 1 : 0);
  Tensor parts = f32(d, {count, rows, h.width});
  float* p = parts.data_ptr<float>();
  if (whole > 0)
    gemm(d.data_ptr(), h.weight.data_ptr(), p, rows, h.width, piece, whole, false, pitch, ldw, h.width, piece,
         piece * ldw, rows * h.width, true, false);
  if (rest > 0)
    gemm(static_cast<char*>(d.data_ptr()) + 2 * whole * piece,
         static_cast<char*>(h.weight.data_ptr()) + 2 * whole * piece * ldw, p + whole * rows * h.width, rows,
         h.width, rest, 1, false, pitch, ldw, h.width, 0, 0, 0, true, false);
  ob::sum_parts(p, out, false, n * h.width, (int)(count * copies), current_stream());
}

// Gradients of hidden states and weight from `gradient(first, rows, out, pitch, two)`, which writes
// d(loss) / d(logits) of some rows in bf16, the operand type of the two products that follow (with
// `two` as a pair, see kPairRows); both accumulate in fp32, the weight's over all chunks and in a fixed
// order.
using GradientOf = std::function<void(int64_t, int64_t, const Tensor&, int64_t, bool)>;
std::pair<Tensor, Tensor> head_backward(const Head& h, at::IntArrayRef hidden_sizes,
                                        torch::ScalarType hidden_type, torch::ScalarType weight_type,
                                        bool need_dh, bool need_dw, bool pairs, int64_t chunk_bytes,
                                        const GradientOf& gradient) {
  const auto options = h.hidden.options();
  Tensor dh, dw;
  if (h.n == 0) {
    if (need_dh) dh = torch::zeros(hidden_sizes, options.dtype(hidden_type));
    if (need_dw) dw = torch::zeros({h.vocab, h.width}, options.dtype(weight_type));
    return {dh, dw};
  }
  const int64_t step = chunk_rows(h, 2 * h.vocab, chunk_bytes);
  const int64_t pitch = (h.vocab + 7) / 8 * 8;
  const bool two = pairs && h.n <= kPairRows;
  const int64_t copies = two ? 2 : 1;
  Tensor d = torch::empty({copies * step, pitch}, options);
  const Tensor hidden = two && need_dw ? torch::cat({h.hidden, h.hidden}) : h.hidden;
  const int64_t ldh = pitch_of(hidden);
  if (need_dh) dh = torch::empty({h.n, h.width}, options);
  if (need_dw)  // the product of a single chunk can be rounded to the weight's type as it is written
    dw = torch::empty({h.vocab, h.width},
                      options.dtype(h.n <= step && weight_type == torch::kBFloat16 ? torch::kBFloat16
                                                                                   : torch::kFloat32));
  for (int64_t first = 0; first < h.n; first += step) {
    const int64_t rows = std::min(step, h.n - first);
    gradient(first, rows, d, pitch, two);
    if (need_dh) hidden_gradient(h, d, rows, copies, pitch, dh, first);
    if (need_dw)
      gemm(d.data_ptr(), static_cast<char*>(hidden.data_ptr()) + 2 * first * ldh, dw.data_ptr(), h.vocab,
           h.width, rows * copies, 1, true, pitch, ldh, h.width, 0, 0, 0, dw.scalar_type() == torch::kFloat32,
           first > 0);
  }
  if (need_dh) dh = dh.view(hidden_sizes).to(hidden_type);
  if (need_dw) dw = dw.to(weight_type);
  return {dh, dw};
}

// With a top list, which needs every logit: fp32 logits of some rows at a time (bf16 ones would put a
// log-probability off by 2^-9 of the logit), then `rows(logits, first)`.
void over_logits(const Head& h, int64_t first, int64_t rows, int64_t chunk_bytes,
                 const std::function<void(const LogitRows&, int64_t)>& use) {
  const int64_t step = chunk_rows(h, 4 * h.vocab, chunk_bytes);
  const int64_t pitch = (h.vocab + 3) / 4 * 4;
  Tensor logits = f32(h.hidden, {std::min(step, rows), pitch});
  for (int64_t at = 0; at < rows; at += step) {
    const int64_t n = std::min(step, rows - at);
    const ob::LinearHead p = h.part(first + at, n);
    ob::gemm_bf16(p.hidden, p.weight, logits.data_ptr(), p.M, p.N, p.K, 1, false, false, p.ldh, p.ldw, pitch,
                  0, 0, 0, false, false, 1, true, 1, false, 1.f, nullptr, nullptr, p.M, p.N,
                  ob::device_sm_count(), nullptr, 0, 0, 0.f, current_stream());
    LogitRows l;
    l.t = logits;
    l.view = pitched(logits.data_ptr(), pitch, n);
    l.type = ob::LogitType::F32;
    l.rows = n;
    l.vocab = (int)h.vocab;
    use(l, first + at);
  }
}

// Rows whose partial statistics fit a chunk.
int64_t statistics_rows(const Head& h, int64_t chunk_bytes) {
  return chunk_rows(h, 16 * ob::linear_head_halves((int)h.vocab), chunk_bytes);
}
Tensor partial_for(const Head& h, int64_t rows) {
  return f32(h.hidden, {ob::linear_head_halves((int)h.vocab), ob::linear_head_rows(rows), 4});
}

struct LinearTokenLogprobsFn : torch::autograd::Function<LinearTokenLogprobsFn> {
  // `picked`: logits of the tokens (without a top list), for the backward pass
  static TokenResults compute(const Tensor& hidden, const Tensor& weight16, const Tensor& tokens,
                              double inv_temperature, bool entropy, int64_t top, int64_t ignore_index,
                              int64_t chunk_bytes, Tensor& picked) {
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Head h = make_head(hidden, weight16);
    TokenResults r = empty_results(hidden, hidden.sizes().slice(0, hidden.dim() - 1), h.n, tokens.defined(),
                                   entropy, top);
    if (h.n == 0) return r;
    if (top > 0) {
      over_logits(h, 0, h.n, chunk_bytes, [&](const LogitRows& l, int64_t first) {
        run_logprobs(l, data<int64_t>(tokens), inv_temperature, ignore_index, r, first, top);
      });
      return r;
    }
    if (tokens.defined()) picked = f32(hidden, {h.n});
    const int64_t step = statistics_rows(h, chunk_bytes);
    Tensor partial = partial_for(h, step);
    for (int64_t first = 0; first < h.n; first += step) {
      const int64_t rows = std::min(step, h.n - first);
      auto at_row = [&](auto* p) { return p == nullptr ? nullptr : p + first; };
      ob::TokenLogprobsArgs a = {};
      a.tokens = at_row(data<int64_t>(tokens));
      a.logprobs = at_row(data<float>(r.logprobs));
      a.entropy = at_row(data<float>(r.entropy));
      a.stats = stats_of(r.stats) + first;
      a.ignore_index = ignore_index;
      a.inv_temperature = (float)inv_temperature;
      a.vocab = (int)h.vocab;
      ob::linear_token_logprobs(h.part(first, rows), a, stats_of(partial), at_row(data<float>(picked)),
                                current_stream());
    }
    return r;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                               const Tensor& weight16, const OptTensor& given, double inv_temperature,
                               bool entropy, int64_t top, int64_t ignore_index, int64_t chunk_bytes) {
    const Tensor tokens = given.value_or(Tensor());
    Tensor picked;
    TokenResults r =
        compute(hidden, weight16, tokens, inv_temperature, entropy, top, ignore_index, chunk_bytes, picked);
    ctx->set_materialize_grads(false);
    if (top > 0) ctx->mark_non_differentiable({r.top_tokens});
    ctx->save_for_backward({hidden, weight, weight16, tokens, r.top_tokens, r.stats, picked});
    ctx->saved_data["inv"] = inv_temperature;
    ctx->saved_data["entropy"] = entropy;
    ctx->saved_data["chunk"] = chunk_bytes;
    return r.list();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &hidden = saved[0], &weight = saved[1], &tokens = saved[3], &top_tokens = saved[4],
                 &stats = saved[5], &picked = saved[6];
    const TokenGrads g(grads, tokens.defined(), ctx->saved_data["entropy"].toBool(), top_tokens.defined());
    variable_list out(9);
    if (!g.any()) return out;
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Head h = make_head(hidden, saved[2]);
    const double inv = ctx->saved_data["inv"].toDouble();
    const int64_t chunk = ctx->saved_data["chunk"].toInt();
    Tensor coef = f32(hidden, {chunk_rows(h, 2 * h.vocab, chunk), 4});
    auto gradient = [&](int64_t first, int64_t rows, const Tensor& d, int64_t pitch, bool two) {
      if (top_tokens.defined()) {
        over_logits(h, first, rows, chunk, [&](const LogitRows& l, int64_t at) {
          run_logprobs_grad(l, stats, tokens, top_tokens, g, inv, at, ob::LogitType::BF16,
                            pitched(static_cast<char*>(d.data_ptr()) + 2 * (at - first) * pitch, pitch, l.rows));
        });
        return;
      }
      auto at_row = [&](auto* p) { return p == nullptr ? nullptr : p + first; };
      ob::VocabGradArgs a = {};
      a.stats = stats_of(stats) + first;
      a.out = pitched(d.data_ptr(), pitch, rows);
      a.grad = at_row(data<float>(g.logprobs));
      a.grad_entropy = at_row(data<float>(g.entropy));
      a.tokens = at_row(data<int64_t>(tokens));
      a.inv_temperature = (float)inv;
      a.vocab = (int)h.vocab;
      ob::linear_vocab_grad(h.part(first, rows), a, false, two, at_row(data<float>(picked)),
                            stats_of(coef), current_stream());
    };
    std::tie(out[0], out[1]) =
        head_backward(h, hidden.sizes(), hidden.scalar_type(), weight.scalar_type(),
                      ctx->needs_input_grad(0), ctx->needs_input_grad(1), !top_tokens.defined(), chunk,
                      gradient);
    return once(std::move(out));
  }
};

variable_list linear_token_logprobs(const Tensor& hidden, const Tensor& weight, const Tensor& weight16,
                                    const OptTensor& tokens, double inv_temperature, bool entropy,
                                    int64_t top, int64_t ignore_index, int64_t chunk_bytes) {
  TORCH_CHECK(hidden.is_cuda() && weight.device() == hidden.device() && hidden.dim() >= 1 &&
                  weight16.dim() == 2 && weight16.device() == hidden.device(),
              "hidden and weight must be on the same CUDA device");
  check_top(top, weight16.size(0));
  const Tensor t = operand(tokens, hidden.device(), torch::kInt64,
                           hidden.size(-1) > 0 ? hidden.numel() / hidden.size(-1) : 0, "tokens");
  if (!wants_grad(hidden) && !wants_grad(weight)) {
    Tensor picked;
    return LinearTokenLogprobsFn::compute(hidden, weight16, t, inv_temperature, entropy, top, ignore_index,
                                          chunk_bytes, picked)
        .list();
  }
  return LinearTokenLogprobsFn::apply(hidden, weight, weight16, optional_of(t), inv_temperature, entropy, top,
                                      ignore_index, chunk_bytes);
}

struct LinearDistillationFn : torch::autograd::Function<LinearDistillationFn> {
  static Tensor compute(const Tensor& hidden, const Tensor& weight16, const Tensor& teacher,
                        const Tensor& tokens, double inv_temperature, bool tail, int64_t chunk_bytes,
                        Tensor& stats, Tensor& picked) {
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Head h = make_head(hidden, weight16);
    const int64_t k = tokens.size(-1);
    Tensor loss = f32(hidden, hidden.sizes().slice(0, hidden.dim() - 1));
    stats = f32(hidden, {h.n, 4});
    picked = f32(hidden, {h.n, k});
    if (h.n == 0) return loss;
    const int64_t step = statistics_rows(h, chunk_bytes);
    Tensor partial = partial_for(h, step), marks;
    if (tail)
      marks = torch::empty({step, ob::linear_head_mark_words((int)h.vocab)},
                           h.hidden.options().dtype(torch::kInt32));
    for (int64_t first = 0; first < h.n; first += step) {
      const int64_t rows = std::min(step, h.n - first);
      ob::linear_distillation(
          h.part(first, rows),
          distillation_args(teacher, tokens, inv_temperature, tail, loss, stats, (int)h.vocab, first),
          stats_of(partial), data<float>(picked) + first * k, reinterpret_cast<uint32_t*>(data<int>(marks)),
          current_stream());
    }
    return loss;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const Tensor& weight16, const Tensor& teacher, const Tensor& tokens,
                        double inv_temperature, bool tail, int64_t chunk_bytes) {
    Tensor stats, picked;
    Tensor loss =
        compute(hidden, weight16, teacher, tokens, inv_temperature, tail, chunk_bytes, stats, picked);
    ctx->save_for_backward({hidden, weight, weight16, teacher, tokens, stats, picked});
    ctx->saved_data["inv"] = inv_temperature;
    ctx->saved_data["tail"] = tail;
    ctx->saved_data["chunk"] = chunk_bytes;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &hidden = saved[0], &weight = saved[1], &teacher = saved[3], &tokens = saved[4],
                 &stats = saved[5], &picked = saved[6];
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Head h = make_head(hidden, saved[2]);
    const Tensor g = grads[0].to(torch::kFloat32).contiguous();
    const int64_t chunk = ctx->saved_data["chunk"].toInt();
    Tensor coef = f32(hidden, {chunk_rows(h, 2 * h.vocab, chunk), 4});
    auto gradient = [&](int64_t first, int64_t rows, const Tensor& d, int64_t pitch, bool two) {
      ob::VocabGradArgs a =
          distillation_grad_args(teacher, tokens, stats, g, ctx->saved_data["inv"].toDouble(),
                                 ctx->saved_data["tail"].toBool(), (int)h.vocab, first);
      a.out = pitched(d.data_ptr(), pitch, rows);
      ob::linear_vocab_grad(h.part(first, rows), a, true, two, data<float>(picked) + first * a.top,
                            stats_of(coef), current_stream());
    };
    variable_list out(8);
    std::tie(out[0], out[1]) =
        head_backward(h, hidden.sizes(), hidden.scalar_type(), weight.scalar_type(),
                      ctx->needs_input_grad(0), ctx->needs_input_grad(1), true, chunk, gradient);
    return once(std::move(out));
  }
};

Tensor linear_distillation_loss(const Tensor& hidden, const Tensor& weight, const Tensor& weight16,
                                const Tensor& teacher, const Tensor& tokens, double inv_temperature,
                                bool tail, int64_t chunk_bytes) {
  TORCH_CHECK(hidden.is_cuda() && weight.device() == hidden.device() && hidden.dim() >= 1 &&
                  weight16.dim() == 2 && weight16.device() == hidden.device(),
              "hidden and weight must be on the same CUDA device");
  const int64_t entries =
      check_list(tokens) * (hidden.size(-1) > 0 ? hidden.numel() / hidden.size(-1) : 0);
  const Tensor p = operand(teacher, hidden.device(), torch::kFloat32, entries, "teacher_logprobs");
  const Tensor t = operand(tokens, hidden.device(), torch::kInt64, entries, "teacher_tokens");
  if (!wants_grad(hidden) && !wants_grad(weight)) {
    Tensor stats, picked;
    return LinearDistillationFn::compute(hidden, weight16, p, t, inv_temperature, tail, chunk_bytes, stats,
                                         picked);
  }
  return LinearDistillationFn::apply(hidden, weight, weight16, p, t, inv_temperature, tail, chunk_bytes);
}

}  // namespace

void register_vocab_ops(pybind11::module_& m) {
  m.attr("MAX_ALTERNATIVES") = ob::kMaxAlternatives;
  m.def("token_logprobs", &token_logprobs);
  m.def("distillation_loss", &distillation_loss);
  m.def("linear_token_logprobs", &linear_token_logprobs);
  m.def("linear_distillation_loss", &linear_distillation_loss);
}
