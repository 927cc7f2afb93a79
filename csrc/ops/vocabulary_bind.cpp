// Python bindings of the vocabulary operators: argument checks, outputs and workspaces from the tensor allocator, launches on
// the current stream of the operands' device. The operators whose kernels take a few microseconds are differentiable functions
// here rather than in Python, where the bookkeeping of one call costs more than its kernels (preference loss of 4 pairs of 300 tokens, both
// directions: 129 us with the function in Python).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>

#include "vocabulary.h"

namespace b200 {

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// Parts of a message as strings: numbers are not put through the error macros' streams, since an extension that was linked with a C++ library
// of its own formats them with facets that the library of torch does not share, which ends the process.
std::string text(int64_t v) { return std::to_string(v); }
std::string text(double v) { return std::to_string(v); }
std::string text(torch::ScalarType t) { return c10::toString(t); }
std::string text(const at::Device& d) { return d.str(); }
std::string text(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}

cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Scalar scalar_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return Scalar::kBf16;
    case torch::kFloat16: return Scalar::kF16;
    case torch::kFloat32: return Scalar::kF32;
    default: TORCH_CHECK(false, name, " must be bf16, fp16 or fp32, got ", text(t.scalar_type()));
  }
  return Scalar::kF32;
}

void check_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", text(like.device()), ", got ", text(t.device()));
}

void check_indices(const Tensor& t, const Tensor& like, const char* name) {
  check_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == torch::kInt64 || t.scalar_type() == torch::kInt32, name, " must be int64 or int32, got ",
      text(t.scalar_type()));
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// fp32 values of `rows` rows as a pointer and a stride (0 for a broadcast value)
const float* row_values(const Tensor& t, const Tensor& like, int64_t rows, const char* name, long long* stride) {
  check_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 && t.dim() == 1 && t.size(0) == rows, name, " must be fp32 [", text(rows), "]");
  *stride = t.stride(0);
  return t.data_ptr<float>();
}

const float* contiguous_f32(const Tensor& t, const Tensor& like, int64_t count, const char* name) {
  check_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 && t.is_contiguous() && t.numel() == count, name, " must be contiguous fp32 with ",
      text(count), " elements");
  return t.data_ptr<float>();
}

Tensor empty_f32(int64_t n, const Tensor& like) { return torch::empty({n}, like.options().dtype(torch::kFloat32)); }

Tensor empty_pairs(int64_t n, const Tensor& like) { return torch::empty({n, 2}, like.options().dtype(torch::kFloat32)); }
float2* pairs(const Tensor& t) { return reinterpret_cast<float2*>(t.data_ptr<float>()); }
const float2* checked_pairs(const Tensor& t, const Tensor& like, int64_t rows) {
  return reinterpret_cast<const float2*>(contiguous_f32(t, like, 2 * rows, "lse"));
}

// logits: [outer, inner, V] with a unit inner stride
RowMap row_map(const Tensor& logits) {
  TORCH_CHECK(logits.dim() == 3, "logits must be [outer, inner, V]");
  TORCH_CHECK(logits.stride(2) == 1 || logits.size(2) == 1, "logits must have a unit inner stride");
  TORCH_CHECK(logits.size(2) > 0 && logits.size(2) <= (1 << 29), "the vocabulary size must be in [1, 2^29]");
  TORCH_CHECK(logits.size(0) * logits.size(1) < (1LL << 31), "at most 2^31 - 1 rows of logits");
  return {std::max<int64_t>(logits.size(1), 1), logits.stride(0), logits.stride(1)};
}

std::tuple<Tensor, Tensor, Tensor> log_probs_fwd(const Tensor& logits, const Tensor& labels, double logit_scale, int64_t ignore_index,
    bool want_entropy) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  const Scalar type = scalar_of(logits, "logits");
  const RowMap map = row_map(logits);
  const int64_t rows = logits.size(0) * logits.size(1);
  check_indices(labels, logits, "labels");
  TORCH_CHECK(labels.numel() == rows, "labels must have one entry per row of logits");
  const c10::cuda::CUDAGuard guard(logits.device());
  // outputs are tensors of their own, not views: a caller may change them in place
  const auto f32 = logits.options().dtype(torch::kFloat32);
  Tensor log_probs = torch::empty(labels.sizes(), f32), lse = empty_pairs(rows, logits),
      entropy = want_entropy ? torch::empty(labels.sizes(), f32) : Tensor();
  token_log_probs_fwd(logits.data_ptr(), type, labels.data_ptr(), labels.scalar_type() == torch::kInt64, log_probs.data_ptr<float>(),
                      want_entropy ? entropy.data_ptr<float>() : nullptr, pairs(lse), rows, (int)logits.size(2), map, (float)logit_scale,
                      ignore_index, stream_of(logits));
  return {log_probs, entropy, lse};
}

// Gradient [outer, inner, V] in the logits' type; its rows start at multiples of 16 bytes (padded when V needs it).
Tensor log_probs_bwd(const Tensor& logits, const Tensor& labels, const Tensor& lse, const OptTensor& entropy, const Tensor& d_log_probs,
                     const OptTensor& d_entropy, double logit_scale, int64_t ignore_index) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  const Scalar type = scalar_of(logits, "logits");
  const RowMap map = row_map(logits);
  const int64_t outer = logits.size(0), inner = logits.size(1), V = logits.size(2), rows = outer * inner;
  check_indices(labels, logits, "labels");
  TORCH_CHECK(labels.numel() == rows, "labels must have one entry per row of logits");
  long long g_stride = 0, h_stride = 0;
  const float* g = row_values(d_log_probs, logits, rows, "d_log_probs", &g_stride);
  const float* h = d_entropy.has_value() ? row_values(*d_entropy, logits, rows, "d_entropy", &h_stride) : nullptr;
  TORCH_CHECK(h == nullptr || entropy.has_value(), "the entropy gradient needs the entropy of the forward pass");
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t per_16 = 16 / logits.element_size();
  const int64_t pitch = (V + per_16 - 1) / per_16 * per_16;
  Tensor grad = torch::empty({outer, inner, pitch}, logits.options()).narrow(2, 0, V);
  token_log_probs_bwd(logits.data_ptr(), type, labels.data_ptr(), labels.scalar_type() == torch::kInt64,
      checked_pairs(lse, logits, rows), h != nullptr ? contiguous_f32(*entropy, logits, rows, "entropy") : nullptr, g, g_stride, h,
      h_stride, grad.data_ptr(), rows, (int)V, map, pitch, (float)logit_scale, ignore_index, stream_of(logits));
  return grad;
}

void check_linear(const Tensor& x, const Tensor& w, const Tensor& labels) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == torch::kBFloat16 && w.scalar_type() == torch::kBFloat16,
      "hidden states and weight must be bf16 CUDA tensors");
  check_device(w, x, "weight");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1), "hidden states must be [T, H] and the weight [V, H]");
  TORCH_CHECK(x.stride(1) == 1 && w.stride(1) == 1, "hidden states and weight must have a unit inner stride");
  TORCH_CHECK(x.size(1) > 0 && x.size(1) % 8 == 0 && x.stride(0) % 8 == 0 && w.stride(0) % 8 == 0,
      "H and the row strides must be multiples of 8");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(x.data_ptr()) | reinterpret_cast<uintptr_t>(w.data_ptr())) % 16 == 0,
      "hidden states and weight must be 16-byte aligned");
  TORCH_CHECK(w.size(0) > 0 && w.size(0) <= (1 << 29) && x.size(1) < (1 << 30) && x.size(0) < (1LL << 31), "sizes out of range");
  check_indices(labels, x, "labels");
  TORCH_CHECK(labels.numel() == x.size(0), "labels must have one entry per row of hidden states");
}

int* status_of(const Tensor& status, const Tensor& like) {
  check_device(status, like, "status");
  TORCH_CHECK(status.scalar_type() == torch::kInt32 && status.numel() >= 1, "status must be int32");
  return status.data_ptr<int>();
}

// Rows that share one statistics buffer: 16 bytes per row and slice stay below 512 MB.
int64_t stats_rows(int64_t rows, int64_t slices) {
  const int64_t most = std::max<int64_t>(256, ((512LL << 20) / (16 * slices)) / 256 * 256);
  return std::min(rows, std::min<int64_t>(most, 1 << 20));
}

// A batch of more rows than one tile is compacted to its live rows first, and so is every batch that will be differentiated: what an
// ignored row holds must not reach the weight's gradient as 0 * NaN. A smaller batch without gradients gains nothing (a tile is computed whole).
constexpr int64_t kCompactAbove = 256;

// map: int32 [T + 1] = index [T], count, or empty where the batch is not compacted
LiveRows live_rows(const Tensor& map, int64_t T, int64_t base, int64_t rows) {
  LiveRows live = {nullptr, nullptr, (int)base, (int)rows};
  if (map.numel() == 0) return live;
  TORCH_CHECK(map.is_cuda() && map.scalar_type() == torch::kInt32 && map.is_contiguous() && map.numel() == T + 1,
      "the row map must be int32 [T + 1]");
  live.index = map.data_ptr<int>();
  live.count = map.data_ptr<int>() + T;
  return live;
}

void* row_ptr(const Tensor& t, int64_t row) { return reinterpret_cast<char*>(t.data_ptr()) + row * t.stride(0) * t.element_size(); }

// Rows that a tensor map can describe: unit inner stride, row stride and base multiples of 16 bytes. Others are copied, also where they
// count as contiguous (at an odd address, or a single row of an odd stride).
Tensor mapped_rows(const Tensor& t) {
  const bool ok = t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// (log_probs, entropy, lse, the rows that were multiplied, row map, their logits if they are kept)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> linear_log_probs_fwd(const Tensor& x, const Tensor& w, const Tensor& labels,
    double logit_scale, int64_t ignore_index, bool want_entropy, bool differentiated, bool keep_logits, const Tensor& status) {
  check_linear(x, w, labels);
  int* st = status_of(status, x);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), H = x.size(1), V = w.size(0), slices = (V + kVocabSlice - 1) / kVocabSlice;
  const bool labels64 = labels.scalar_type() == torch::kInt64;
  const cudaStream_t stream = stream_of(x);
  Tensor log_probs = empty_f32(rows, x), lse = empty_pairs(rows, x), entropy = want_entropy ? empty_f32(rows, x) : Tensor();
  float* ent = want_entropy ? entropy.data_ptr<float>() : nullptr;
  const bool compact = differentiated || rows > kCompactAbove;
  Tensor map = torch::empty({compact ? rows + 1 : 0}, x.options().dtype(torch::kInt32)), xc = x;
  Tensor logits;
  if (keep_logits) logits = empty_f32(rows * ((V + 3) / 4 * 4), x).view({rows, (V + 3) / 4 * 4});
  if (rows == 0) return {log_probs, entropy, lse, xc, map, logits};
  if (compact) {
    int* m = map.data_ptr<int>();
    xc = torch::empty({rows, H}, x.options());
    vocab_compact_rows(labels.data_ptr(), labels64, ignore_index, (int)rows, (int)V, x.data_ptr(), x.stride(0), (int)H, m, m + rows,
        xc.data_ptr(), log_probs.data_ptr<float>(), ent, pairs(lse), stream);
  }
  const int64_t most = stats_rows(rows, slices);
  Tensor stats = empty_f32(most * slices * 4, x);
  for (int64_t r = 0; r < rows; r += most) {
    const LiveRows live = live_rows(map, rows, r, std::min(most, rows - r));
    vocab_gemm_stats(row_ptr(xc, r), w.data_ptr(), labels.data_ptr(), labels64, stats.data_ptr<float>(),
        keep_logits ? reinterpret_cast<float*>(row_ptr(logits, r)) : nullptr, keep_logits ? logits.stride(0) : 0, want_entropy, live,
        (int)V, (int)H, xc.stride(0), w.stride(0), (float)logit_scale, st, stream);
    token_log_probs_join(stats.data_ptr<float>(), (int)slices, kVocabSlice, labels.data_ptr(), labels64, log_probs.data_ptr<float>(),
        ent, pairs(lse), live, (int)V, (float)logit_scale, ignore_index, stream);
  }
  return {log_probs, entropy, lse, xc, map, logits};
}

// ------------------------------------------------------------------------- losses over sequences
PackedTokens packed_tokens(const Tensor& values, const OptTensor& cu, int64_t length, int64_t sequences, const OptTensor& mask) {
  PackedTokens p = {};
  p.T = values.numel();
  TORCH_CHECK(p.T < (1LL << 31) && sequences >= 0 && sequences < (1LL << 31) - 1, "at most 2^31 - 1 tokens and sequences");
  p.length = length;
  p.sequences = (int)sequences;
  if (cu.has_value()) {
    check_device(*cu, values, "cu_seqlens");
    TORCH_CHECK(cu->scalar_type() == torch::kInt32 && cu->is_contiguous() && cu->numel() == sequences + 1,
        "cu_seqlens must be contiguous int32 [sequences + 1]");
    p.cu = cu->data_ptr<int>();
  } else {
    TORCH_CHECK(length * sequences == p.T, "sequences of one length must cover all tokens");
  }
  if (mask.has_value()) {
    check_device(*mask, values, "mask");
    TORCH_CHECK((mask->scalar_type() == torch::kBool || mask->scalar_type() == torch::kUInt8) && mask->is_contiguous() && mask->numel() == p.T,
                "mask must be contiguous, boolean, one entry per token");
    p.mask = reinterpret_cast<const unsigned char*>(mask->data_ptr());
  }
  return p;
}

// (loss, chosen rewards, rejected rewards, slope [2 * pairs])
std::tuple<Tensor, Tensor, Tensor, Tensor> preference_fwd(const Tensor& log_probs, const OptTensor& reference, const OptTensor& cu,
    int64_t length, int64_t sequences, const OptTensor& mask, int64_t kind, double beta, double label_smoothing, bool average,
    int64_t reduction) {
  TORCH_CHECK(log_probs.is_cuda(), "log_probs must be a CUDA tensor");
  TORCH_CHECK(sequences > 0 && sequences % 2 == 0, "an even number of sequences is needed: chosen, then rejected");
  TORCH_CHECK(kind >= 0 && kind <= 2 && reduction >= 0 && reduction <= 2, "unknown loss type or reduction");
  const PackedTokens p = packed_tokens(log_probs, cu, length, sequences, mask);
  const float* lp = contiguous_f32(log_probs, log_probs, p.T, "log_probs");
  const float* ref = reference.has_value() ? contiguous_f32(*reference, log_probs, p.T, "reference_log_probs") : nullptr;
  const c10::cuda::CUDAGuard guard(log_probs.device());
  Tensor loss = reduction == 0 ? empty_f32(sequences / 2, log_probs) : torch::empty({}, log_probs.options());
  Tensor chosen = empty_f32(sequences / 2, log_probs), rejected = empty_f32(sequences / 2, log_probs),
      slope = empty_f32(sequences, log_probs), partials = empty_f32(packed_partials(p.T, p.sequences), log_probs);
  const PreferenceArgs args = {(PreferenceKind)kind, (float)beta, (float)label_smoothing, average, (int)reduction};
  preference_loss_fwd(lp, ref, p, args, partials.data_ptr<float>(), loss.data_ptr<float>(), chosen.data_ptr<float>(),
      rejected.data_ptr<float>(), slope.data_ptr<float>(), stream_of(log_probs));
  return {loss, chosen, rejected, slope};
}

Tensor preference_bwd(const Tensor& slope, const Tensor& d_loss, at::IntArrayRef shape, const OptTensor& cu, int64_t length,
    const OptTensor& mask) {
  const int64_t sequences = slope.numel();
  const c10::cuda::CUDAGuard guard(slope.device());
  Tensor grad = torch::empty(shape, slope.options());
  const PackedTokens p = packed_tokens(grad, cu, length, sequences, mask);
  contiguous_f32(slope, slope, sequences, "slope");
  long long stride = 0;
  const float* d = nullptr;
  if (d_loss.dim() == 0) {
    d = contiguous_f32(d_loss, slope, 1, "d_loss");
  } else {
    d = row_values(d_loss, slope, sequences / 2, "d_loss", &stride);
  }
  preference_loss_bwd(slope.data_ptr<float>(), d, stride, p, grad.data_ptr<float>(), stream_of(slope));
  return grad;
}

// (loss, kl, clipped share, factor [1], slope [T] or undefined, weight [sequences])
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> policy_fwd(const Tensor& log_probs, const Tensor& old_log_probs,
    const OptTensor& reference, const Tensor& advantages, bool per_token, const OptTensor& cu, int64_t length, int64_t sequences,
    const OptTensor& mask, double clip_low, double clip_high, double dual_clip, double kl_coef, int64_t reduction, bool want_slope) {
  TORCH_CHECK(log_probs.is_cuda(), "log_probs must be a CUDA tensor");
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "unknown reduction");
  const PackedTokens p = packed_tokens(log_probs, cu, length, sequences, mask);
  const float* lp = contiguous_f32(log_probs, log_probs, p.T, "log_probs");
  const float* old = contiguous_f32(old_log_probs, log_probs, p.T, "old_log_probs");
  const float* ref = reference.has_value() ? contiguous_f32(*reference, log_probs, p.T, "reference_log_probs") : nullptr;
  const float* adv = contiguous_f32(advantages, log_probs, per_token ? p.T : sequences, "advantages");
  const c10::cuda::CUDAGuard guard(log_probs.device());
  Tensor loss = torch::empty({}, log_probs.options()), kl = torch::empty_like(loss), clipped = torch::empty_like(loss),
      factor = empty_f32(1, log_probs), slope = want_slope ? empty_f32(p.T, log_probs) : Tensor();
  Tensor weight = empty_f32(reduction == 2 ? sequences : 0, log_probs), partials = empty_f32(packed_partials(p.T, p.sequences), log_probs);
  PolicyArgs args = {};
  args.log_low = std::log1p(-clip_low);
  args.log_high = std::log1p(clip_high);
  args.ratio_low = (float)(1.0 - clip_low);
  args.ratio_high = (float)(1.0 + clip_high);
  args.dual_clip = (float)dual_clip;
  args.kl_coef = (float)kl_coef;
  args.per_token_advantage = per_token;
  args.reduction = (int)reduction;
  policy_loss_fwd(lp, old, ref, adv, p, args, partials.data_ptr<float>(), {loss.data_ptr<float>(), kl.data_ptr<float>(),
      clipped.data_ptr<float>(), factor.data_ptr<float>()}, want_slope ? slope.data_ptr<float>() : nullptr, weight.data_ptr<float>(),
      stream_of(log_probs));
  return {loss, kl, clipped, factor, slope, weight};
}

Tensor policy_bwd(const Tensor& slope, const Tensor& factor, const Tensor& weight, const Tensor& d_loss, at::IntArrayRef shape,
    const OptTensor& cu, int64_t length, int64_t sequences, const OptTensor& mask, int64_t reduction) {
  const PackedTokens p = packed_tokens(slope, cu, length, sequences, mask);
  contiguous_f32(slope, slope, p.T, "slope");
  contiguous_f32(factor, slope, 1, "factor");
  contiguous_f32(weight, slope, reduction == 2 ? sequences : 0, "weight");
  contiguous_f32(d_loss, slope, 1, "d_loss");
  const c10::cuda::CUDAGuard guard(slope.device());
  Tensor grad = torch::empty(shape, slope.options());
  TORCH_CHECK(grad.numel() == p.T, "shape mismatch");
  policy_loss_bwd(slope.data_ptr<float>(), factor.data_ptr<float>(), weight.data_ptr<float>(), d_loss.data_ptr<float>(), p,
      (int)reduction, grad.data_ptr<float>(), stream_of(slope));
  return grad;
}

// ------------------------------------------------------------------------- embedding
Tensor embedding_lookup_(const Tensor& weight, const Tensor& ids, double scale, const Tensor& status) {
  TORCH_CHECK(weight.is_cuda() && weight.dim() == 2 && weight.is_contiguous(), "weight must be a contiguous [V, H] CUDA tensor");
  const Scalar type = scalar_of(weight, "weight");
  check_indices(ids, weight, "ids");
  TORCH_CHECK(ids.numel() <= (1LL << 30) && weight.size(1) < (1 << 30), "sizes out of range");
  int* st = status_of(status, weight);
  const c10::cuda::CUDAGuard guard(weight.device());
  auto shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor out = torch::empty(shape, weight.options());
  embedding_lookup(weight.data_ptr(), type, ids.data_ptr(), ids.scalar_type() == torch::kInt64, out.data_ptr(), ids.numel(),
      weight.size(0), (int)weight.size(1), (float)scale, st, stream_of(weight));
  return out;
}

// dweight (fp32, added to) or, without it, a new [V, H] gradient in dout's type.
Tensor embedding_gradient_(const Tensor& dout, const Tensor& ids, int64_t V, const OptTensor& dweight, double scale) {
  TORCH_CHECK(dout.is_cuda() && dout.is_contiguous() && dout.dim() >= 1, "dout must be a contiguous CUDA tensor");
  const Scalar type = scalar_of(dout, "dout");
  check_indices(ids, dout, "ids");
  const int64_t T = ids.numel(), H = dout.size(-1);
  TORCH_CHECK(dout.numel() == T * H && T <= (1LL << 30) && H < (1 << 30) && V >= 0 && V < (1LL << 31) - 1,
      "dout must be [T, H] for T ids; at most 2^30 tokens and 2^31 - 2 rows");
  const c10::cuda::CUDAGuard guard(dout.device());
  Tensor dw;
  if (dweight.has_value()) {
    dw = *dweight;
    contiguous_f32(dw, dout, V * H, "dweight");
  } else {
    dw = torch::empty({V, H}, dout.options());
  }
  Tensor workspace = torch::empty({embedding_gradient_workspace(T, (int)H, type)}, dout.options().dtype(torch::kUInt8));
  embedding_gradient(dout.data_ptr(), type, ids.data_ptr(), ids.scalar_type() == torch::kInt64, dw.data_ptr(), dweight.has_value(),
      workspace.data_ptr(), T, V, (int)H, (float)scale, stream_of(dout));
  return dw;
}

// ------------------------------------------------------------------------- launch sites of the backward passes
// The function of lm_engine/ops/timeline.py that opens a site by name, while sites are on. Kept for the process's life and touched with the
// interpreter's lock held; the flag alone is read without it, so that a pass pays nothing while they are off.
std::atomic<bool> sites_on{false};
py::object& site_function() {
  static py::object* f = new py::object(py::none());
  return *f;
}

void set_site(const py::object& function) {
  site_function() = function;
  sites_on = !function.is_none();
}

class Site {
 public:
  explicit Site(const char* name) {
    if (!sites_on.load(std::memory_order_relaxed)) return;
    const py::gil_scoped_acquire gil;
    if (site_function().is_none()) return;
    std::string error;
    try {
      auto context = std::make_unique<py::object>(site_function()(name));
      context->attr("__enter__")();
      context_ = context.release();
    } catch (py::error_already_set& e) {  // the engine's threads know the library's errors only
      error = e.what();
    }
    TORCH_CHECK(error.empty(), "launch site ", name, ": ", error);
  }
  ~Site() {
    if (context_ == nullptr) return;
    const py::gil_scoped_acquire gil;
    try {
      context_->attr("__exit__")(py::none(), py::none(), py::none());
    } catch (py::error_already_set& e) {
      e.discard_as_unraisable("launch site");
    }
    delete context_;
  }
  Site(const Site&) = delete;
  Site& operator=(const Site&) = delete;

 private:
  py::object* context_ = nullptr;
};

// ------------------------------------------------------------------------- differentiable functions
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The kernels' gradients have no derivative: with create_graph they are handed on with a node that says so when it is reached.
Tensor once(const Tensor& grad, const char* name) {
  if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
  Tensor leaf = grad.detach();
  leaf.set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " cannot be differentiated twice", 1);
  return (*node)({leaf})[0];
}

// Upstream gradient of a per-row output as fp32 values with one stride; a missing one is zeros.
Tensor row_gradient(const Tensor& grad, int64_t rows, const Tensor& like) {
  if (!grad.defined()) return torch::zeros({}, like.options().dtype(torch::kFloat32)).expand({rows});
  return grad.reshape({rows});
}

// [outer, inner, V] form of a batch of logits (a shifted [B, S, V] slice stays a view); a copy only where its layout has none.
Tensor rows3(const Tensor& logits) {
  Tensor t = logits.dim() == 1 ? logits.unsqueeze(0).unsqueeze(0) : logits.dim() == 2 ? logits.unsqueeze(0) : logits.dim() > 3 ? logits.flatten(0, -3) : logits;
  return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous();
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, double logit_scale,
      int64_t ignore_index, bool want_entropy) {
    auto [log_probs, entropy, lse] = log_probs_fwd(rows3(logits), labels.contiguous(), logit_scale, ignore_index, want_entropy);
    ctx->save_for_backward({logits, labels, lse, entropy});
    ctx->saved_data["logit_scale"] = logit_scale;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    if (!want_entropy) return {log_probs};
    return {log_probs, entropy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &labels = saved[1], &lse = saved[2], &entropy = saved[3];
    const bool has_h = grads.size() > 1 && grads[1].defined();
    if (!grads[0].defined() && !has_h) return variable_list(5);
    const int64_t rows = labels.numel();
    const Site site("token_log_probs.bwd");
    Tensor grad = log_probs_bwd(rows3(logits), labels.contiguous(), lse, entropy.defined() ? OptTensor(entropy) : OptTensor(),
        row_gradient(grads[0], rows, lse), has_h ? OptTensor(row_gradient(grads[1], rows, lse)) : OptTensor(),
        ctx->saved_data["logit_scale"].toDouble(), ctx->saved_data["ignore_index"].toInt());
    return {once(grad.view(logits.sizes()), "token_log_probs"), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// The engine's fp32 gradient buffer of a parameter (its Python attribute main_grad), if it has one. It is looked up in the backward
// pass, on the tensor that forward was given: a variable that was saved may come back as another one (recomputed, or moved away and
// back) without the attribute. So the functions keep weights in `saved_data`, which hands back what it was given, and so they do with
// the status word, whose value takes no part in a gradient.
OptTensor main_grad(const Tensor& weight) {
  const py::gil_scoped_acquire gil;
  const py::object p = py::cast(weight);
  const py::object target = py::getattr(p, "main_grad", py::none());
  if (target.is_none()) return OptTensor();
  Tensor t = py::cast<Tensor>(target).view(weight.sizes());
  TORCH_CHECK(t.is_cuda() && t.device() == weight.device() && t.scalar_type() == torch::kFloat32 && t.is_contiguous(),
      "main_grad must be a contiguous fp32 tensor on the weight's device");
  return t;
}

// Forward reduces the logits to 16 bytes per row and 128 columns. Backward needs them again: kept in fp32 where `keep_logits` says so, else
// formed a second time; either way they become, chunk of rows by chunk, their bf16 gradient, which is multiplied with the weight and
// the hidden states. Both ways see the same fp32 logits. The batch is compacted to the rows whose label counts, and all products end
// there.
struct LinearTokenLogProbs : torch::autograd::Function<LinearTokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& labels, double logit_scale,
      int64_t ignore_index, bool want_entropy, int64_t chunk, bool differentiated, bool keep_logits, const Tensor& status) {
    const Tensor w = mapped_rows(weight);
    auto [log_probs, entropy, lse, xc, map, logits] = linear_log_probs_fwd(mapped_rows(x), w, labels, logit_scale, ignore_index, want_entropy,
        differentiated, keep_logits, status);
    ctx->save_for_backward({xc, w, labels, lse, entropy, map, logits});
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["status"] = status;
    ctx->saved_data["logit_scale"] = logit_scale;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["chunk"] = chunk;
    ctx->set_materialize_grads(false);
    if (!want_entropy) return {log_probs};
    return {log_probs, entropy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &xc = saved[0], &w = saved[1], &labels = saved[2], &lse = saved[3], &entropy = saved[4], &map = saved[5],
        &logits = saved[6];
    const bool has_h = grads.size() > 1 && grads[1].defined();
    if (!grads[0].defined() && !has_h) return variable_list(10);
    const int64_t T = xc.size(0), H = xc.size(1), V = w.size(0);
    const int64_t chunk = std::max<int64_t>(std::min(ctx->saved_data["chunk"].toInt(), T), 1);
    const bool need_dx = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1);
    const Tensor g = row_gradient(grads[0], T, lse), h = has_h ? row_gradient(grads[1], T, lse) : Tensor();
    long long g_stride = 0, h_stride = 0;
    const float* gp = row_values(g, xc, T, "d_log_probs", &g_stride);
    const float* hp = has_h ? row_values(h, xc, T, "d_entropy", &h_stride) : nullptr;
    int* st = status_of(ctx->saved_data["status"].toTensor(), xc);
    const c10::cuda::CUDAGuard guard(xc.device());
    const cudaStream_t stream = stream_of(xc);
    Tensor dx, dw, dxc, partials;
    if (need_dx) {
      dx = torch::zeros({T, H}, xc.options());  // rows that take no part
      dxc = torch::empty({std::min(chunk, T), H}, xc.options());
      partials = empty_f32(balanced_partials(), xc);
    }
    OptTensor target;
    if (need_dw) {
      target = main_grad(ctx->saved_data["weight"].toTensor());
      // one chunk writes the weight's gradient in its own type; several add up in fp32
      if (target.has_value()) dw = *target;
      else if (chunk == T) dw = torch::empty({V, H}, w.options());
      else dw = torch::zeros({V, H}, w.options().dtype(torch::kFloat32));
    }
    Tensor dlogits = torch::empty({std::min(chunk, T), (V + 7) / 8 * 8}, xc.options()).narrow(1, 0, V);
    for (int64_t r = 0; r < T; r += chunk) {
      const int64_t n = std::min(chunk, T - r);
      const LiveRows live = live_rows(map, T, r, n);
      const Tensor dl = dlogits.narrow(0, 0, n), xr = xc.narrow(0, r, n);
      const bool labels64 = labels.scalar_type() == torch::kInt64;
      const float logit_scale = (float)ctx->saved_data["logit_scale"].toDouble();
      const int64_t ignore_index = ctx->saved_data["ignore_index"].toInt();
      const float* ent = has_h ? entropy.data_ptr<float>() : nullptr;
      {
        const Site site("loss.lm_head.dlogits");
        if (logits.defined())
          token_log_probs_grad_rows(reinterpret_cast<const float*>(row_ptr(logits, r)), logits.stride(0), labels.data_ptr(), labels64,
              pairs(lse), ent, gp, g_stride, hp, h_stride, dl.data_ptr(), dl.stride(0), live, (int)V, logit_scale, ignore_index, stream);
        else
          vocab_gemm_grad(xr.data_ptr(), w.data_ptr(), labels.data_ptr(), labels64, pairs(lse), ent, gp, g_stride, hp, h_stride,
              dl.data_ptr(), live, (int)V, (int)H, xc.stride(0), w.stride(0), dl.stride(0), logit_scale, ignore_index, st, stream);
      }
      if (need_dx) {
        const Site site("loss.lm_head.dgrad");
        balanced_gemm(dl.data_ptr(), w.data_ptr(), dxc.data_ptr(), partials.data_ptr<float>(), live, (int)H, (int)V, dl.stride(0),
            w.stride(0), st, stream);
        balanced_rows(dxc.data_ptr(), partials.data_ptr<float>(), live, dx.data_ptr(), (int)H, (int)V, stream);
      }
      if (need_dw) {
        const Site site("loss.lm_head.wgrad");
        gemm_bf16_2sm_live(dl.data_ptr(), xr.data_ptr(), dw.data_ptr(), (int)V, (int)H, (int)n, dl.stride(0), xr.stride(0),
            dw.stride(0), dw.scalar_type() == torch::kFloat32, live, st, stream);
      }
    }
    variable_list out(10);
    if (need_dx) out[0] = once(dx, "fused_linear_token_log_probs");
    if (need_dw && !target.has_value()) out[1] = once(dw.to(w.scalar_type()), "fused_linear_token_log_probs");
    return out;
  }
};

void check_logit_scale(double logit_scale) {
  TORCH_CHECK_VALUE(std::isfinite(logit_scale) && logit_scale > 0, "logit_scale must be positive and finite, got ", text(logit_scale));
}

void check_label_shape(const Tensor& labels, at::IntArrayRef shape, const Tensor& like) {
  TORCH_CHECK_VALUE(labels.scalar_type() == torch::kInt64 || labels.scalar_type() == torch::kInt32,
      "labels must be int64 or int32, got ", text(labels.scalar_type()));
  TORCH_CHECK_VALUE(labels.sizes() == shape, "labels must have the shape ", text(shape), ", got ", text(labels.sizes()));
  TORCH_CHECK_VALUE(labels.device() == like.device(), "labels must be on ", text(like.device()), ", got ", text(labels.device()));
}

variable_list token_log_probs(const Tensor& logits, const Tensor& labels, double logit_scale, int64_t ignore_index, bool return_entropy) {
  check_logit_scale(logit_scale);
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) > 0, "logits must have a last dimension of at least 1, got ",
      text(logits.sizes()));
  check_label_shape(labels, logits.sizes().slice(0, logits.dim() - 1), logits);
  return TokenLogProbs::apply(logits, labels, logit_scale, ignore_index, return_entropy);
}

variable_list linear_token_log_probs(const Tensor& x, const Tensor& w, const Tensor& labels, double logit_scale, int64_t ignore_index,
    bool return_entropy, int64_t chunk, int64_t keep_bytes, const Tensor& status) {
  check_logit_scale(logit_scale);
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.size(0) > 0 && w.size(1) > 0,
      "hidden states [..., H] and a weight [V, H] are needed, got ", text(x.sizes()), " and ", text(w.sizes()));
  TORCH_CHECK_VALUE(x.device() == w.device() && x.scalar_type() == w.scalar_type(),
      "hidden states and weight must be of one type on one device, got ", text(x.scalar_type()), " on ", text(x.device()), " and ",
      text(w.scalar_type()), " on ", text(w.device()));
  const auto shape = x.sizes().slice(0, x.dim() - 1);
  check_label_shape(labels, shape, x);
  const bool differentiated = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad());
  const bool keep = differentiated && 4.0 * (double)labels.numel() * (double)w.size(0) <= (double)keep_bytes;
  variable_list out = LinearTokenLogProbs::apply(x.reshape({labels.numel(), x.size(-1)}), w,
      labels.reshape({labels.numel()}).contiguous(), logit_scale, ignore_index, return_entropy, chunk, differentiated, keep, status);
  if (x.dim() != 2)
    for (auto& t : out) t = t.view(shape);
  return out;
}

// ---- losses: (log_probs as given, the same in fp32) so that the type conversion stays a differentiable step of its own
struct Sequences {
  int64_t count, length;
  OptTensor cu, mask;
};

Sequences check_sequences(const Tensor& log_probs, const OptTensor& cu_seqlens, const OptTensor& mask) {
  Sequences s = {};
  TORCH_CHECK_VALUE(log_probs.is_floating_point(), "log_probs must be floating point, got ", text(log_probs.scalar_type()));
  if (mask.has_value()) {
    TORCH_CHECK_VALUE(mask->sizes() == log_probs.sizes() && mask->device() == log_probs.device() && !mask->is_floating_point(),
        "mask must be boolean or integer, shaped ", text(log_probs.sizes()), " on ", text(log_probs.device()), ", got ",
        text(mask->scalar_type()), " ", text(mask->sizes()), " on ", text(mask->device()));
    s.mask = (mask->scalar_type() == torch::kBool ? *mask : mask->ne(0)).contiguous();
  }
  if (!cu_seqlens.has_value()) {
    TORCH_CHECK_VALUE(log_probs.dim() == 2, "log_probs must be [sequences, length], or [tokens] with cu_seqlens, got ",
        text(log_probs.sizes()));
    s.count = log_probs.size(0);
    s.length = log_probs.size(1);
    return s;
  }
  TORCH_CHECK_VALUE(log_probs.dim() == 1, "with cu_seqlens log_probs must be [tokens], got ", text(log_probs.sizes()));
  const Tensor& cu = *cu_seqlens;
  TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 1 && (cu.scalar_type() == torch::kInt32 || cu.scalar_type() == torch::kInt64) && cu.device() == log_probs.device(),
                    "cu_seqlens must be int32 or int64 [sequences + 1] on ", text(log_probs.device()), ", got ", text(cu.scalar_type()), " ", text(cu.sizes()), " on ", text(cu.device()));
  s.count = cu.numel() - 1;
  s.cu = cu.to(torch::kInt32).contiguous();
  return s;
}

Tensor check_values(const Tensor& t, at::IntArrayRef shape, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == shape && t.device() == like.device() && t.is_floating_point(), name,
      " must be floating point, shaped ", text(shape), " on ", text(like.device()), ", got ", text(t.scalar_type()), " ",
      text(t.sizes()), " on ", text(t.device()));
  TORCH_CHECK_VALUE(!t.requires_grad(), name,
      " must not require a gradient (detach it): the loss is differentiated with respect to log_probs alone");
  return t.to(torch::kFloat32).contiguous();
}

OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& log_probs, const OptTensor& reference, const OptTensor& cu,
      const OptTensor& mask, int64_t length, int64_t sequences, int64_t kind, double beta, double label_smoothing, bool average,
      int64_t reduction) {
    auto [loss, chosen, rejected, slope] = preference_fwd(log_probs, reference, cu, length, sequences, mask, kind, beta,
        label_smoothing, average, reduction);
    ctx->save_for_backward({slope, cu.value_or(Tensor()), mask.value_or(Tensor())});
    ctx->saved_data["shape"] = log_probs.sizes().vec();
    ctx->saved_data["length"] = length;
    ctx->mark_non_differentiable({chosen, rejected});
    ctx->set_materialize_grads(false);
    return {loss, chosen, rejected};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(11);
    if (!grads[0].defined()) return out;
    const Site site("preference_loss.bwd");
    out[0] = once(preference_bwd(saved[0], grads[0], ctx->saved_data["shape"].toIntVector(), optional(saved[1]),
        ctx->saved_data["length"].toInt(), optional(saved[2])), "preference_loss");
    return out;
  }
};

variable_list preference_loss(const Tensor& log_probs, const OptTensor& reference, const OptTensor& cu_seqlens, const OptTensor& mask,
    int64_t kind, double beta, double label_smoothing, bool average, int64_t reduction) {
  const Sequences s = check_sequences(log_probs, cu_seqlens, mask);
  TORCH_CHECK_VALUE(s.count > 0 && s.count % 2 == 0, "an even number of answers is needed (chosen, then rejected), got ", text(s.count));
  TORCH_CHECK_VALUE(std::isfinite(beta) && beta > 0, "beta must be positive and finite, got ", text(beta));
  TORCH_CHECK_VALUE(label_smoothing >= 0 && label_smoothing < 0.5 && (label_smoothing == 0 || kind == 0),
                    "label_smoothing must be in [0, 0.5) and goes with loss_type='sigmoid', got ", text(label_smoothing));
  OptTensor ref;
  if (reference.has_value()) ref = check_values(*reference, log_probs.sizes(), log_probs, "reference_log_probs");
  return PreferenceLoss::apply(log_probs.to(torch::kFloat32).contiguous(), ref, s.cu, s.mask, s.length, s.count, kind, beta,
      label_smoothing, average, reduction);
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& log_probs, const Tensor& old, const OptTensor& reference,
      const Tensor& advantages, bool per_token, const OptTensor& cu, const OptTensor& mask, int64_t length, int64_t sequences,
      double clip_low, double clip_high, double dual_clip, double kl_coef, int64_t reduction, bool want_slope) {
    auto [loss, kl, clipped, factor, slope, weight] = policy_fwd(log_probs, old, reference, advantages, per_token, cu, length,
        sequences, mask, clip_low, clip_high, dual_clip, kl_coef, reduction, want_slope);
    ctx->save_for_backward({slope, factor, weight, cu.value_or(Tensor()), mask.value_or(Tensor())});
    ctx->saved_data["shape"] = log_probs.sizes().vec();
    ctx->saved_data["length"] = length;
    ctx->saved_data["sequences"] = sequences;
    ctx->saved_data["reduction"] = reduction;
    ctx->mark_non_differentiable({kl, clipped});
    ctx->set_materialize_grads(false);
    return {loss, kl, clipped};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(15);
    if (!grads[0].defined()) return out;
    const Site site("policy_loss.bwd");
    out[0] = once(policy_bwd(saved[0], saved[1], saved[2], grads[0], ctx->saved_data["shape"].toIntVector(), optional(saved[3]),
        ctx->saved_data["length"].toInt(), ctx->saved_data["sequences"].toInt(), optional(saved[4]),
        ctx->saved_data["reduction"].toInt()), "policy_loss");
    return out;
  }
};

variable_list policy_loss(const Tensor& log_probs, const Tensor& old, const Tensor& advantages, const OptTensor& reference,
    const OptTensor& cu_seqlens, const OptTensor& mask, double clip_low, double clip_high, double dual_clip, double kl_coef,
    int64_t reduction) {
  const Sequences s = check_sequences(log_probs, cu_seqlens, mask);
  const Tensor o = check_values(old, log_probs.sizes(), log_probs, "old_log_probs");
  OptTensor ref;
  if (reference.has_value()) ref = check_values(*reference, log_probs.sizes(), log_probs, "reference_log_probs");
  const bool per_sequence = advantages.dim() == 1 && advantages.size(0) == s.count;  // also where there are as many tokens
  const bool per_token = !per_sequence && advantages.sizes() == log_probs.sizes();
  const Tensor a = per_token ? check_values(advantages, log_probs.sizes(), log_probs, "advantages")
                             : check_values(advantages, {s.count}, log_probs, "advantages");
  TORCH_CHECK_VALUE(clip_low >= 0 && clip_low <= 1 && clip_high >= 0, "clip_low must be in [0, 1] and clip_high at least 0, got ",
      text(clip_low), " and ", text(clip_high));
  TORCH_CHECK_VALUE(std::isfinite(kl_coef) && kl_coef >= 0, "kl_coef must be finite and at least 0, got ", text(kl_coef));
  TORCH_CHECK_VALUE(kl_coef == 0 || reference.has_value(), "kl_coef needs reference_log_probs");
  TORCH_CHECK_VALUE(dual_clip == 0 || (std::isfinite(dual_clip) && dual_clip > 1), "dual_clip must be finite and above 1, got ",
      text(dual_clip));
  const Tensor lp = log_probs.to(torch::kFloat32).contiguous();
  const bool want_slope = at::GradMode::is_enabled() && lp.requires_grad();
  return PolicyLoss::apply(lp, o, ref, a, per_token, s.cu, s.mask, s.length, s.count, clip_low, clip_high, dual_clip, kl_coef,
      reduction, want_slope);
}

struct EmbeddingSorted : torch::autograd::Function<EmbeddingSorted> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, const Tensor& status) {
    Tensor out = embedding_lookup_(weight.contiguous(), ids, scale, status);
    ctx->save_for_backward({ids});
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return variable_list(4);
    const Tensor weight = ctx->saved_data["weight"].toTensor();
    const OptTensor target = main_grad(weight);
    const Site site("embedding.bwd");
    Tensor dw = embedding_gradient_(grads[0].contiguous(), saved[0], weight.size(0), target, ctx->saved_data["scale"].toDouble());
    return {target.has_value() ? Tensor() : once(dw, "embedding_sorted"), Tensor(), Tensor(), Tensor()};
  }
};

Tensor embedding_sorted(const Tensor& weight, const Tensor& ids, double scale, const Tensor& status) {
  TORCH_CHECK_VALUE(weight.dim() == 2, "the embedding table must be [V, H], got ", text(weight.sizes()));
  TORCH_CHECK_VALUE(ids.scalar_type() == torch::kInt64 || ids.scalar_type() == torch::kInt32, "ids must be int64 or int32, got ",
      text(ids.scalar_type()));
  TORCH_CHECK_VALUE(ids.device() == weight.device(), "ids must be on ", text(weight.device()), ", got ", text(ids.device()));
  return EmbeddingSorted::apply(weight, ids.contiguous(), scale, status);
}

}  // namespace

void register_vocabulary(pybind11::module_& m) {
  m.def("token_log_probs", &token_log_probs, "log-probabilities of given tokens (and entropies) under rows of logits");
  m.def("linear_token_log_probs", &linear_token_log_probs, "the same from hidden states and the output weight");
  m.def("preference_loss", &preference_loss, "loss over pairs of answers: (loss, chosen rewards, rejected rewards)");
  m.def("policy_loss", &policy_loss, "clipped policy loss with a KL term: (loss, KL estimate, clipped share)");
  m.def("set_site", &set_site, "opens the launch sites of backward passes: a function of the name, or None");
  m.def("embedding_sorted", &embedding_sorted, "embedding whose gradient is summed in sorted token order");
}

}  // namespace b200
