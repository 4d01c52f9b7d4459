// lm_ops.cpp -- the language-model operators of an ensemble, in the `churten`
// operator library, over the C ABI of include/churten_lm.h (GPU tensors) and
// lm_cpu.cpp (CPU tensors).
//
// Every operator takes tensors with a leading replica dimension N, as the
// consolidated State's views have it, or all of them without (one replica, as
// inside torch.func.vmap). Tensors that are not a replica's own -- tokens,
// positions, the teacher's entries, labels, row weights -- may leave it out
// and are then shared by the replicas.
//
// Outputs are fresh and contiguous. Inputs may have any strides; one whose
// innermost dimension is not contiguous is copied first. Work runs on the
// current stream; workspaces come from torch's caching allocator.

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "lm_cpu.h"

namespace churten {
namespace {

constexpr int64_t kMaxReplicas = 65535;
constexpr int64_t kMaxEntries = 1024;
constexpr int64_t kMaxWidth = 512;
constexpr int64_t kMost = (int64_t(1) << 31) - 2;

ts_dtype dtype_of(const at::Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return TS_FLOAT32;
    case at::kHalf: return TS_FLOAT16;
    case at::kBFloat16: return TS_BFLOAT16;
    default: break;
  }
  TORCH_CHECK(false, op, ": unsupported dtype ", t.scalar_type(), " of ", name,
              " (float32, float16 and bfloat16 are supported)");
}

void check_device(const at::Tensor& first, const at::Tensor& t, const char* op,
                  const char* name) {
  TORCH_CHECK(t.device() == first.device(), op, ": ", name, " must be on ", first.device(),
              ", got ", t.device());
}

void check_like(const at::Tensor& first, const at::Tensor& t, const char* op, const char* name) {
  check_device(first, t, op, name);
  TORCH_CHECK(t.scalar_type() == first.scalar_type(), op, ": ", name, " must have dtype ",
              first.scalar_type(), ", got ", t.scalar_type());
}

void check_replicas(int64_t N, const char* op) {
  TORCH_CHECK(N <= kMaxReplicas, op, ": at most ", kMaxReplicas, " replicas; got ", N);
}

void check_size(int64_t size, const char* op, const char* name) {
  TORCH_CHECK(size <= kMost, op, ": ", name, " must be at most 2^31 - 2, got ", size);
}

// Rows that are contiguous inside.
at::Tensor with_unit_rows(const at::Tensor& t) {
  return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t;
}

// A tensor that the replicas may share, of `rank` dimensions with the replica
// one: `t` with that dimension, of size N.
at::Tensor per_replica(const at::Tensor& t, int64_t rank, int64_t N, const char* op,
                       const char* name) {
  TORCH_CHECK(t.dim() == rank || t.dim() == rank - 1, op, ": ", name, " must have ", rank - 1,
              " dimensions, or ", rank, " with the replicas'; got ", t.sizes());
  at::Tensor out = t.dim() == rank ? t : t.unsqueeze(0);
  if (out.size(0) != N && out.size(0) == 1) {
    c10::SmallVector<int64_t, 4> shape(out.sizes().begin(), out.sizes().end());
    shape[0] = N;
    out = out.expand(shape);
  }
  TORCH_CHECK(out.size(0) == N, op, ": ", name, " must have ", N, " replicas, got ", t.sizes());
  return out;
}

void check_indices(const at::Tensor& first, const at::Tensor& t, const char* op,
                   const char* name) {
  check_device(first, t, op, name);
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, op, ": ", name,
              " must be int64 or int32, got ", t.scalar_type());
}

// Replicas that share a tensor have stride 0 along them.
int64_t replica_stride(const at::Tensor& t) { return t.size(0) == 1 ? 0 : t.stride(0); }

ts_index index_of(const at::Tensor& t) {
  return ts_index{t.data_ptr(), replica_stride(t), t.stride(1),
                  t.scalar_type() == at::kLong ? 64 : 32};
}

ts_rows rows_of(const at::Tensor& t) {
  return ts_rows{t.data_ptr(), t.stride(0), t.stride(1)};
}

// An (N,) vector of float32: a replica's hyperparameter.
at::Tensor vector_of(const at::Tensor& first, const at::Tensor& t, int64_t N, const char* op,
                     const char* name) {
  check_device(first, t, op, name);
  TORCH_CHECK(t.numel() == N, op, ": ", name, " must have N = ", N,
              " elements (one per replica), got ", t.numel());
  if (t.dim() == 1 && t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
  return t.reshape({N}).to(at::kFloat).contiguous();
}

void check_status(int status, const char* op) {
  TORCH_CHECK(status == 0, op, ": HIP launch failed with error ", status);
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

c10::DataPtr workspace_for(const at::Tensor& t, size_t bytes) {
  return bytes == 0 ? c10::DataPtr{} : c10::GetAllocator(t.device().type())->allocate(bytes);
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------
at::Tensor embedding(const at::Tensor& weight, const at::Tensor& tokens, double scale) {
  constexpr const char* op = "churten::embedding";
  TORCH_CHECK(weight.dim() == 2 || weight.dim() == 3, op,
              ": weight must be (V, D), or (N, V, D) with the replicas'; got ", weight.sizes());
  const bool single = weight.dim() == 2;
  const ts_dtype dtype = dtype_of(weight, op, "weight");
  const at::Tensor w = with_unit_rows(single ? weight.unsqueeze(0) : weight);
  const int64_t N = w.size(0), V = w.size(1), D = w.size(2);
  check_replicas(N, op);
  check_indices(weight, tokens, op, "tokens");
  TORCH_CHECK(!single || tokens.dim() == 1, op,
              ": tokens must be (B,) beside a weight without replicas, got ", tokens.sizes());
  const at::Tensor ids = per_replica(tokens, 2, N, op, "tokens");
  const int64_t B = ids.size(1);
  check_size(V, op, "the number of embeddings");
  check_size(B, op, "the number of tokens");
  check_size(D, op, "the width");
  const c10::DeviceGuard guard(weight.device());
  at::Tensor out = at::empty({N, B, D}, weight.options());
  if (weight.is_cuda()) {
    check_status(ts_embedding(rows_of(w), index_of(ids), rows_of(out), dtype, N, B, V, D,
                              static_cast<float>(scale), stream_of(weight)),
                 op);
  } else {
    lm_cpu::embedding(rows_of(w), index_of(ids), rows_of(out), dtype, N, B, V, D,
                      static_cast<float>(scale));
  }
  return single ? out.squeeze(0) : out;
}

// `out` is (N, V, D) with unit rows, `grad` (N, B, D).
void embedding_grad_into(const at::Tensor& out, const at::Tensor& grad, const at::Tensor& tokens,
                         double scale, bool accumulate, const char* op) {
  const int64_t N = out.size(0), V = out.size(1), D = out.size(2);
  check_replicas(N, op);
  check_indices(out, tokens, op, "tokens");
  const at::Tensor ids = per_replica(tokens, 2, N, op, "tokens");
  const int64_t B = ids.size(1);
  TORCH_CHECK(grad.size(0) == N && grad.size(1) == B && grad.size(2) == D, op,
              ": grad must be the lookup's shape ", at::IntArrayRef({N, B, D}), ", got ",
              grad.sizes());
  const ts_dtype dtype = dtype_of(out, op, "weight_grad");
  check_like(out, grad, op, "grad");
  check_size(V, op, "the number of embeddings");
  check_size(B, op, "the number of tokens");
  check_size(D, op, "the width");
  const at::Tensor g = with_unit_rows(grad);
  const c10::DeviceGuard guard(out.device());
  if (out.is_cuda()) {
    const ts_index index = index_of(ids);
    const size_t bytes =
        ts_embedding_grad_workspace(dtype, N, B, V, D, index.stride_n == 0 ? 1 : 0);
    const c10::DataPtr ws = workspace_for(out, bytes);
    check_status(ts_embedding_grad(rows_of(out), rows_of(g), index, dtype, N, B, V, D,
                                   static_cast<float>(scale), accumulate ? TS_ACCUMULATE : 0u,
                                   ws.get(), bytes, stream_of(out)),
                 op);
  } else {
    lm_cpu::embedding_grad(rows_of(out), rows_of(g), index_of(ids), dtype, N, B, V, D,
                           static_cast<float>(scale), accumulate);
  }
}

at::Tensor embedding_grad(const at::Tensor& grad, const at::Tensor& tokens,
                          int64_t num_embeddings, double scale) {
  constexpr const char* op = "churten::embedding_grad";
  TORCH_CHECK(grad.dim() == 2 || grad.dim() == 3, op,
              ": grad must be (B, D), or (N, B, D) with the replicas'; got ", grad.sizes());
  TORCH_CHECK(num_embeddings >= 0, op, ": num_embeddings must not be negative, got ",
              num_embeddings);
  const bool single = grad.dim() == 2;
  TORCH_CHECK(!single || tokens.dim() == 1, op,
              ": tokens must be (B,) beside a grad without replicas, got ", tokens.sizes());
  const at::Tensor g = single ? grad.unsqueeze(0) : grad;
  dtype_of(grad, op, "grad");
  at::Tensor out = at::empty({g.size(0), num_embeddings, g.size(2)}, grad.options());
  embedding_grad_into(out, g, tokens, scale, false, op);
  return single ? out.squeeze(0) : out;
}

void embedding_grad_(at::Tensor weight_grad, const at::Tensor& grad, const at::Tensor& tokens,
                     double scale, bool accumulate) {
  constexpr const char* op = "churten::embedding_grad_";
  const bool single = weight_grad.dim() == 2;
  TORCH_CHECK((single || weight_grad.dim() == 3) && grad.dim() == weight_grad.dim(), op,
              ": weight_grad and grad must be (V, D) and (B, D), or (N, V, D) and (N, B, D); got ",
              weight_grad.sizes(), " and ", grad.sizes());
  TORCH_CHECK(!single || tokens.dim() == 1, op,
              ": tokens must be (B,) beside a grad without replicas, got ", tokens.sizes());
  TORCH_CHECK(weight_grad.size(-1) <= 1 || weight_grad.stride(-1) == 1, op,
              ": weight_grad's rows must be contiguous");
  TORCH_CHECK(at::has_internal_overlap(weight_grad) != at::MemOverlap::Yes, op,
              ": weight_grad's elements must not share memory");
  embedding_grad_into(single ? weight_grad.unsqueeze(0) : weight_grad,
                      single ? grad.unsqueeze(0) : grad, tokens, scale, accumulate, op);
}

// ---------------------------------------------------------------------------
// Norm and rotation of queries and keys
// ---------------------------------------------------------------------------
ts_heads heads_of(const at::Tensor& t) {
  return ts_heads{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

struct Heads {
  bool single;
  at::Tensor q, k, qw, kw, cos, sin, positions;
  ts_qk_shape shape;
  ts_dtype dtype;
};

Heads heads_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                 const at::Tensor& k_weight, const at::Tensor& cos, const at::Tensor& sin,
                 const at::Tensor& positions, double eps, bool interleaved, const char* op) {
  Heads h;
  TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim(), op,
              ": q and k must be (M, H, D), or (N, M, H, D) with the replicas'; got ", q.sizes(),
              " and ", k.sizes());
  h.single = q.dim() == 3;
  h.dtype = dtype_of(q, op, "q");
  check_like(q, k, op, "k");
  h.q = with_unit_rows(h.single ? q.unsqueeze(0) : q);
  h.k = with_unit_rows(h.single ? k.unsqueeze(0) : k);
  const int64_t N = h.q.size(0), M = h.q.size(1), D = h.q.size(3);
  check_replicas(N, op);
  check_size(M, op, "the number of tokens");
  TORCH_CHECK(h.k.size(0) == N && h.k.size(1) == M && h.k.size(3) == D, op,
              ": q and k must agree but in the number of heads; got ", q.sizes(), " and ",
              k.sizes());
  TORCH_CHECK(D >= 1 && D <= kMaxWidth, op, ": heads must be 1 to ", kMaxWidth, " wide, got ", D);
  for (const at::Tensor* t : {&h.q, &h.k}) {
    TORCH_CHECK(t->size(2) >= 1 && t->size(2) <= 65535, op, ": 1 to 65535 heads, got ",
                t->size(2));
  }
  const auto weight = [&](const at::Tensor& w, const char* name) {
    check_like(q, w, op, name);
    TORCH_CHECK(w.dim() == (h.single ? 1 : 2) && w.size(-1) == D && (h.single || w.size(0) == N),
                op, ": ", name, " must be ", h.single ? "(D,)" : "(N, D)", " = ",
                h.single ? at::IntArrayRef({D}) : at::IntArrayRef({N, D}), ", got ", w.sizes());
    return with_unit_rows(h.single ? w.unsqueeze(0) : w);
  };
  h.qw = weight(q_weight, "q_weight");
  h.kw = weight(k_weight, "k_weight");
  const auto table = [&](const at::Tensor& t, const char* name) {
    check_device(q, t, op, name);
    TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kFloat, op, ": ", name,
                " must be a float32 (positions, rotated pairs) table, got ", t.scalar_type(), " ",
                t.sizes());
    return with_unit_rows(t);
  };
  h.cos = table(cos, "cos");
  h.sin = table(sin, "sin");
  TORCH_CHECK(cos.sizes() == sin.sizes(), op, ": cos and sin must have one shape, got ",
              cos.sizes(), " and ", sin.sizes());
  TORCH_CHECK(2 * cos.size(1) <= D, op, ": ", cos.size(1), " rotated pairs need heads at least ",
              2 * cos.size(1), " wide, got ", D);
  if (h.cos.stride(0) != h.sin.stride(0)) {
    h.cos = h.cos.contiguous();
    h.sin = h.sin.contiguous();
  }
  check_indices(q, positions, op, "positions");
  TORCH_CHECK(!h.single || positions.dim() == 1, op,
              ": positions must be (M,) beside heads without replicas, got ", positions.sizes());
  h.positions = per_replica(positions, 2, N, op, "positions");
  TORCH_CHECK(h.positions.size(1) == M, op, ": positions must have M = ", M, " tokens, got ",
              positions.sizes());
  h.shape = ts_qk_shape{N,
                        M,
                        h.q.size(2),
                        h.k.size(2),
                        D,
                        2 * cos.size(1),
                        cos.size(0),
                        static_cast<const float*>(h.cos.data_ptr()),
                        static_cast<const float*>(h.sin.data_ptr()),
                        h.cos.stride(0),
                        index_of(h.positions),
                        static_cast<float>(eps),
                        interleaved ? TS_INTERLEAVED : 0u};
  return h;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
    const at::Tensor& k_weight, const at::Tensor& cos, const at::Tensor& sin,
    const at::Tensor& positions, double eps, bool interleaved) {
  constexpr const char* op = "churten::qk_norm_rope";
  const c10::DeviceGuard guard(q.device());
  const Heads h = heads_args(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, op);
  at::Tensor q_out = at::empty(h.q.sizes(), q.options());
  at::Tensor k_out = at::empty(h.k.sizes(), q.options());
  if (q.is_cuda()) {
    check_status(ts_qk_norm_rope(&h.shape, h.dtype, heads_of(h.q), heads_of(h.k),
                                 h.qw.data_ptr(), h.qw.stride(0), h.kw.data_ptr(),
                                 h.kw.stride(0), heads_of(q_out), heads_of(k_out),
                                 stream_of(q)),
                 op);
  } else {
    lm_cpu::qk_norm_rope(h.shape, h.dtype, heads_of(h.q), heads_of(h.k), h.qw.data_ptr(),
                         h.qw.stride(0), h.kw.data_ptr(), h.kw.stride(0), heads_of(q_out),
                         heads_of(k_out));
  }
  if (h.single) return {q_out.squeeze(0), k_out.squeeze(0)};
  return {q_out, k_out};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_grad(
    const at::Tensor& grad_q, const at::Tensor& grad_k, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& q_weight, const at::Tensor& k_weight, const at::Tensor& cos,
    const at::Tensor& sin, const at::Tensor& positions, double eps, bool interleaved) {
  constexpr const char* op = "churten::qk_norm_rope_grad";
  const c10::DeviceGuard guard(q.device());
  const Heads h = heads_args(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, op);
  const auto grad = [&](const at::Tensor& g, const at::Tensor& of, const char* name) {
    check_like(q, g, op, name);
    TORCH_CHECK(g.sizes() == of.sizes(), op, ": ", name, " must have the shape ", of.sizes(),
                ", got ", g.sizes());
    return with_unit_rows(h.single ? g.unsqueeze(0) : g);
  };
  const at::Tensor dq = grad(grad_q, q, "grad_q"), dk = grad(grad_k, k, "grad_k");
  at::Tensor q_grad = at::empty(h.q.sizes(), q.options());
  at::Tensor k_grad = at::empty(h.k.sizes(), q.options());
  at::Tensor qw_grad = at::empty(h.qw.sizes(), q.options());
  at::Tensor kw_grad = at::empty(h.kw.sizes(), q.options());
  if (q.is_cuda()) {
    const size_t bytes = ts_qk_norm_rope_grad_workspace(&h.shape, h.dtype);
    const c10::DataPtr ws = workspace_for(q, bytes);
    check_status(ts_qk_norm_rope_grad(&h.shape, h.dtype, heads_of(dq), heads_of(dk),
                                      heads_of(h.q), heads_of(h.k), h.qw.data_ptr(),
                                      h.qw.stride(0), h.kw.data_ptr(), h.kw.stride(0),
                                      heads_of(q_grad), heads_of(k_grad), qw_grad.data_ptr(),
                                      kw_grad.data_ptr(), ws.get(), bytes, stream_of(q)),
                 op);
  } else {
    lm_cpu::qk_norm_rope_grad(h.shape, h.dtype, heads_of(dq), heads_of(dk), heads_of(h.q),
                              heads_of(h.k), h.qw.data_ptr(), h.qw.stride(0), h.kw.data_ptr(),
                              h.kw.stride(0), heads_of(q_grad), heads_of(k_grad),
                              qw_grad.data_ptr(), kw_grad.data_ptr());
  }
  if (h.single) {
    return {q_grad.squeeze(0), k_grad.squeeze(0), qw_grad.squeeze(0), kw_grad.squeeze(0)};
  }
  return {q_grad, k_grad, qw_grad, kw_grad};
}

// ---------------------------------------------------------------------------
// Distillation
// ---------------------------------------------------------------------------
std::tuple<at::Tensor, at::Tensor> distill(
    const at::Tensor& logits, const at::Tensor& teacher_logits, const at::Tensor& teacher_index,
    const at::Tensor& temperature, const std::optional<at::Tensor>& weight,
    const std::optional<at::Tensor>& labels, const std::optional<at::Tensor>& hard,
    bool with_grad, const char* op) {
  TORCH_CHECK(logits.dim() == 2 || logits.dim() == 3, op,
              ": logits must be (B, V), or (N, B, V) with the replicas'; got ", logits.sizes());
  const bool single = logits.dim() == 2;
  const ts_dtype dtype = dtype_of(logits, op, "logits");
  const c10::DeviceGuard guard(logits.device());
  const at::Tensor x = with_unit_rows(single ? logits.unsqueeze(0) : logits);
  const int64_t N = x.size(0), B = x.size(1), V = x.size(2);
  check_replicas(N, op);
  check_size(B, op, "the number of tokens");
  check_size(V, op, "the vocabulary");
  const auto shared = [&](const at::Tensor& t, int64_t rank, const char* name) {
    TORCH_CHECK(!single || t.dim() == rank - 1, op, ": ", name, " must have ", rank - 1,
                " dimensions beside logits without replicas, got ", t.sizes());
    const at::Tensor out = per_replica(t, rank, N, op, name);
    TORCH_CHECK(out.size(1) == B, op, ": ", name, " must have B = ", B, " rows, got ",
                t.sizes());
    return out;
  };
  check_device(logits, teacher_logits, op, "teacher_logits");
  TORCH_CHECK(teacher_logits.is_floating_point(), op,
              ": teacher_logits must be floating point, got ", teacher_logits.scalar_type());
  check_indices(logits, teacher_index, op, "teacher_index");
  // float32 before the replicas' dimension: a shared teacher is converted once.
  const at::Tensor z =
      shared(with_unit_rows(teacher_logits.to(at::kFloat)), 3, "teacher_logits");
  const at::Tensor index = shared(with_unit_rows(teacher_index), 3, "teacher_index");
  const int64_t K = z.size(2);
  TORCH_CHECK(index.size(2) == K, op,
              ": teacher_logits and teacher_index must have one shape, got ", teacher_logits.sizes(), " and ", teacher_index.sizes());
  TORCH_CHECK(K <= kMaxEntries, op, ": at most ", kMaxEntries, " teacher entries per row, got ",
              K);
  const at::Tensor t = vector_of(logits, temperature, N, op, "temperature");
  TORCH_CHECK(labels.has_value() == hard.has_value(), op,
              ": labels and hard go together; got only ", labels.has_value() ? "labels" : "hard");
  at::Tensor row_weight, label, share;
  if (weight.has_value()) {
    check_device(logits, *weight, op, "weight");
    TORCH_CHECK(weight->is_floating_point(), op, ": weight must be floating point, got ",
                weight->scalar_type());
    row_weight = shared(weight->to(at::kFloat), 2, "weight");
  }
  if (labels.has_value()) {
    check_indices(logits, *labels, op, "labels");
    label = shared(*labels, 2, "labels");
    share = vector_of(logits, *hard, N, op, "hard");
  }
  at::Tensor loss = at::empty({N, B}, logits.options().dtype(at::kFloat));
  at::Tensor grad;
  if (with_grad) grad = at::empty({N, B, V}, logits.options());

  ts_distill_args a{};
  a.N = N;
  a.B = B;
  a.V = V;
  a.K = K;
  a.logits = rows_of(x);
  a.teacher = rows_of(z);
  a.index = index_of(index);
  a.temperature = static_cast<const float*>(t.data_ptr());
  if (label.defined()) {
    a.labels = index_of(label);
    a.hard = static_cast<const float*>(share.data_ptr());
  }
  if (row_weight.defined()) {
    a.weight = static_cast<const float*>(row_weight.data_ptr());
    a.weight_stride_n = row_weight.stride(0);
    a.weight_stride_b = row_weight.stride(1);
  }
  a.loss = static_cast<float*>(loss.data_ptr());
  if (with_grad) a.grad = rows_of(grad);
  if (N > 0 && B > 0) {
    if (logits.is_cuda()) {
      const size_t bytes = ts_distill_workspace(&a, dtype);
      const c10::DataPtr ws = workspace_for(logits, bytes);
      check_status(ts_distill(&a, dtype, ws.get(), bytes, stream_of(logits)), op);
    } else {
      lm_cpu::distill(a, dtype);
    }
  }
  if (!single) return {loss, grad};
  return {loss.squeeze(0), with_grad ? grad.squeeze(0) : grad};
}

at::Tensor distill_loss(const at::Tensor& logits, const at::Tensor& teacher_logits,
                        const at::Tensor& teacher_index, const at::Tensor& temperature,
                        const std::optional<at::Tensor>& weight,
                        const std::optional<at::Tensor>& labels,
                        const std::optional<at::Tensor>& hard) {
  return std::get<0>(distill(logits, teacher_logits, teacher_index, temperature, weight, labels,
                             hard, false, "churten::distill_loss"));
}

std::tuple<at::Tensor, at::Tensor> distill_loss_grad(
    const at::Tensor& logits, const at::Tensor& teacher_logits, const at::Tensor& teacher_index,
    const at::Tensor& temperature, const std::optional<at::Tensor>& weight,
    const std::optional<at::Tensor>& labels, const std::optional<at::Tensor>& hard) {
  return distill(logits, teacher_logits, teacher_index, temperature, weight, labels, hard, true,
                 "churten::distill_loss_grad");
}

template <typename Library>
void implement(Library& m) {
  m.impl("embedding", &embedding);
  m.impl("embedding_grad", &embedding_grad);
  m.impl("embedding_grad_", &embedding_grad_);
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_grad", &qk_norm_rope_grad);
  m.impl("distill_loss", &distill_loss);
  m.impl("distill_loss_grad", &distill_loss_grad);
}

// ---------------------------------------------------------------------------
// Derivatives
// ---------------------------------------------------------------------------
// Asking for a derivative that is not there, in reverse or in forward mode,
// raises (torch's default for an operator of a library is a warning, zeros, and
// a tangent that is dropped). The heads and the distillation have none at this
// level: those of the forward operators are formed a level above, in Python.
// torch's own kernel for that goes through every argument in its boxed form, 0.2
// us of a lookup's 2.2 us on the host; this one 0.05.
bool needs_derivative(const at::Tensor& t) { return t.requires_grad(); }
bool needs_derivative(const std::optional<at::Tensor>& t) {
  return t.has_value() && t->requires_grad();
}
bool has_tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const std::optional<at::Tensor>& t) { return t.has_value() && has_tangent(*t); }
bool needs_derivative(double) { return false; }
bool has_tangent(double) { return false; }

void set_history(const std::shared_ptr<torch::autograd::Node>& node, const at::Tensor& out) {
  torch::autograd::set_history(out, node);
}
template <typename... T>
void set_history(const std::shared_ptr<torch::autograd::Node>& node,
                 const std::tuple<T...>& outs) {
  std::apply([&](const T&... out) { (torch::autograd::set_history(out, node), ...); }, outs);
}

template <typename Function>
struct Underived;
template <typename R, typename... A>
struct Underived<R(A...)> {
  template <const char* NAME>
  static R call(c10::DispatchKeySet keys, A... args) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow(NAME, "")
                               .template typed<R(A...)>();
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(args) || ...), NAME,
                                " has no derivative in forward AD mode");
    R out = [&] {
      const at::AutoDispatchBelowADInplaceOrView below;
      return op.redispatch(keys & c10::after_autograd_keyset, args...);
    }();
    if (at::GradMode::is_enabled() && (needs_derivative(args) || ...)) {
      // Its edges only make the outputs ask for gradients: it raises when run.
      set_history(std::shared_ptr<torch::autograd::Node>(
                      new torch::autograd::NotImplemented(NAME, edges(args...)),
                      torch::autograd::deleteNode),
                  out);
    }
    return out;
  }

 private:
  static torch::autograd::edge_list edges(const A&... args) {
    torch::autograd::edge_list list;
    (add(list, args), ...);
    return list;
  }
  static void add(torch::autograd::edge_list& list, const at::Tensor& t) {
    list.push_back(torch::autograd::impl::gradient_edge(t));
  }
  static void add(torch::autograd::edge_list& list, const std::optional<at::Tensor>& t) {
    if (t.has_value()) add(list, *t);
  }
  static void add(torch::autograd::edge_list&, double) {}
};

template <typename Function>
auto operator_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Function>();
}
const auto& embedding_op() {
  static const auto op = operator_of<decltype(embedding)>("churten::embedding");
  return op;
}
const auto& embedding_grad_op() {
  static const auto op = operator_of<decltype(embedding_grad)>("churten::embedding_grad");
  return op;
}
const auto& embedding_grad_into_op() {
  static const auto op = operator_of<decltype(embedding_grad_)>("churten::embedding_grad_");
  return op;
}

void refuse_tangent(const char* op, const at::Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), op, " has no derivative in forward AD mode");
}

// The lookup is linear in the table and its gradient in the incoming one; each is
// the other's derivative, so both have derivatives of every order.
struct LookupDerivative : torch::autograd::Node {
  torch::autograd::SavedVariable tokens;
  int64_t num_embeddings = 0;
  double scale = 1;
  bool of_gradient = false;

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    const at::Tensor& grad = grads[0];
    if (!grad.defined()) return {at::Tensor()};
    const at::Tensor ids = tokens.unpack();
    return {of_gradient ? embedding_op().call(grad, ids, scale)
                        : embedding_grad_op().call(grad, ids, num_embeddings, scale)};
  }
  void release_variables() override { tokens.reset_data(); }
};

// `out` with the derivative in `in`, if that asks for one.
at::Tensor derived(const at::Tensor& in, const at::Tensor& tokens, at::Tensor out,
                   int64_t num_embeddings, double scale, bool of_gradient) {
  if (!at::GradMode::is_enabled() || !in.requires_grad()) return out;
  const std::shared_ptr<LookupDerivative> node(new LookupDerivative,
                                               torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(in));
  node->tokens = torch::autograd::SavedVariable(tokens, /*is_output=*/false);
  node->num_embeddings = num_embeddings;
  node->scale = scale;
  node->of_gradient = of_gradient;
  torch::autograd::set_history(out, node);
  return out;
}

at::Tensor embedding_derived(c10::DispatchKeySet keys, const at::Tensor& weight,
                             const at::Tensor& tokens, double scale) {
  refuse_tangent("churten::embedding", weight);
  at::Tensor out = [&] {
    const at::AutoDispatchBelowADInplaceOrView below;
    return embedding_op().redispatch(keys & c10::after_autograd_keyset, weight, tokens, scale);
  }();
  // Traced with sizes as symbols, the table's is made a number.
  const int64_t V = weight.sym_size(-2).guard_int(__FILE__, __LINE__);
  return derived(weight, tokens, std::move(out), V, scale, false);
}

at::Tensor embedding_grad_derived(c10::DispatchKeySet keys, const at::Tensor& grad,
                                  const at::Tensor& tokens, int64_t num_embeddings,
                                  double scale) {
  refuse_tangent("churten::embedding_grad", grad);
  at::Tensor out = [&] {
    const at::AutoDispatchBelowADInplaceOrView below;
    return embedding_grad_op().redispatch(keys & c10::after_autograd_keyset, grad, tokens,
                                          num_embeddings, scale);
  }();
  return derived(grad, tokens, std::move(out), num_embeddings, scale, true);
}

// In place, as torch's own: a target that gradients would go through is refused or
// remembers that they cannot, and its version counter rises.
void embedding_grad_underived(c10::DispatchKeySet keys, at::Tensor weight_grad,
                              const at::Tensor& grad, const at::Tensor& tokens, double scale,
                              bool accumulate) {
  constexpr const char* op = "churten::embedding_grad_";
  refuse_tangent(op, weight_grad);
  refuse_tangent(op, grad);
  const bool any = at::GradMode::is_enabled() &&
                   (needs_derivative(weight_grad) || needs_derivative(grad));
  torch::autograd::check_inplace(weight_grad, any);
  std::shared_ptr<torch::autograd::Node> node;
  if (any) {
    node = std::shared_ptr<torch::autograd::Node>(
        new torch::autograd::NotImplemented(
            op, torch::autograd::collect_next_edges(weight_grad, grad)),
        torch::autograd::deleteNode);
  }
  {
    const at::AutoDispatchBelowAutograd below;
    embedding_grad_into_op().redispatch(keys & c10::after_autograd_keyset, weight_grad, grad,
                                        tokens, scale, accumulate);
  }
  if (any) torch::autograd::rebase_history(weight_grad, node);
}

void embedding_grad_written(c10::DispatchKeySet keys, at::Tensor weight_grad,
                            const at::Tensor& grad, const at::Tensor& tokens, double scale,
                            bool accumulate) {
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    embedding_grad_into_op().redispatch(keys & c10::after_ADInplaceOrView_keyset, weight_grad,
                                        grad, tokens, scale, accumulate);
  }
  // One made in inference mode has no counter.
  if (!weight_grad.is_inference()) torch::autograd::increment_version(weight_grad);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(churten, m) {
  m.def("embedding(Tensor weight, Tensor tokens, float scale=1.0) -> Tensor");
  m.def("embedding_grad(Tensor grad, Tensor tokens, int num_embeddings, float scale=1.0) -> "
        "Tensor");
  m.def("embedding_grad_(Tensor(a!) weight_grad, Tensor grad, Tensor tokens, float scale=1.0, "
        "bool accumulate=False) -> ()");
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, "
        "Tensor sin, Tensor positions, float eps=1e-06, bool interleaved=False) -> "
        "(Tensor, Tensor)");
  m.def("qk_norm_rope_grad(Tensor grad_q, Tensor grad_k, Tensor q, Tensor k, Tensor q_weight, "
        "Tensor k_weight, Tensor cos, Tensor sin, Tensor positions, float eps=1e-06, "
        "bool interleaved=False) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("distill_loss(Tensor logits, Tensor teacher_logits, Tensor teacher_index, "
        "Tensor temperature, Tensor? weight=None, Tensor? labels=None, Tensor? hard=None) -> "
        "Tensor");
  m.def("distill_loss_grad(Tensor logits, Tensor teacher_logits, Tensor teacher_index, "
        "Tensor temperature, Tensor? weight=None, Tensor? labels=None, Tensor? hard=None) -> "
        "(Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(churten, CUDA, m) { implement(m); }
TORCH_LIBRARY_IMPL(churten, CPU, m) { implement(m); }

namespace {
constexpr char kQkNormRope[] = "churten::qk_norm_rope";
constexpr char kQkNormRopeGrad[] = "churten::qk_norm_rope_grad";
constexpr char kDistillLoss[] = "churten::distill_loss";
constexpr char kDistillLossGrad[] = "churten::distill_loss_grad";
}  // namespace

TORCH_LIBRARY_IMPL(churten, Autograd, m) {
  m.impl("embedding", &embedding_derived);
  m.impl("embedding_grad", &embedding_grad_derived);
  m.impl("embedding_grad_", &embedding_grad_underived);
  m.impl("qk_norm_rope", &Underived<decltype(qk_norm_rope)>::call<kQkNormRope>);
  m.impl("qk_norm_rope_grad", &Underived<decltype(qk_norm_rope_grad)>::call<kQkNormRopeGrad>);
  m.impl("distill_loss", &Underived<decltype(distill_loss)>::call<kDistillLoss>);
  m.impl("distill_loss_grad", &Underived<decltype(distill_loss_grad)>::call<kDistillLossGrad>);
}

TORCH_LIBRARY_IMPL(churten, ADInplaceOrView, m) {
  m.impl("embedding_grad_", &embedding_grad_written);
}

}  // namespace churten
