// lm_cpu.cpp -- the language-model operators on CPU tensors: the formulas as
// loops over rows in float32, rounded once, on torch's intra-op threads. For
// development and tests on hosts without a GPU; GPU tensors never come here.

#include "lm_cpu.h"

#include <ATen/Parallel.h>
#include <c10/util/BFloat16.h>
#include <c10/util/Exception.h>
#include <c10/util/Half.h>

#include <cmath>
#include <limits>
#include <vector>

namespace churten {
namespace lm_cpu {
namespace {

template <typename U>
struct type_tag {
  using type = U;
};

template <typename F>
void by_dtype(ts_dtype dtype, F&& f) {
  switch (dtype) {
    case TS_FLOAT32: return f(type_tag<float>{});
    case TS_FLOAT16: return f(type_tag<c10::Half>{});
    case TS_BFLOAT16: return f(type_tag<c10::BFloat16>{});
    default: TORCH_INTERNAL_ASSERT(false, "dtype");
  }
}

int64_t index_at(const ts_index& t, int64_t n, int64_t b, int64_t k = 0) {
  const int64_t at = n * t.stride_n + b * t.stride_b + k;
  return t.bits == 64 ? static_cast<const int64_t*>(t.data)[at]
                      : static_cast<const int32_t*>(t.data)[at];
}

// Rows of about this many elements make one task.
int64_t grain(int64_t elements) {
  return std::max<int64_t>(1, 16384 / std::max<int64_t>(1, elements));
}

template <typename T>
T* row_of(const ts_rows& t, int64_t n, int64_t b) {
  return static_cast<T*>(t.data) + n * t.stride_n + b * t.stride_b;
}

}  // namespace

void embedding(ts_rows weight, ts_index tokens, ts_rows out, ts_dtype dtype, int64_t N,
               int64_t B, int64_t V, int64_t D, float scale) {
  by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    at::parallel_for(0, N * B, grain(D), [&](int64_t begin, int64_t end) {
      for (int64_t i = begin; i < end; ++i) {
        const int64_t n = i / B, b = i % B, token = index_at(tokens, n, b);
        T* to = row_of<T>(out, n, b);
        const bool known = token >= 0 && token < V;
        const T* from = known ? row_of<T>(weight, n, token) : nullptr;
        for (int64_t d = 0; d < D; ++d) {
          to[d] = known ? static_cast<T>(static_cast<float>(from[d]) * scale) : T(0.0f);
        }
      }
    });
  });
}

void embedding_grad(ts_rows weight_grad, ts_rows grad, ts_index tokens, ts_dtype dtype,
                    int64_t N, int64_t B, int64_t V, int64_t D, float scale, bool accumulate) {
  by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    std::vector<float> sum;
    for (int64_t n = 0; n < N; ++n) {
      // The positions of each token, in order: lists through `next`.
      std::vector<int64_t> first(V, -1), last(V, -1), next(B, -1);
      for (int64_t b = 0; b < B; ++b) {
        const int64_t token = index_at(tokens, n, b);
        if (token < 0 || token >= V) continue;
        (last[token] < 0 ? first[token] : next[last[token]]) = b;
        last[token] = b;
      }
      at::parallel_for(0, V, grain(D), [&](int64_t begin, int64_t end) {
        std::vector<float> total(D);
        for (int64_t v = begin; v < end; ++v) {
          if (accumulate && first[v] < 0) continue;
          std::fill(total.begin(), total.end(), 0.0f);
          for (int64_t b = first[v]; b >= 0; b = next[b]) {
            const T* from = row_of<T>(grad, n, b);
            for (int64_t d = 0; d < D; ++d) total[d] += static_cast<float>(from[d]);
          }
          T* to = row_of<T>(weight_grad, n, v);
          for (int64_t d = 0; d < D; ++d) {
            const float value = total[d] * scale;
            to[d] = static_cast<T>(accumulate ? value + static_cast<float>(to[d]) : value);
          }
        }
      });
    }
  });
}

namespace {

// The members of pair j of a head's rotated elements.
struct Pair {
  int64_t a, b;
};
Pair pair_of(const ts_qk_shape& s, int64_t j) {
  return (s.flags & TS_INTERLEAVED) != 0 ? Pair{2 * j, 2 * j + 1} : Pair{j, j + s.rot / 2};
}

// Turns y by the angles of token m, or back for sign -1.
void rotate(const ts_qk_shape& s, int64_t n, int64_t m, float sign, float* y) {
  if (s.rot == 0) return;
  const int64_t position = index_at(s.positions, n, m);
  if (position < 0 || position >= s.P) return;
  const float* cos = s.cos + position * s.table_stride;
  const float* sin = s.sin + position * s.table_stride;
  for (int64_t j = 0; j < s.rot / 2; ++j) {
    const Pair p = pair_of(s, j);
    const float a = y[p.a], b = y[p.b], w = sign * sin[j];
    y[p.a] = a * cos[j] - b * w;
    y[p.b] = b * cos[j] + a * w;
  }
}

template <typename T>
T* head_of(const ts_heads& t, int64_t n, int64_t m, int64_t h) {
  return static_cast<T*>(t.data) + n * t.stride_n + m * t.stride_m + h * t.stride_h;
}

template <typename T>
float reciprocal_norm(const T* x, const ts_qk_shape& s) {
  float square = 0;
  for (int64_t d = 0; d < s.D; ++d) square += static_cast<float>(x[d]) * static_cast<float>(x[d]);
  return 1.0f / std::sqrt(square / static_cast<float>(s.D) + s.eps);
}

template <typename T>
void qk_side(const ts_qk_shape& s, int64_t heads, const ts_heads& in, const T* weight,
             int64_t weight_stride, const ts_heads& out) {
  at::parallel_for(0, s.N * s.M, grain(heads * s.D), [&](int64_t begin, int64_t end) {
    std::vector<float> y(s.D);
    for (int64_t i = begin; i < end; ++i) {
      const int64_t n = i / s.M, m = i % s.M;
      for (int64_t h = 0; h < heads; ++h) {
        const T* x = head_of<T>(in, n, m, h);
        const T* w = weight + n * weight_stride;
        const float r = reciprocal_norm(x, s);
        for (int64_t d = 0; d < s.D; ++d) {
          y[d] = static_cast<float>(x[d]) * r * static_cast<float>(w[d]);
        }
        rotate(s, n, m, 1, y.data());
        T* to = head_of<T>(out, n, m, h);
        for (int64_t d = 0; d < s.D; ++d) to[d] = static_cast<T>(y[d]);
      }
    }
  });
}

template <typename T>
void qk_grad_side(const ts_qk_shape& s, int64_t heads, const ts_heads& dout, const ts_heads& in,
                  const T* weight, int64_t weight_stride, const ts_heads& out, T* weight_grad) {
  // One task per replica: its weight gradient has one order of additions.
  at::parallel_for(0, s.N, 1, [&](int64_t begin, int64_t end) {
    std::vector<float> u(s.D), dw(s.D);
    for (int64_t n = begin; n < end; ++n) {
      std::fill(dw.begin(), dw.end(), 0.0f);
      const T* w = weight + n * weight_stride;
      for (int64_t m = 0; m < s.M; ++m) {
        for (int64_t h = 0; h < heads; ++h) {
          const T* x = head_of<T>(in, n, m, h);
          const T* dy = head_of<T>(dout, n, m, h);
          const float r = reciprocal_norm(x, s);
          for (int64_t d = 0; d < s.D; ++d) u[d] = static_cast<float>(dy[d]);
          rotate(s, n, m, -1, u.data());
          float along = 0;
          for (int64_t d = 0; d < s.D; ++d) {
            along += u[d] * static_cast<float>(w[d]) * static_cast<float>(x[d]);
            dw[d] += u[d] * (static_cast<float>(x[d]) * r);
          }
          const float c = along / static_cast<float>(s.D) * r * r;
          T* to = head_of<T>(out, n, m, h);
          for (int64_t d = 0; d < s.D; ++d) {
            to[d] = static_cast<T>(
                (u[d] * static_cast<float>(w[d]) - static_cast<float>(x[d]) * c) * r);
          }
        }
      }
      for (int64_t d = 0; d < s.D; ++d) weight_grad[n * s.D + d] = static_cast<T>(dw[d]);
    }
  });
}

}  // namespace

void qk_norm_rope(const ts_qk_shape& shape, ts_dtype dtype, ts_heads q, ts_heads k,
                  const void* q_weight, int64_t qw_stride, const void* k_weight,
                  int64_t kw_stride, ts_heads q_out, ts_heads k_out) {
  by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    qk_side<T>(shape, shape.Hq, q, static_cast<const T*>(q_weight), qw_stride, q_out);
    qk_side<T>(shape, shape.Hk, k, static_cast<const T*>(k_weight), kw_stride, k_out);
  });
}

void qk_norm_rope_grad(const ts_qk_shape& shape, ts_dtype dtype, ts_heads dq, ts_heads dk,
                       ts_heads q, ts_heads k, const void* q_weight, int64_t qw_stride,
                       const void* k_weight, int64_t kw_stride, ts_heads q_grad,
                       ts_heads k_grad, void* qw_grad, void* kw_grad) {
  by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    qk_grad_side<T>(shape, shape.Hq, dq, q, static_cast<const T*>(q_weight), qw_stride, q_grad,
                    static_cast<T*>(qw_grad));
    qk_grad_side<T>(shape, shape.Hk, dk, k, static_cast<const T*>(k_weight), kw_stride, k_grad,
                    static_cast<T*>(kw_grad));
  });
}

namespace {

template <typename T>
void distill_row(const ts_distill_args& a, int64_t n, int64_t b) {
  const T* x = row_of<T>(a.logits, n, b);
  T* grad = a.grad.data == nullptr ? nullptr : row_of<T>(a.grad, n, b);
  const float weight =
      a.weight == nullptr ? 1.0f : a.weight[n * a.weight_stride_n + b * a.weight_stride_b];
  float& loss = a.loss[n * a.B + b];
  loss = 0;
  if (grad != nullptr) std::fill(grad, grad + a.V, T(0.0f));
  if (weight == 0) return;

  constexpr float kNone = -std::numeric_limits<float>::infinity();
  const float t = a.temperature[n];
  const float* z = row_of<float>(a.teacher, n, b);
  const auto entry = [&](int64_t k) -> int64_t {
    const int64_t i = index_at(a.index, n, b, k);
    return i >= 0 && i < a.V && z[k] != kNone ? i : -1;
  };
  float z_top = kNone;
  for (int64_t k = 0; k < a.K; ++k) {
    if (entry(k) >= 0) z_top = std::fmax(z_top, z[k]);
  }
  int64_t label = -1;
  float share = 0;
  if (a.hard != nullptr) {
    share = a.hard[n];
    label = index_at(a.labels, n, b);
    // A part without a share is left out: it may be infinite.
    if (label >= a.V || share == 0) label = -1;
  }
  float m = std::numeric_limits<float>::lowest();
  for (int64_t v = 0; v < a.V; ++v) m = std::fmax(m, static_cast<float>(x[v]));
  // In double: the sums are as long as the vocabulary, and in one order here.
  double s = 0, s1 = 0;
  for (int64_t v = 0; v < a.V; ++v) {
    const float d = static_cast<float>(x[v]) - m;
    s += std::exp(d / t);
    if (label >= 0) s1 += std::exp(d);
  }
  float Z = 0, own = 0, cross = 0;
  for (int64_t k = 0; k < a.K; ++k) {
    const int64_t i = entry(k);
    if (i < 0) continue;
    const float d = z[k] - z_top, e = std::exp(d / t);
    if (e <= 0) continue;
    Z += e;
    own += e * d;
    cross += e * (static_cast<float>(x[i]) - m);
  }
  const bool taught = Z != 0 && share != 1;
  if (taught) {
    const float kl = (own - cross) / (Z * t) - std::log(Z) + static_cast<float>(std::log(s));
    loss += (1 - share) * t * t * kl;
  }
  if (label >= 0) {
    loss += share * (static_cast<float>(std::log(s1)) - (static_cast<float>(x[label]) - m));
  }
  loss *= weight;
  if (grad == nullptr || (!taught && label < 0)) return;

  const float soft = taught ? weight * (1 - share) * t : 0, hard = label >= 0 ? weight * share : 0;
  const float f = soft / static_cast<float>(s);
  const float f1 = label >= 0 ? hard / static_cast<float>(s1) : 0;
  const auto base = [&](int64_t v) {
    const float d = static_cast<float>(x[v]) - m;
    const float g = f * std::exp(d / t);
    return label >= 0 ? g + f1 * std::exp(d) : g;
  };
  for (int64_t v = 0; v < a.V; ++v) grad[v] = static_cast<T>(base(v));
  const auto corrected = [&](int64_t v) {
    float taken = 0;
    for (int64_t k = 0; k < a.K; ++k) {
      if (entry(k) == v) taken += std::exp((z[k] - z_top) / t);
    }
    return static_cast<T>(base(v) - (taught ? taken * (soft / Z) : 0) - (v == label ? hard : 0));
  };
  for (int64_t k = 0; k < a.K; ++k) {
    if (entry(k) >= 0) grad[entry(k)] = corrected(entry(k));
  }
  if (label >= 0) grad[label] = corrected(label);
}

}  // namespace

void distill(const ts_distill_args& args, ts_dtype dtype) {
  by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    at::parallel_for(0, args.N * args.B, grain(args.V), [&](int64_t begin, int64_t end) {
      for (int64_t i = begin; i < end; ++i) distill_row<T>(args, i / args.B, i % args.B);
    });
  });
}

}  // namespace lm_cpu
}  // namespace churten
