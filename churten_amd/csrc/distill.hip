// distill.hip -- distillation from a teacher's top logits: loss and gradient.
//
// For a row of V student logits x, K teacher logits z at the indices i, a
// temperature t and a share h of hard labels:
//   p = softmax(z / t),  q = softmax(x / t),  q1 = softmax(x)
//   loss = weight ((1 - h) t^2 sum_k p_k (log p_k - log q[i_k]) + h (-log q1[label]))
//   grad = weight ((1 - h) t (q - p) + h (q1 - onehot(label)))
// Bound by memory: V elements read, and V written for the gradient; the K
// entries are a few of the row. With m = max x, s = sum exp((x - m) / t),
// s1 = sum exp(x - m), and e_k = exp((z_k - max z) / t), Z = sum e:
//   KL = (sum e_k (z_k - max z) - sum e_k (x[i_k] - m)) / (Z t) - log Z + log s
// so one pass over the row with a running maximum gives the loss, and the
// gradient needs the row once more: from registers where it fits
// (staged_kernel), from memory, mostly a cache, where not (row_kernel).
//
// Exponents are formed as (x - m) c, not x c - m c: rows whose largest element
// is the type's lowest value (masked throughout) stay finite.

#include <cfloat>

#include "lm_common.h"

namespace churten {
namespace lm {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxWaves = kMaxThreads / kWave;
constexpr int kMaxEntries = 1024;
constexpr int64_t kMaxRows = int64_t(1) << 21;  // of one launch, a workgroup each
constexpr float kLog2e = 1.44269504088896340736f;

struct Args {
  ts_distill_args a;
  float* parts;  // (rows, splits, 3): m, s, s1 of each slice of a row
  int splits;
  int64_t first_row;  // of the launch
};

// The same value in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, x)));
}

// What a slice of a row sums to: the maximum, and relative to it the sums of
// the exponentials at the temperature and (HARD) at temperature 1.
template <bool HARD>
struct Sums {
  // The lowest finite value: masked logits of -infinity add exp(-infinity) = 0.
  float m = -FLT_MAX;
  float s = 0, s1 = 0;

  __device__ __forceinline__ void raise(float to, float c) {
    const float m2 = fmaxf(m, to);
    const float d = m - m2;
    s *= __builtin_amdgcn_exp2f(d * c);
    if constexpr (HARD) s1 *= __builtin_amdgcn_exp2f(d * kLog2e);
    m = m2;
  }
  template <int E>
  __device__ __forceinline__ void add(Vec<float, E> x, float c) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) top = fmaxf(top, x[i]);
    raise(top, c);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float d = x[i] - m;
      s += __builtin_amdgcn_exp2f(d * c);
      if constexpr (HARD) s1 += __builtin_amdgcn_exp2f(d * kLog2e);
    }
  }
};

// A row cut into aligned packs, and the elements before and after them. Those
// are fewer than E each; thread e < 2 E of the workgroup takes one.
template <typename T>
struct Row {
  static constexpr int E = kPack<T>;
  const T* x;
  int64_t lead, packs, V;

  __device__ __forceinline__ Row(const T* x_, int64_t V_) : x(x_), V(V_) {
    const int past = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16);
    lead = std::min<int64_t>(V, past == 0 ? 0 : (16 - past) / int(sizeof(T)));
    packs = (V - lead) / E;
  }

  __device__ __forceinline__ Vec<T, E> pack(int64_t p) const {
    return reinterpret_cast<const Vec<T, E>*>(x + lead)[p];
  }
  // The element that edge slot e < 2 E stands for, -1 if none.
  __device__ __forceinline__ int64_t edge(int e) const {
    if (e < E) return e < lead ? e : -1;
    const int64_t at = lead + packs * E + (e - E);
    return e < 2 * E && at < V ? at : -1;
  }
};

// Reduces COUNT values over the workgroup, but for those of the bits NEVER;
// every thread gets the results.
template <uint32_t NEVER, int COUNT, typename Op>
__device__ __forceinline__ void block_reduce(float (&v)[COUNT], float (*lds)[kMaxWaves], Op op,
                                             float neutral) {
  const int waves = blockDim.x / kWave, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if ((NEVER >> i & 1) == 0) v[i] = reduce<kWave>(v[i], op);
  }
  if (waves > 1 && lane == 0) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      if ((NEVER >> i & 1) == 0) lds[i][wave] = v[i];
    }
  }
  __syncthreads();
  if (waves == 1) return;
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if ((NEVER >> i & 1) != 0) continue;
    const int at = lane % kMaxWaves;
    v[i] = reduce<kMaxWaves>(at < waves ? lds[i][at] : neutral, op);
  }
}

__device__ __forceinline__ float weight_of(const ts_distill_args& a, int64_t n, int64_t b) {
  return a.weight == nullptr ? 1.0f
                             : a.weight[n * a.weight_stride_n + b * a.weight_stride_b];
}

// Entries are looked through four at a time; those that fill up the last four
// are absent.
__host__ __device__ constexpr int padded(int K) { return (K + 3) / 4 * 4; }

// What the entries of an element sum to takes a look at all K of them, once for
// each entry. More than a wavefront's are first looked through for an element
// that several name: none does in a teacher's top K, and then an entry's own e
// is all that is taken off its element. Entries are put into a table of open
// addresses, at most half full, where two that name one element meet. bfloat16,
// 7616 rows of 4278 with hard labels, 153 entries: 44 us, 62 us without the
// table; 8192 rows of 131072, 64 entries: 800 us, 766 us without.
constexpr int kScanned = kWave;
__host__ __device__ constexpr int table_log2(int K) {
  return K <= kScanned ? 0 : 33 - __builtin_clz(K - 1);
}

// The workgroup's memory for a row's reductions, and what its entries find.
struct Shared {
  float tops[2][kMaxWaves];
  float sums[5][kMaxWaves];
  int repeated;  // two entries name one element
  int labelled;  // an entry names the label's
};

// Keeps the compiler from carrying what it computed from v, four registers of
// 16-bit elements, in the eight registers of their float32 values.
template <typename V>
__device__ __forceinline__ void forget(V& v) {
  auto bits = __builtin_bit_cast(Vec<uint32_t, 4>, v);
  asm volatile("" : "+v"(bits));
  v = __builtin_bit_cast(V, bits);
}

// What the gradient is formed from once the row's sums are known.
struct Scales {
  float m, c;      // exponents are (x - m) c
  float a, a1;     // factors of exp((x - m) / t) and exp(x - m)
  float soft, hard;  // what p and the label's one are subtracted with
};

template <bool HARD>
__device__ __forceinline__ float gradient(const Scales& k, float x) {
  const float d = x - k.m;
  float g = k.a * __builtin_amdgcn_exp2f(d * k.c);
  if constexpr (HARD) g = fmaf(k.a1, __builtin_amdgcn_exp2f(d * kLog2e), g);
  return g;
}

// Adds packs [begin, end) of a row, this thread's share, to its sums.
template <typename T, bool HARD>
__device__ __forceinline__ void add_packs(const Row<T>& row, int64_t begin, int64_t end, float c,
                                          Sums<HARD>& sums) {
  constexpr int E = kPack<T>;
  constexpr int kAhead = 4;
  const int threads = blockDim.x;
  int64_t p = begin + threadIdx.x;
  for (; p + (kAhead - 1) * threads < end; p += kAhead * threads) {
    Vec<T, E> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = row.pack(p + j * threads);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) sums.template add<E>(widen<T, E>(v[j]), c);
  }
  for (; p < end; p += threads) sums.template add<E>(widen<T, E>(row.pack(p)), c);
}

template <typename T>
__device__ __forceinline__ Row<T> row_of(const ts_distill_args& a, int64_t n, int64_t b) {
  return Row<T>(static_cast<const T*>(a.logits.data) + n * a.logits.stride_n +
                    b * a.logits.stride_b,
                a.V);
}

template <typename T>
__device__ __forceinline__ T* grad_of(const ts_distill_args& a, int64_t n, int64_t b) {
  return a.grad.data == nullptr
             ? nullptr
             : static_cast<T*>(a.grad.data) + n * a.grad.stride_n + b * a.grad.stride_b;
}

// Entry k of a row: its element of the row, -1 if it is absent, and its logit.
struct Entry {
  int index;
  float z;
};
__device__ __forceinline__ Entry entry_of(const ts_distill_args& a, int64_t n, int64_t b, int k) {
  const int64_t i = index_at(a.index, n, b, k);
  const float z = (static_cast<const float*>(a.teacher.data) + n * a.teacher.stride_n +
                   b * a.teacher.stride_b)[k];
  return {i >= 0 && i < a.V && z != -INFINITY ? static_cast<int>(i) : -1, z};
}

// An entry's e and its terms of the totals Z, sum e (z - max z), sum e (x - m).
__device__ __forceinline__ float add_entry(const Entry& entry, float x, float z_top, float m,
                                           float c, float* total) {
  if (entry.index < 0) return 0;
  const float d = entry.z - z_top;
  const float e = __builtin_amdgcn_exp2f(d * c);
  if (!(e <= 0)) {  // p log q is 0 where p is, also for q = 0
    total[0] += e;
    total[1] = fmaf(e, d, total[1]);
    total[2] = fmaf(e, x - m, total[2]);
  }
  return e;
}

// The label of a row (-1: none, or the replica has no share of it) and that share.
struct Label {
  int64_t at = -1;
  float share = 0;
};
template <bool HARD>
__device__ __forceinline__ Label label_of(const ts_distill_args& a, int64_t n, int64_t b) {
  Label label;
  if constexpr (HARD) {
    label.share = a.hard[n];
    label.at = index_at(a.labels, n, b);
    if (label.at >= a.V || label.share == 0) label.at = -1;
  }
  return label;
}

// A replica with nothing but hard labels has no teacher, whatever the entries hold.
template <bool HARD>
__device__ __forceinline__ void drop_unshared(float (&total)[5], const Label& label) {
  if (HARD && label.share == 1) total[2] = 0;
}

// The loss from the totals: s, s1, Z, sum e (z - max z), sum e (x - m).
__device__ __forceinline__ float loss_of(const float (&total)[5], float m, float temperature,
                                         float weight, const Label& label, float label_x) {
  float loss = 0;
  if (total[2] != 0) {
    const float kl =
        (total[3] - total[4]) / (total[2] * temperature) - logf(total[2]) + logf(total[0]);
    loss = (1 - label.share) * temperature * temperature * kl;
  }
  if (label.at >= 0) loss += label.share * (logf(total[1]) - (label_x - m));
  return weight * loss;
}

template <bool HARD>
__device__ __forceinline__ Scales scales_of(const float (&total)[5], float m, float c,
                                            float temperature, float weight,
                                            const Label& label) {
  Scales k;
  k.m = m;
  k.c = c;
  k.soft = total[2] != 0 ? weight * (1 - label.share) * temperature : 0;
  k.hard = HARD && label.at >= 0 ? weight * label.share : 0;
  k.a = k.soft / total[0];
  k.a1 = HARD ? k.hard / total[1] : 0;
  return k;
}

// What the entries that name element i (e at `entry`, index at `index`) sum to.
// Entries that name one element all get the same sum in the same order.
__device__ __forceinline__ float taken_at(int i, const int* index, const float* entry, int K) {
  // Four entries at a time and without branches: an element's own entry is
  // mostly the only one, but all have to be looked at.
  float taken = 0;
#pragma unroll 2
  for (int other = 0; other < K; other += 4) {
    const auto who = *reinterpret_cast<const Vec<int, 4>*>(index + other);
    const auto what = *reinterpret_cast<const Vec<float, 4>*>(entry + other);
#pragma unroll
    for (int j = 0; j < 4; ++j) taken += who[j] == i ? what[j] : 0.0f;
  }
  return taken;
}

// The gradient at an element x whose entries sum to `taken`.
template <bool HARD>
__device__ __forceinline__ float taken_gradient(const Scales& k, float Z, float x, float taken,
                                                bool labelled) {
  float g = gradient<HARD>(k, x);
  if (Z != 0) g -= taken * (k.soft / Z);
  if (HARD && labelled) g -= k.hard;
  return g;
}

template <typename T, bool HARD>
__device__ __forceinline__ Vec<T, kPack<T>> gradient_pack(const Scales& k, Vec<T, kPack<T>> v) {
  constexpr int E = kPack<T>;
  const Vec<float, E> x = widen<T, E>(v);
  Vec<float, E> g;
#pragma unroll
  for (int i = 0; i < E; ++i) g[i] = gradient<HARD>(k, x[i]);
  return narrow<T, E>(g);
}

// One slice of a row, read from memory for the sums and again for the gradient;
// the loss alone reads it once: bfloat16 16384 rows of 50001 258 us, 6.4 TB/s.
// With more than one slice the sums come from `parts`, which part_kernel wrote.
template <typename T, bool HARD>
__global__ __launch_bounds__(kMaxThreads) void row_kernel(Args args) {
  constexpr int E = kPack<T>;
  constexpr int kAhead = 4;
  const ts_distill_args& a = args.a;
  // The entries' indices (as ints), and their logits, later e; both padded.
  extern __shared__ __attribute__((aligned(16))) float entries[];
  __shared__ Shared shared;
  const int64_t row_at = args.first_row + blockIdx.x, n = row_at / a.B, b = row_at % a.B;
  const int t = threadIdx.x, threads = blockDim.x, K = static_cast<int>(a.K);
  const int split = blockIdx.y;
  const Row<T> row = row_of<T>(a, n, b);
  T* grad = grad_of<T>(a, n, b);
  const int64_t each = (row.packs + args.splits - 1) / args.splits;
  const int64_t begin = std::min(row.packs, each * split);
  const int64_t end = std::min(row.packs, begin + each);
  const int64_t edge = split == 0 ? row.edge(t) : -1;
  const float weight = weight_of(a, n, b);

  const auto zero_slice = [&] {
    for (int64_t p = begin + t; p < end; p += threads) {
      store_streaming<E>(grad + row.lead + p * E, Vec<T, E>{});
    }
    if (edge >= 0) grad[edge] = T(0);
  };
  if (weight == 0) {
    if (split == 0 && t == 0) a.loss[row_at] = 0;
    if (grad != nullptr) zero_slice();
    return;
  }

  const float temperature = a.temperature[n];
  const float c = kLog2e / temperature;
  int* index = reinterpret_cast<int*>(entries);
  float* entry = entries + padded(K);
  float z_top = -INFINITY;
  for (int k = t; k < padded(K); k += threads) {
    const Entry e = k < K ? entry_of(a, n, b, k) : Entry{-1, 0};
    index[k] = e.index;
    entry[k] = e.z;
    if (e.index >= 0) z_top = fmaxf(z_top, e.z);
  }
  Sums<HARD> sums;
  if (args.splits == 1) {
    add_packs<T, HARD>(row, begin, end, c, sums);
    if (edge >= 0) sums.template add<1>(Vec<float, 1>(static_cast<float>(row.x[edge])), c);
  } else if (t < args.splits) {
    const float* part = args.parts + (row_at * args.splits + t) * 3;
    sums.m = part[0];
    sums.s = part[1];
    sums.s1 = part[2];
  }
  float tops[2] = {sums.m, z_top};
  block_reduce<0>(tops, shared.tops, Largest{}, -INFINITY);
  sums.raise(tops[0], c);
  float total[5] = {sums.s, sums.s1, 0, 0, 0};
  for (int k = t; k < padded(K); k += threads) {
    const float x = index[k] >= 0 ? static_cast<float>(row.x[index[k]]) : 0.0f;
    entry[k] = add_entry({index[k], entry[k]}, x, tops[1], tops[0], c, total + 2);
  }
  block_reduce<HARD ? 0 : 2>(total, shared.sums, Plus{}, 0.0f);

  const Label label = label_of<HARD>(a, n, b);
  drop_unshared<HARD>(total, label);
  if (split == 0 && t == 0) {
    const float label_x = label.at >= 0 ? static_cast<float>(row.x[label.at]) : 0.0f;
    a.loss[row_at] = loss_of(total, tops[0], temperature, weight, label, label_x);
  }
  if (grad == nullptr) return;
  if (total[2] == 0 && label.at < 0) {
    zero_slice();
    return;
  }
  const Scales k = scales_of<HARD>(total, tops[0], c, temperature, weight, label);
  int64_t p = begin + t;
  for (; p + (kAhead - 1) * threads < end; p += kAhead * threads) {
    Vec<T, E> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = row.pack(p + j * threads);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      store_streaming<E>(grad + row.lead + (p + j * threads) * E, gradient_pack<T, HARD>(k, v[j]));
    }
  }
  for (; p < end; p += threads) {
    store_streaming<E>(grad + row.lead + p * E, gradient_pack<T, HARD>(k, row.pack(p)));
  }
  if (edge >= 0) grad[edge] = static_cast<T>(gradient<HARD>(k, static_cast<float>(row.x[edge])));

  // The entries' elements again: after the slice's stores.
  __syncthreads();
  const int64_t slice_begin = row.lead + begin * E, slice_end = row.lead + end * E;
  for (int j = t; j < K + (HARD ? 1 : 0); j += threads) {
    const int64_t i = j < K ? index[j] : label.at;
    if (i < 0) continue;
    const bool here = (i >= slice_begin && i < slice_end) ||
                      (split == 0 && (i < row.lead || i >= row.lead + row.packs * E));
    if (!here) continue;
    grad[i] = static_cast<T>(
        taken_gradient<HARD>(k, total[2], static_cast<float>(row.x[i]),
                             taken_at(static_cast<int>(i), index, entry, K), i == label.at));
  }
}

// Elements or packs of a row as a buffer whose bounds the hardware checks: a
// load beyond them gives 0, a store is dropped. Loads without branches keep the
// compiler's count of those in flight exact, so that the wait for one does not
// wait for all that follow.
struct Buffer {
  __amdgpu_buffer_rsrc_t buffer;

  __device__ __forceinline__ Buffer(const void* first, int bytes)
      : buffer(__builtin_amdgcn_make_buffer_rsrc(scalar(first), 0, uniform(bytes),
                                                 0x00020000)) {}
  template <typename V>
  __device__ __forceinline__ V load_pack(int pack) const {
    return __builtin_bit_cast(
        V, __builtin_amdgcn_raw_buffer_load_b128(buffer, pack * 16, 0, kStreaming));
  }
  template <typename V>
  __device__ __forceinline__ void store_pack(int pack, V v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Vec<uint32_t, 4>, v), buffer,
                                           pack * 16, 0, kStreaming);
  }
  // Element i, or 0 for i < 0.
  template <typename T>
  __device__ __forceinline__ T load_element(int i) const {
    const uint32_t byte = i < 0 ? ~0u : i * static_cast<uint32_t>(sizeof(T));
    if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(buffer, byte, 0, 0));
    } else {
      const uint16_t bits = __builtin_amdgcn_raw_buffer_load_b16(buffer, byte, 0, 0);
      return __builtin_bit_cast(T, bits);
    }
  }
  __device__ __forceinline__ uint32_t load_word(int i) const {
    return __builtin_amdgcn_raw_buffer_load_b32(buffer, i * 4, 0, 0);
  }

 private:
  static constexpr int kStreaming = 2;  // past the caches
  static __device__ __forceinline__ void* scalar(const void* p) {
    const auto bits = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = uniform(static_cast<int>(bits));
    const uint32_t hi = uniform(static_cast<int>(bits >> 32));
    return reinterpret_cast<void*>(uint64_t(hi) << 32 | lo);
  }
};

// A whole row, kept in registers between the sums and the gradient: at most
// STAGED packs and one entry per thread. The packs are summed as they arrive.
// Nothing outside a row's workgroup overlaps its phases; the rows of the CU's
// other workgroups do, and new wavefronts start as old ones end: workgroups
// that took rows in turn and loaded the next one behind the stores of the last
// were slower (bfloat16 8192 rows of 131072: 852 us against 795 us). Bound by
// memory: those rows 760 us, 5.7 TB/s; float32 4096 rows of 32000 178 us, 5.9 TB/s.
// Rows of a few packs per lane are bound by their instructions, two exponentials
// per element and pass with hard labels (bfloat16 28336 rows of 602: 37 us, 1.8 TB/s).
template <typename T, int STAGED, bool HARD>
__global__ __launch_bounds__(kMaxThreads) void staged_kernel(Args args) {
  constexpr int E = kPack<T>;
  const ts_distill_args& a = args.a;
  // The entries' indices (as ints) and e, both padded.
  extern __shared__ __attribute__((aligned(16))) float entries[];
  __shared__ Shared shared;
  const int t = threadIdx.x, threads = blockDim.x, K = static_cast<int>(a.K);
  const int64_t row_at = args.first_row + blockIdx.x, n = row_at / a.B, b = row_at % a.B;
  const Row<T> row = row_of<T>(a, n, b);
  const int packs = static_cast<int>(row.packs);
  T* grad = grad_of<T>(a, n, b);
  const Buffer to(grad + row.lead, packs * 16);
  const int edge = static_cast<int>(row.edge(t));
  const float weight = uniform(weight_of(a, n, b));
  if (weight == 0) {
    if (t == 0) a.loss[row_at] = 0;
    for (int p = t; p < packs; p += threads) to.store_pack(p, Vec<uint32_t, 4>{});
    if (edge >= 0) grad[edge] = T(0);
    return;
  }

  // Loads in the order of their use, which is that of their return. The
  // entries' indices go first and are looked at behind the packs' loads.
  const float temperature = uniform(a.temperature[n]);
  const Label label = label_of<HARD>(a, n, b);
  const bool wide = a.index.bits == 64;
  const Buffer indices(static_cast<const char*>(a.index.data) +
                           (n * a.index.stride_n + b * a.index.stride_b) * (wide ? 8 : 4),
                       K * (wide ? 8 : 4));
  const Buffer logits(static_cast<const float*>(a.teacher.data) + n * a.teacher.stride_n +
                          b * a.teacher.stride_b,
                      K * 4);
  const uint32_t index_lo = indices.load_word(wide ? 2 * t : t);
  const uint32_t index_hi = indices.load_word(2 * t + 1);
  const float z = __builtin_bit_cast(float, logits.load_word(t));
  const Buffer from(row.x + row.lead, packs * 16);
  Vec<T, E> staged[STAGED];
#pragma unroll
  for (int j = 0; j < STAGED; ++j) staged[j] = from.load_pack<Vec<T, E>>(t + j * threads);
  __builtin_amdgcn_sched_barrier(0);
  const int64_t at = wide ? static_cast<int64_t>(uint64_t(index_hi) << 32 | index_lo)
                          : static_cast<int32_t>(index_lo);
  const bool present = t < K && at >= 0 && at < a.V && z != -INFINITY;
  const Entry entry{present ? static_cast<int>(at) : -1, z};
  const Buffer elements(row.x, static_cast<int>(a.V * sizeof(T)));
  const T raw_edge = elements.load_element<T>(edge);
  const T raw_entry = elements.load_element<T>(entry.index);
  const T raw_label = elements.load_element<T>(static_cast<int>(label.at));
  __builtin_amdgcn_sched_barrier(0);

  const float c = kLog2e / temperature;
  Sums<HARD> sums;
  const int left = packs - uniform(t);  // packs from the wavefront's first on
#pragma unroll
  for (int j = 0; j < STAGED; ++j) {
    if (left > j * threads) {
      // Selected before it is widened: four registers, not eight.
      Vec<T, E> v = t % kWave < left - j * threads ? staged[j]
                                                   : Vec<T, E>(static_cast<T>(-INFINITY));
      forget(v);
      sums.template add<E>(widen<T, E>(v), c);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // All packs have arrived, also those that the wavefront has skipped.
#pragma unroll
  for (int j = 0; j < STAGED; ++j) forget(staged[j]);
  const float edge_x = edge >= 0 ? static_cast<float>(raw_edge) : -INFINITY;
  const float entry_x = static_cast<float>(raw_entry), label_x = static_cast<float>(raw_label);
  sums.template add<1>(Vec<float, 1>(edge_x), c);
  int* index = reinterpret_cast<int*>(entries);
  float* e = entries + padded(K);
  if (t < padded(K)) index[t] = entry.index;
  int* table = index + 2 * padded(K);
  const int slots_log2 = table_log2(K), slots = 1 << slots_log2;
  if (slots_log2 > 0) {
    for (int i = t; i < slots; i += threads) table[i] = -1;
  }
  if (t == 0) shared.repeated = shared.labelled = 0;
  float tops[2] = {sums.m, entry.index >= 0 ? entry.z : -INFINITY};
  block_reduce<0>(tops, shared.tops, Largest{}, -INFINITY);
  const float m = uniform(tops[0]);
  sums.raise(m, c);
  float total[5] = {sums.s, sums.s1, 0, 0, 0};
  const float own = add_entry(entry, entry_x, tops[1], m, c, total + 2);
  if (t < padded(K)) e[t] = own;
  if (entry.index >= 0) {
    if (slots_log2 > 0) {
      // Ends at a free slot: half of them stay free.
      for (uint32_t at = uint32_t(entry.index) * 0x9E3779B1u >> (32 - slots_log2);;
           at = (at + 1) & (slots - 1)) {
        const int other = atomicCAS(&table[at], -1, t);
        if (other < 0) break;
        if (index[other] == entry.index) {
          shared.repeated = 1;
          break;
        }
      }
    }
    if (HARD && entry.index == label.at) shared.labelled = 1;
  }
  block_reduce<HARD ? 0 : 2>(total, shared.sums, Plus{}, 0.0f);
#pragma unroll
  for (int i = 0; i < 5; ++i) total[i] = uniform(total[i]);
  drop_unshared<HARD>(total, label);
  if (t == 0) a.loss[row_at] = loss_of(total, m, temperature, weight, label, label_x);
  const float Z = total[2];
  const bool zero = Z == 0 && label.at < 0;
  const uint32_t keep = zero ? 0 : ~0u;
  const Scales k = scales_of<HARD>(total, m, c, temperature, weight, label);
#pragma unroll
  for (int j = 0; j < STAGED; ++j) {
    if (left > j * threads) {
      to.store_pack(t + j * threads,
                    __builtin_bit_cast(Vec<uint32_t, 4>,
                                       gradient_pack<T, HARD>(k, staged[j])) & keep);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (edge >= 0) grad[edge] = zero ? T(0) : static_cast<T>(gradient<HARD>(k, edge_x));

  // The entries' elements again: after the row's stores.
  __syncthreads();
  if (entry.index >= 0 && !zero) {
    const float taken = slots_log2 == 0 || shared.repeated != 0
                            ? taken_at(entry.index, index, e, K)
                            : own;
    grad[entry.index] = static_cast<T>(
        taken_gradient<HARD>(k, Z, entry_x, taken, entry.index == label.at));
  }
  if (HARD && label.at >= 0 && t == 0 && shared.labelled == 0) {
    grad[label.at] = static_cast<T>(taken_gradient<HARD>(k, Z, label_x, 0.0f, true));
  }
}

// The sums of one slice of a row, for rows too few to fill the chip.
template <typename T, bool HARD>
__global__ __launch_bounds__(kMaxThreads) void part_kernel(Args args) {
  const ts_distill_args& a = args.a;
  __shared__ Shared shared;
  const int64_t row_at = args.first_row + blockIdx.x, n = row_at / a.B, b = row_at % a.B;
  if (weight_of(a, n, b) == 0) return;
  const int split = blockIdx.y;
  const Row<T> row = row_of<T>(a, n, b);
  const int64_t each = (row.packs + args.splits - 1) / args.splits;
  const int64_t begin = std::min(row.packs, each * split);
  const int64_t end = std::min(row.packs, begin + each);
  const float c = kLog2e / a.temperature[n];
  Sums<HARD> sums;
  add_packs<T, HARD>(row, begin, end, c, sums);
  const int64_t edge = split == 0 ? row.edge(threadIdx.x) : -1;
  if (edge >= 0) sums.template add<1>(Vec<float, 1>(static_cast<float>(row.x[edge])), c);
  float tops[1] = {sums.m};
  block_reduce<0>(tops, shared.tops, Largest{}, -INFINITY);
  sums.raise(tops[0], c);
  float all[2] = {sums.s, sums.s1};
  block_reduce<HARD ? 0 : 2>(all, shared.sums, Plus{}, 0.0f);
  if (threadIdx.x == 0) {
    float* part = args.parts + (row_at * args.splits + split) * 3;
    part[0] = tops[0];
    part[1] = all[0];
    part[2] = all[1];
  }
}

struct Plan {
  int splits, threads, staged;
};

Plan plan_of(const ts_distill_args& a, int width) {
  const int64_t rows = a.N * a.B, packs = a.V * width / 16;
  const auto threads_for = [&](int64_t per) {
    return static_cast<int>(std::max<int64_t>(
        kWave, std::min<int64_t>(kMaxThreads, ceil_div(ceil_div(packs, per), kWave) * kWave)));
  };
  // Long rows too few to fill the chip are cut up: 20 rows of 50000 float32 14 us
  // (23 us whole), 64 of 32000 15 us (14 us); rows that no workgroup can hold
  // up to a row for each CU.
  if (rows <= (packs > 16 * kMaxThreads ? 256 : 32) && packs >= 4096) {
    const int splits = static_cast<int>(std::min<int64_t>(
        std::min<int64_t>(32, ceil_div(512, std::max<int64_t>(1, rows))), packs / 1024));
    if (splits > 1) return {splits, 256, 0};
  }
  if (a.grad.data == nullptr) return {1, std::min(512, threads_for(16)), 0};
  // As few packs per thread as a workgroup allows: few registers let more
  // wavefronts share a CU (bfloat16 16384 rows of 30000: 388 us with 4 packs, 434
  // us with 16; float32 4096 rows of 32000: 181 us with 8 packs, 187 us with 16;
  // with 8 packs of 16-bit elements and hard labels the registers are too many
  // for that: 8192 rows of 50001 442 us, 360 us with 16). A thread for each entry.
  const int staged = packs <= 4 * kMaxThreads                 ? 4
                     : width == 4 && packs <= 8 * kMaxThreads ? 8
                                                              : 16;
  const int threads = std::max(threads_for(staged),
                               static_cast<int>(ceil_div(a.K, kWave)) * kWave);
  if (packs <= int64_t(staged) * threads) return {1, threads, staged};
  return {1, kMaxThreads, 0};
}

template <typename T, bool HARD>
int launch(Args args, const Plan& plan, hipStream_t stream) {
  const int64_t rows = args.a.N * args.a.B;
  const int K = static_cast<int>(args.a.K);
  const size_t lds = static_cast<size_t>(padded(K)) * 8;
  const size_t staged_lds = lds + (K > kScanned ? sizeof(int) << table_log2(K) : 0);
  const dim3 block(plan.threads);
  for (args.first_row = 0; args.first_row < rows; args.first_row += kMaxRows) {
    const uint32_t x = static_cast<uint32_t>(std::min(kMaxRows, rows - args.first_row));
    const uint32_t splits = static_cast<uint32_t>(plan.splits);
    if (splits > 1) {
      hipLaunchKernelGGL((part_kernel<T, HARD>), dim3(x, splits), block, 0, stream, args);
      if (const int err = launched()) return err;
    }
    // Without a gradient the first slice has all that is left to do.
    const dim3 grid(x, args.a.grad.data == nullptr ? 1 : splits);
    switch (plan.staged) {
      case 0: hipLaunchKernelGGL((row_kernel<T, HARD>), grid, block, lds, stream, args); break;
      case 4:
        hipLaunchKernelGGL((staged_kernel<T, 4, HARD>), grid, block, staged_lds, stream, args);
        break;
      case 8:
        if constexpr (sizeof(T) == 4) {
          hipLaunchKernelGGL((staged_kernel<T, 8, HARD>), grid, block, staged_lds, stream, args);
        }
        break;
      default:
        hipLaunchKernelGGL((staged_kernel<T, 16, HARD>), grid, block, staged_lds, stream, args);
        break;
    }
    if (const int err = launched()) return err;
  }
  return 0;
}

bool args_ok(const ts_distill_args* a, ts_dtype dtype) {
  constexpr int64_t kMost = (int64_t(1) << 31) - 2;
  if (a == nullptr ||
      (dtype != TS_FLOAT32 && dtype != TS_FLOAT16 && dtype != TS_BFLOAT16)) {
    return false;
  }
  if (a->N < 0 || a->N > kMaxReplicas || a->B < 0 || a->B > kMost || a->V < 0 || a->V > kMost ||
      a->K < 0 || a->K > kMaxEntries) {
    return false;
  }
  return true;
}

}  // namespace
}  // namespace lm
}  // namespace churten

using namespace churten::lm;

extern "C" {

size_t ts_distill_workspace(const ts_distill_args* args, ts_dtype dtype) {
  if (!args_ok(args, dtype)) return 0;
  const Plan plan = plan_of(*args, dtype == TS_FLOAT32 ? 4 : 2);
  return plan.splits > 1 ? static_cast<size_t>(args->N * args->B) * plan.splits * 12 : 0;
}

int ts_distill(const ts_distill_args* args, ts_dtype dtype, void* workspace,
               size_t workspace_bytes, void* stream) {
  if (!args_ok(args, dtype)) return kInvalid;
  const ts_distill_args& a = *args;
  if (a.N == 0 || a.B == 0) return 0;
  const bool hard = a.hard != nullptr;
  if (a.loss == nullptr || a.temperature == nullptr || (a.V > 0 && a.logits.data == nullptr) ||
      (a.K > 0 && (a.teacher.data == nullptr || !index_ok(a.index))) ||
      hard != (a.labels.data != nullptr) || (hard && !index_ok(a.labels))) {
    return kInvalid;
  }
  const Plan plan = plan_of(a, dtype == TS_FLOAT32 ? 4 : 2);
  const size_t need = ts_distill_workspace(args, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
    return kInvalid;
  }
  const Args full{a, static_cast<float*>(workspace), plan.splits, 0};
  const auto s = static_cast<hipStream_t>(stream);
  return by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    return hard ? launch<T, true>(full, plan, s) : launch<T, false>(full, plan, s);
  });
}

}  // extern "C"
