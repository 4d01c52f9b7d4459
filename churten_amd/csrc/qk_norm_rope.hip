// qk_norm_rope.hip -- the norm of each query and key head and the rotation by
// position, in one pass over the heads, and its backward pass.
//
// A head x (D elements, learned weight w of its replica):
//   r = rsqrt(mean(x^2) + eps),  y = x r w,  out = R y
// with R the rotation of y's first `rot` elements, pair by pair, by the angles
// of the head's position. Backward, from dout:
//   u = R^T dout,  dw = sum over tokens and heads of u x r,
//   dx = r (u w - x r^2 mean(u w x))
// Both are bound by memory: D elements read and written per head forward, 2 D
// read and D written backward.
//
// A head is held by G lanes, two packs of VE elements each, chosen so that a
// lane holds both members of its pairs and the rotation crosses no lanes; the
// norm and the backward's dot product are reduced over the G lanes. Everything
// between load and store is float32, rounded once.

#include "lm_common.h"

namespace churten {
namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxWidth = 512;
// Wavefronts per SIMD that the registers must leave room for. Forward of 8 x 4096 x
// 20 bfloat16 heads of 128, neighbouring pairs: 59 us; with room for 5, where
// registers spill, 65 us.
constexpr int kWaves = 4;

// Where the pairs lie.
enum Pairing {
  kAcross,  // (first pack's i-th, second pack's i-th element)
  kInside,  // neighbouring elements of one pack
};

struct Side {
  ts_heads in, dout, out;  // dout: backward only
  const void* weight;
  int64_t weight_stride;
  void* weight_grad;  // backward only
  int64_t heads;
  int64_t per, shares;  // heads per unit of work, units per token
  int64_t blocks;  // workgroups per replica
};

struct QkArgs {
  Side side[2];  // queries, keys
  const float* cos;
  const float* sin;
  int64_t table_stride;
  ts_index positions;
  float* parts;  // (N, both sides' blocks, D)
  int64_t M, P;
  int D, rot, pair_units;
  float eps, inverse_width;
  bool interleaved;
};

// This workgroup's side, read with its index from the kernel's arguments (which
// the first argument begins): selecting between both sides' fields kept both in
// scalar registers, more than there are.
__device__ __forceinline__ Side side_of(int which) {
  using Args = const __attribute__((address_space(4))) QkArgs;
  const auto* args = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
  Side side;
  __builtin_memcpy(&side, &args->side[which], sizeof(Side));
  return side;
}

// The two packs that a lane holds in slot `unit`: element offsets, whether they
// rotate, and where their angles start. Lanes left over repeat the last pack, and
// a pack without a second one stands for both: they load, compute and store
// what another does and only their sums are left out (not in_a, not in_b), which
// takes no branches.
struct Unit {
  int a, b, angle_a, angle_b;
  bool in_a, in_b, turn_a, turn_b;
};

// Neighbouring lanes hold neighbouring packs, in both of their halves. FULL: the
// head rotates throughout and its packs are as many as the lanes hold.
template <int VE, Pairing PAIRING, bool FULL>
__device__ __forceinline__ Unit unit_of(const QkArgs& s, int unit) {
  Unit u;
  if constexpr (FULL) {
    u.in_a = u.in_b = u.turn_a = u.turn_b = true;
    u.a = unit * VE;
    u.b = s.D / 2 + unit * VE;
    u.angle_a = PAIRING == kInside ? u.a / 2 : u.a;
    u.angle_b = u.b / 2;
    return u;
  }
  if constexpr (PAIRING == kInside) {
    const int half = (s.D / VE + 1) / 2;
    u.in_a = unit < half;
    unit = min(unit, half - 1);
    u.a = unit * VE;
    u.b = (half + unit) * VE;
    u.in_b = u.in_a && u.b < s.D;
    if (u.b >= s.D) u.b = u.a;
    u.turn_a = u.a < s.rot;
    u.turn_b = u.b < s.rot;
    u.angle_a = u.a / 2;
    u.angle_b = u.b / 2;
    return u;
  }
  const int half = ((s.D - s.rot) / VE + 1) / 2;
  u.in_a = u.in_b = unit < s.pair_units + half;
  unit = min(unit, s.pair_units + half - 1);
  u.turn_a = u.turn_b = unit < s.pair_units;
  u.angle_a = u.angle_b = unit * VE;
  if (!u.turn_a) {
    const int past = unit - s.pair_units;
    u.a = s.rot + past * VE;
    u.b = s.rot + (half + past) * VE;
    u.in_b = u.in_a && u.b < s.D;
    if (u.b >= s.D) u.b = u.a;
  } else if (VE == 1 && s.interleaved) {
    u.a = 2 * unit;
    u.b = u.a + 1;
  } else {
    u.a = unit * VE;
    u.b = s.rot / 2 + unit * VE;
  }
  return u;
}

template <int VE, typename T>
__device__ __forceinline__ Vec<T, VE> load_if(bool here, const T* p) {
  Vec<T, VE> v = {};
  if (here) v = load<VE>(p);
  return v;
}

// Past the caches where a store covers whole 128-byte lines; parts of lines
// are put together in them (bfloat16 forward of 8 x 4096 x 20 heads of 96:
// 59 us past them, 53 us through them; of 8 x 16384 x 20 heads of 128: 237 us
// and 249 us).
template <int VE, bool WHOLE_LINES, typename T>
__device__ __forceinline__ void put(T* p, Vec<T, VE> v) {
  if constexpr (WHOLE_LINES) {
    store_streaming<VE>(p, v);
  } else {
    store<VE>(p, v);
  }
}

// The angles of a pack (pair): VE of them across packs, VE / 2 inside one.
template <int VE, Pairing PAIRING>
struct Turn {
  static constexpr int kAngles = PAIRING == kInside ? VE / 2 : VE;
  Vec<float, kAngles> cos, sin;
  bool on;

  __device__ __forceinline__ void fetch(const QkArgs& s, bool turn, int64_t row, int at) {
    cos = sin = Vec<float, kAngles>{};
    on = turn && row >= 0;
    if (on) {
      cos = load<kAngles>(s.cos + row + at);
      sin = load<kAngles>(s.sin + row + at);
    }
  }
};

template <int VE, int SIGN>
__device__ __forceinline__ void rotate_inside(Vec<float, VE>& v, const Turn<VE, kInside>& t) {
  if (t.on) {
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      const float sin = t.sin[i] * SIGN, a = v[2 * i], b = v[2 * i + 1];
      v[2 * i] = a * t.cos[i] - b * sin;
      v[2 * i + 1] = b * t.cos[i] + a * sin;
    }
  }
}

// Rotates the packs a, b by their angles, or back for SIGN = -1. What does not
// turn is left alone: turned by no angle, a x 1 - b x 0, an infinity would reach the
// element beside it.
template <int VE, Pairing PAIRING, int SIGN>
__device__ __forceinline__ void rotate(Vec<float, VE>& a, Vec<float, VE>& b,
                                       const Turn<VE, PAIRING>& ta,
                                       const Turn<VE, PAIRING>& tb) {
  if constexpr (PAIRING == kAcross) {
    if (ta.on) {
      const Vec<float, VE> sin = ta.sin * float(SIGN), x = a, y = b;
      a = x * ta.cos - y * sin;
      b = y * ta.cos + x * sin;
    }
  } else {
    rotate_inside<VE, SIGN>(a, ta);
    rotate_inside<VE, SIGN>(b, tb);
  }
}

// sum + x y of a lane's packs a and b, as far as they count.
template <int E, bool FULL>
__device__ __forceinline__ float dot(const Unit& u, Vec<float, E> xa, Vec<float, E> ya,
                                     Vec<float, E> xb, Vec<float, E> yb, float sum) {
  float of_a = FULL ? sum : 0, of_b = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) of_a = fmaf(xa[i], ya[i], of_a);
  if constexpr (FULL) of_b = of_a;
#pragma unroll
  for (int i = 0; i < E; ++i) of_b = fmaf(xb[i], yb[i], of_b);
  return FULL ? of_b : sum + (u.in_a ? of_a : 0) + (u.in_b ? of_b : 0);
}

__device__ __forceinline__ int64_t table_row(const QkArgs& s, int64_t n, int64_t m) {
  if (s.rot == 0) return -1;
  const int64_t p = index_at(s.positions, n, m);
  return p >= 0 && p < s.P ? p * s.table_stride : -1;
}

// A group's unit of work: up to HEADS heads of one token, which share its
// angles; a side has M * shares units. The position is loaded ahead of the
// heads: loads return in order, and the angles wait for it.
struct Work {
  int64_t units, step, at, m;
  int shares, per, heads, h, count;

  __device__ __forceinline__ Work(const QkArgs& s, const Side& side, int64_t first,
                                  int64_t step_)
      : units(s.M * side.shares),
        step(step_),
        at(first),
        shares(static_cast<int>(side.shares)),
        per(static_cast<int>(side.per)),
        heads(static_cast<int>(side.heads)) {
    place();
  }
  __device__ __forceinline__ bool more() const { return at < units; }
  __device__ __forceinline__ void place() {
    if (shares == 1) {
      m = at;
      h = 0;
    } else if (units < int64_t(1) << 32) {
      const uint32_t u = static_cast<uint32_t>(at), q = u / static_cast<uint32_t>(shares);
      m = q;
      h = static_cast<int>(u - q * static_cast<uint32_t>(shares)) * per;
    } else {
      m = at / shares;
      h = static_cast<int>(at % shares) * per;
    }
    count = min(per, heads - h);
  }
  __device__ __forceinline__ void next() {
    at += step;
    place();
  }
};

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
// bfloat16, 8 x 16384 x 20 heads of 128: 223 us, 6.0 TB/s; 8 x 4096 x 20 heads of 96
// 51 us, 4.9 TB/s.
template <typename T, int VE, int G, int S, Pairing PAIRING, int HEADS, bool FULL>
__global__ __launch_bounds__(kThreads, kWaves) void forward_kernel(QkArgs s) {
  constexpr int kGroups = kThreads / G;
  constexpr bool kWholeLines = FULL && G * VE * sizeof(T) % 128 == 0;
  const int64_t n = blockIdx.y;
  const bool is_k = blockIdx.x >= s.side[0].blocks;
  const Side side = side_of(is_k);
  const int64_t block = int64_t(blockIdx.x) - (is_k ? s.side[0].blocks : 0);
  const int lane = threadIdx.x % G;
  const T* weight = static_cast<const T*>(side.weight) + n * side.weight_stride;
  const T* in = static_cast<const T*>(side.in.data) + n * side.in.stride_n;
  T* out = static_cast<T*>(side.out.data) + n * side.out.stride_n;
  Unit u[S];
  Vec<float, VE> wa[S], wb[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    u[i] = unit_of<VE, PAIRING, FULL>(s, lane + i * G);
    wa[i] = widen<T, VE>(load<VE>(weight + u[i].a));
    wb[i] = widen<T, VE>(load<VE>(weight + u[i].b));
  }
  Work work(s, side, block * kGroups + threadIdx.x / G, side.blocks * kGroups);
  for (; work.more(); work.next()) {
    const int64_t m = work.m, row = table_row(s, n, m);
    const int h = work.h, count = work.count;
    const T* x = in + m * side.in.stride_m + h * side.in.stride_h;
    T* y = out + m * side.out.stride_m + h * side.out.stride_h;
    Vec<T, VE> xa[HEADS][S], xb[HEADS][S];
    Turn<VE, PAIRING> ta[S], tb[S];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const bool here = k == 0 || k < count;
        xa[k][i] = load_if<VE>(here, x + k * side.in.stride_h + u[i].a);
        xb[k][i] = load_if<VE>(here, x + k * side.in.stride_h + u[i].b);
      }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
      ta[i].fetch(s, u[i].turn_a, row, u[i].angle_a);
      if constexpr (PAIRING == kInside) tb[i].fetch(s, u[i].turn_b, row, u[i].angle_b);
    }
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
      float square = 0;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const Vec<float, VE> a = widen<T, VE>(xa[k][i]), b = widen<T, VE>(xb[k][i]);
        square = dot<VE, FULL>(u[i], a, a, b, b, square);
      }
      const float r = rsqrtf(reduce<G>(square, Plus{}) * s.inverse_width + s.eps);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        Vec<float, VE> a = widen<T, VE>(xa[k][i]) * r * wa[i];
        Vec<float, VE> b = widen<T, VE>(xb[k][i]) * r * wb[i];
        rotate<VE, PAIRING, 1>(a, b, ta[i], tb[i]);
        T* to = y + k * side.out.stride_h;
        if (k == 0 || k < count) {
          put<VE, kWholeLines>(to + u[i].a, narrow<T, VE>(a));
          put<VE, kWholeLines>(to + u[i].b, narrow<T, VE>(b));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// The weights' gradient is summed in a lane's registers over all its units, then
// over the workgroup; a second launch adds up the workgroups. bfloat16, 8 x 16384 x
// 20 heads of 128: 376 us, 5.4 TB/s.
template <typename T, int VE, int G, int S, Pairing PAIRING, int HEADS, bool FULL>
__global__ __launch_bounds__(kThreads, kWaves) void backward_kernel(QkArgs s) {
  constexpr int kGroups = kThreads / G;
  constexpr bool kWholeLines = FULL && G * VE * sizeof(T) % 128 == 0;
  // Every group's share of dw: its lanes' columns.
  __shared__ float shares[kGroups * G * S * 2 * VE];
  const int64_t n = blockIdx.y;
  const bool is_k = blockIdx.x >= s.side[0].blocks;
  const Side side = side_of(is_k);
  const int64_t block = int64_t(blockIdx.x) - (is_k ? s.side[0].blocks : 0);
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const T* weight = static_cast<const T*>(side.weight) + n * side.weight_stride;
  const T* in = static_cast<const T*>(side.in.data) + n * side.in.stride_n;
  const T* dout = static_cast<const T*>(side.dout.data) + n * side.dout.stride_n;
  T* out = static_cast<T*>(side.out.data) + n * side.out.stride_n;
  Unit u[S];
  Vec<float, VE> wa[S], wb[S], dwa[S], dwb[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    u[i] = unit_of<VE, PAIRING, FULL>(s, lane + i * G);
    wa[i] = widen<T, VE>(load<VE>(weight + u[i].a));
    wb[i] = widen<T, VE>(load<VE>(weight + u[i].b));
    dwa[i] = dwb[i] = Vec<float, VE>{};
  }
  Work work(s, side, block * kGroups + group, side.blocks * kGroups);
  for (; work.more(); work.next()) {
    const int64_t m = work.m, row = table_row(s, n, m);
    const int h = work.h, count = work.count;
    const T* x = in + m * side.in.stride_m + h * side.in.stride_h;
    const T* dy = dout + m * side.dout.stride_m + h * side.dout.stride_h;
    T* dx = out + m * side.out.stride_m + h * side.out.stride_h;
    Vec<T, VE> xa[HEADS][S], xb[HEADS][S], da[HEADS][S], db[HEADS][S];
    Turn<VE, PAIRING> ta[S], tb[S];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const bool here = k == 0 || k < count;
        xa[k][i] = load_if<VE>(here, x + k * side.in.stride_h + u[i].a);
        xb[k][i] = load_if<VE>(here, x + k * side.in.stride_h + u[i].b);
        da[k][i] = load_if<VE>(here, dy + k * side.dout.stride_h + u[i].a);
        db[k][i] = load_if<VE>(here, dy + k * side.dout.stride_h + u[i].b);
      }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
      ta[i].fetch(s, u[i].turn_a, row, u[i].angle_a);
      if constexpr (PAIRING == kInside) tb[i].fetch(s, u[i].turn_b, row, u[i].angle_b);
    }
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
      Vec<float, VE> ua[S], ub[S];
      float square = 0, along = 0;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const Vec<float, VE> a = widen<T, VE>(xa[k][i]), b = widen<T, VE>(xb[k][i]);
        square = dot<VE, FULL>(u[i], a, a, b, b, square);
        ua[i] = widen<T, VE>(da[k][i]);
        ub[i] = widen<T, VE>(db[k][i]);
        rotate<VE, PAIRING, -1>(ua[i], ub[i], ta[i], tb[i]);
        along = dot<VE, FULL>(u[i], ua[i] * wa[i], a, ub[i] * wb[i], b, along);
      }
      const float r = rsqrtf(reduce<G>(square, Plus{}) * s.inverse_width + s.eps);
      const float c = reduce<G>(along, Plus{}) * s.inverse_width * r * r;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const Vec<float, VE> a = widen<T, VE>(xa[k][i]), b = widen<T, VE>(xb[k][i]);
        T* to = dx + k * side.out.stride_h;
        if (k == 0 || k < count) {
          dwa[i] += ua[i] * (a * r);
          dwb[i] += ub[i] * (b * r);
          put<VE, kWholeLines>(to + u[i].a, narrow<T, VE>((ua[i] * wa[i] - a * c) * r));
          put<VE, kWholeLines>(to + u[i].b, narrow<T, VE>((ub[i] * wb[i] - b * c) * r));
        }
      }
    }
  }
  // The groups' shares, added up in their order.
#pragma unroll
  for (int i = 0; i < S; ++i) {
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      if (u[i].in_a) shares[group * s.D + u[i].a + j] = dwa[i][j];
      if (u[i].in_b) shares[group * s.D + u[i].b + j] = dwb[i][j];
    }
  }
  __syncthreads();
  for (int col = threadIdx.x; col < s.D; col += kThreads) {
    float sum = 0;
#pragma unroll 4
    for (int g = 0; g < kGroups; ++g) sum += shares[g * s.D + col];
    if (side.blocks == 1) {
      static_cast<T*>(side.weight_grad)[n * s.D + col] = static_cast<T>(sum);
    } else {
      s.parts[(n * (s.side[0].blocks + s.side[1].blocks) + blockIdx.x) * s.D + col] = sum;
    }
  }
}

// Adds up the workgroups' shares of one replica's q or k weight gradient. A
// wavefront takes 64 columns and every 16th workgroup's share; then the 16
// sums, in order. 8 x 511 shares of 128: 5.4 us, latency.
constexpr int kJoinWaves = 16;

template <typename T>
__global__ __launch_bounds__(kJoinWaves* kWave) void weight_grad_kernel(QkArgs s) {
  __shared__ float sums[kJoinWaves][kWave];
  const int64_t n = blockIdx.y;
  const bool is_k = blockIdx.z == 1;
  const Side side = side_of(is_k);
  if (side.blocks <= 1) return;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int col = blockIdx.x * kWave + lane;
  const float* parts =
      s.parts + col +
      (n * (s.side[0].blocks + s.side[1].blocks) + (is_k ? s.side[0].blocks : 0)) * s.D;
  float sum = 0;
  if (col < s.D) {
#pragma unroll 8
    for (int64_t b = wave; b < side.blocks; b += kJoinWaves) sum += parts[b * s.D];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || col >= s.D) return;
  for (int i = 1; i < kJoinWaves; ++i) sum += sums[i][lane];
  static_cast<T*>(side.weight_grad)[n * s.D + col] = static_cast<T>(sum);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Elements per pack and lanes per head for a shape: the widest packs that its
// pairs divide into. Two lanes are the fewest with those, four with others
// (bfloat16 backward of 24 x 619 x 64 heads of 32: 46 us, 57 us with four).
struct Split {
  int pack, lanes, slots;
  Pairing pairing;
  bool full;
};

Split split_of(const ts_qk_shape& s, int width) {
  const bool inside = (s.flags & TS_INTERLEAVED) != 0;
  for (int pack : {16 / width, 8 / width}) {
    const int64_t unit = inside ? s.rot : s.rot / 2;
    if (inside && pack != 16 / width) break;
    if (s.D % pack != 0 || unit % pack != 0) continue;
    const int64_t units = ceil_div(s.D, 2 * pack);
    if (units <= kWave) {
      const int lanes = std::max(pack == 16 / width ? 2 : 4, pow2_at_least(units));
      const bool full = pack == 16 / width && s.rot == s.D && s.D == 2 * lanes * pack;
      return {pack, lanes, 1, inside ? kInside : kAcross, full};
    }
  }
  const int64_t units = s.rot / 2 + ceil_div(s.D - s.rot, 2);
  if (units <= kWave) return {1, std::max(4, pow2_at_least(units)), 1, kAcross, false};
  return {1, kWave, 4, kAcross, false};
}

// Heads of a token that a group holds at a time (one where a head takes several
// slots per lane): as many as leave room for enough wavefronts. Forward of 8 x
// 4096 x 20 bfloat16 heads of 96: 1 head 58 us, 2 heads 53 us; of 80 with 40
// rotating 69 and 57 us; of 128 the same. float32 backward of 3 x 1021 x 9 heads
// of 80: 1 head 13.8 us, 2 heads 12.0 us. Registers spill with 4 heads forward,
// and with 2 in the backward of 16-bit types.
constexpr int kForwardHeads = 2;
template <typename T>
constexpr int kBackwardHeads = sizeof(T) == 4 ? 2 : 1;

// Workgroups over the whole chip: each replica's and side's share by its heads,
// none with less than one round of work. Forward of 8 x 16384 x 20 bfloat16 heads
// of 128: 8192 workgroups 237 us, 16384 230 us, 32768 224 us, 65536 222 us; the
// backward, whose workgroups each leave a share of the weights' gradient: 1024
// 403 us, 2048 389 us, 4096 382 us, 8192 384 us.
constexpr int64_t kForwardBlocks = 32768, kBackwardBlocks = 4096;

void set_blocks(QkArgs& a, int64_t N, int groups, int64_t most, int64_t blocks) {  // N >= 1
  const int64_t heads = a.side[0].heads + a.side[1].heads;
  for (Side& side : a.side) {
    side.shares = ceil_div(side.heads, most);
    side.per = ceil_div(side.heads, side.shares);
    const int64_t rounds = ceil_div(a.M * side.shares, groups);
    const int64_t share = std::max<int64_t>(1, blocks * side.heads / (heads * N));
    side.blocks = std::max<int64_t>(1, std::min(rounds, share));
  }
}

bool shape_ok(const ts_qk_shape* s) {
  if (s == nullptr) return false;
  constexpr int64_t kMost = int64_t(1) << 31;
  if (s->N < 0 || s->N > kMaxReplicas || s->M < 0 || s->M >= kMost || s->Hq < 1 ||
      s->Hq >= 65536 || s->Hk < 1 || s->Hk >= 65536 || s->D < 1 || s->D > kMaxWidth ||
      s->rot < 0 || s->rot > s->D || s->rot % 2 != 0 || s->P < 0 ||
      (s->flags & ~TS_INTERLEAVED) != 0) {
    return false;
  }
  if (s->N == 0 || s->M == 0) return true;
  return s->rot == 0 || (index_ok(s->positions) &&
                         (s->P == 0 || (s->cos != nullptr && s->sin != nullptr)));
}

QkArgs args_of(const ts_qk_shape& s, int width, bool backward, Split* split) {
  QkArgs a{};
  *split = split_of(s, width);
  a.cos = s.cos;
  a.sin = s.sin;
  a.table_stride = s.table_stride;
  a.positions = s.positions;
  a.M = s.M;
  a.P = s.P;
  a.D = static_cast<int>(s.D);
  a.rot = static_cast<int>(s.rot);
  a.pair_units = static_cast<int>(s.rot / 2 / split->pack);
  a.eps = s.eps;
  a.inverse_width = 1.0f / static_cast<float>(s.D);
  a.interleaved = (s.flags & TS_INTERLEAVED) != 0;
  a.side[0].heads = s.Hq;
  a.side[1].heads = s.Hk;
  if (s.N > 0) {
    const int most = split->slots > 1 ? 1
                     : !backward      ? kForwardHeads
                     : width == 4     ? kBackwardHeads<float>
                                      : kBackwardHeads<_Float16>;
    set_blocks(a, s.N, kThreads / split->lanes, most,
               backward ? kBackwardBlocks : kForwardBlocks);
  }
  return a;
}

// Calls `f` with the pack, lanes, slots, pairing and fullness as constants.
template <typename T, typename F>
int by_split(const Split& s, F&& f) {
  constexpr int kWide = kPack<T>;
  using std::integral_constant;
  constexpr integral_constant<int, 1> one{};
  constexpr integral_constant<int, kWide> wide{};
  constexpr integral_constant<Pairing, kAcross> across{};
  constexpr integral_constant<Pairing, kInside> inside{};
  constexpr std::true_type full{};
  constexpr std::false_type partial{};
  if (s.slots == 4) {
    return f(one, integral_constant<int, kWave>{}, integral_constant<int, 4>{}, across, partial);
  }
  const auto widest = [&](auto lanes) {
    if (s.pairing == kInside) {
      return s.full ? f(wide, lanes, one, inside, full) : f(wide, lanes, one, inside, partial);
    }
    return s.full ? f(wide, lanes, one, across, full) : f(wide, lanes, one, across, partial);
  };
  if (s.lanes == 2) return widest(integral_constant<int, 2>{});
  return by_lanes(s.lanes, [&](auto lanes) {
    if constexpr (decltype(lanes)::value * 2 * kWide <= kMaxWidth) {
      if (s.pack == kWide) return widest(lanes);
    }
    if (s.pack == kWide / 2) {
      return f(integral_constant<int, kWide / 2>{}, lanes, one, across, partial);
    }
    return f(one, lanes, one, across, partial);
  });
}

size_t parts_bytes(const QkArgs& a, int64_t N) {
  if (a.side[0].blocks <= 1 && a.side[1].blocks <= 1) return 0;
  return static_cast<size_t>(N * (a.side[0].blocks + a.side[1].blocks) * a.D) * sizeof(float);
}

int width_of(ts_dtype dtype) {
  return dtype == TS_FLOAT32 ? 4 : dtype == TS_FLOAT16 || dtype == TS_BFLOAT16 ? 2 : 0;
}

}  // namespace
}  // namespace lm
}  // namespace churten

using namespace churten::lm;

extern "C" {

int ts_qk_norm_rope(const ts_qk_shape* shape, ts_dtype dtype, ts_heads q, ts_heads k,
                    const void* q_weight, int64_t qw_stride, const void* k_weight,
                    int64_t kw_stride, ts_heads q_out, ts_heads k_out, void* stream) {
  if (!shape_ok(shape) || width_of(dtype) == 0) return kInvalid;
  const ts_qk_shape& s = *shape;
  if (s.N == 0 || s.M == 0) return 0;
  if (q.data == nullptr || k.data == nullptr || q_out.data == nullptr ||
      k_out.data == nullptr || q_weight == nullptr || k_weight == nullptr) {
    return kInvalid;
  }
  Split split;
  QkArgs a = args_of(s, width_of(dtype), false, &split);
  a.side[0].in = q;
  a.side[1].in = k;
  a.side[0].out = q_out;
  a.side[1].out = k_out;
  a.side[0].weight = q_weight;
  a.side[0].weight_stride = qw_stride;
  a.side[1].weight = k_weight;
  a.side[1].weight_stride = kw_stride;
  const dim3 grid(static_cast<uint32_t>(a.side[0].blocks + a.side[1].blocks),
                  static_cast<uint32_t>(s.N));
  return by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    return by_split<T>(split, [&](auto pack, auto lanes, auto slots, auto pairing, auto full) {
      constexpr int kHeads = slots == 1 ? kForwardHeads : 1;
      hipLaunchKernelGGL((forward_kernel<T, pack, lanes, slots, pairing, kHeads, full>), grid,
                         dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
      return launched();
    });
  });
}

size_t ts_qk_norm_rope_grad_workspace(const ts_qk_shape* shape, ts_dtype dtype) {
  if (!shape_ok(shape) || width_of(dtype) == 0) return 0;
  Split split;
  return parts_bytes(args_of(*shape, width_of(dtype), true, &split), shape->N);
}

int ts_qk_norm_rope_grad(const ts_qk_shape* shape, ts_dtype dtype, ts_heads dq, ts_heads dk,
                         ts_heads q, ts_heads k, const void* q_weight, int64_t qw_stride,
                         const void* k_weight, int64_t kw_stride, ts_heads q_grad,
                         ts_heads k_grad, void* qw_grad, void* kw_grad, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (!shape_ok(shape) || width_of(dtype) == 0) return kInvalid;
  const ts_qk_shape& s = *shape;
  if (s.N == 0) return 0;
  if (qw_grad == nullptr || kw_grad == nullptr || q_weight == nullptr || k_weight == nullptr ||
      (s.M > 0 && (dq.data == nullptr || dk.data == nullptr || q.data == nullptr ||
                   k.data == nullptr || q_grad.data == nullptr || k_grad.data == nullptr))) {
    return kInvalid;
  }
  Split split;
  QkArgs a = args_of(s, width_of(dtype), true, &split);
  const size_t need = parts_bytes(a, s.N);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
    return kInvalid;
  }
  a.parts = static_cast<float*>(workspace);
  a.side[0].in = q;
  a.side[1].in = k;
  a.side[0].dout = dq;
  a.side[1].dout = dk;
  a.side[0].out = q_grad;
  a.side[1].out = k_grad;
  a.side[0].weight = q_weight;
  a.side[0].weight_stride = qw_stride;
  a.side[1].weight = k_weight;
  a.side[1].weight_stride = kw_stride;
  a.side[0].weight_grad = qw_grad;
  a.side[1].weight_grad = kw_grad;
  const auto st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(a.side[0].blocks + a.side[1].blocks),
                  static_cast<uint32_t>(s.N));
  return by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    const int err = by_split<T>(split, [&](auto pack, auto lanes, auto slots, auto pairing,
                                           auto full) {
      constexpr int kHeads = slots == 1 ? kBackwardHeads<T> : 1;
      hipLaunchKernelGGL((backward_kernel<T, pack, lanes, slots, pairing, kHeads, full>), grid,
                         dim3(kThreads), 0, st, a);
      return launched();
    });
    if (err != 0 || need == 0) return err;
    hipLaunchKernelGGL(weight_grad_kernel<T>,
                       dim3(static_cast<uint32_t>(ceil_div(s.D, kWave)),
                            static_cast<uint32_t>(s.N), 2),
                       dim3(kJoinWaves * kWave), 0, st, a);
    return launched();
  });
}

}  // extern "C"
