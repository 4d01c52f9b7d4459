// embedding.hip -- scaled rows of every replica's embedding table, and the
// tables' gradient.
//
// Forward: out[n][b] = scale * W[n][tok[n][b]]. A copy by rows: bound by memory.
//
// Gradient: dW[n][v] = scale * sum_{b: tok[n][b] = v} dout[n][b], a sum by
// token. Adding rows with atomics would make the order, and with it the last
// bits, a matter of timing; here the tokens are sorted by (token, position),
// so that each table row's sum is one run of the sorted list, added up in the
// order of its positions:
//   1. sort_kernel sorts tiles of the token list in LDS; merge_kernel joins up
//      to kFan sorted runs per launch (none for lists of one tile).
//   2. sum_kernel: its summing groups each take some consecutive entries of the
//      sorted list, a chunk, whatever runs they are of (words' frequencies fall
//      as 1/rank: equal shares of the list are equal work, equal shares of the
//      table are not). A run inside one chunk is written to the table's
//      gradient at once; the parts of a run that crosses chunks go to a
//      float32 workspace.
//   3. join_kernel adds up the parts of the runs that cross chunks, in order.
// Zeros for the rows that no token names are written by further workgroups of
// the merges, whose few searches leave the memory idle (without merges, of
// sum_kernel). They know such rows from the witnesses that sort_kernel left.
// A call of few tokens takes one launch instead (direct_kernel).

#include "lm_common.h"

namespace churten {
namespace lm {
namespace {

constexpr int kThreads = 256;

// A lane's pack of a row of D elements. A row's last pack starts early enough
// to be whole, so its first elements are also the pack before's: both lanes
// load, compute and store the same values there. Only rows shorter than a pack
// (NARROW) go element by element.
template <typename T, bool NARROW>
struct Pack {
  static constexpr int E = kPack<T>;
  bool any;     // the lane has a pack
  int64_t col;  // its first element
  int count;    // its elements (E but for NARROW)
  int fresh;    // the elements from here on are not also the pack before's

  __device__ __forceinline__ Pack(int64_t pack, int64_t D) {
    const int64_t at = pack * E;
    any = at < D;
    count = NARROW ? static_cast<int>(D) : E;
    col = NARROW ? 0 : std::min<int64_t>(at, D - E);
    fresh = static_cast<int>(at - col);
  }
  template <typename U>
  __device__ __forceinline__ Vec<U, E> load_from(const U* row) const {
    if constexpr (NARROW) return load_first<E>(row, count);
    return load<E>(row + col);
  }
  template <typename U>
  __device__ __forceinline__ Vec<U, E> stream_from(const U* row) const {
    if constexpr (NARROW) return load_first<E>(row, count);
    return load_streaming<E>(row + col);
  }
  template <typename U>
  __device__ __forceinline__ void store_to(U* row, Vec<U, E> v) const {
    if constexpr (NARROW) return store_first<E>(row, v, count);
    store<E>(row + col, v);
  }
  template <typename U>
  __device__ __forceinline__ void stream_to(U* row, Vec<U, E> v) const {
    if constexpr (NARROW) return store_first<E>(row, v, count);
    store_streaming<E>(row + col, v);
  }
  template <typename U>
  __device__ __forceinline__ void put_to(U* row, Vec<U, E> v, bool past) const {
    if (past) {
      asm volatile("");  // keeps the compiler from making the two stores one, without the hint
      stream_to(row, v);
      asm volatile("");
    } else {
      store_to(row, v);
    }
  }
  // row += v, where two lanes must not both do so.
  template <typename U>
  __device__ __forceinline__ void add_to(U* row, Vec<float, E> v) const {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (i >= fresh && i < count) {
        row[col + i] = static_cast<U>(static_cast<float>(row[col + i]) + v[i]);
      }
    }
  }
};

// Whether a table's gradient is written past the caches: not where a wavefront's
// parts of its rows end inside lines of 128 bytes, which are put together in them
// (float32 4 x 30 tokens x 1001, 60000 rows: 240 us past them, 199 us through them;
// bfloat16 8 x 9000 x 512, 32000 rows: 88 us and 90 us; 23 x 4 x 226, two rows to a
// wavefront, 44 us and 46 us).
template <typename T, int G>
__device__ __forceinline__ bool past_caches(const ts_rows& table) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(table.data) |
                        uint64_t(table.stride_n) * sizeof(T) |
                        uint64_t(table.stride_b) * sizeof(T);
  return G < kWave || bits % 128 == 0;
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
struct LookupArgs {
  ts_rows weight, out;
  ts_index tokens;
  int64_t B, V, D;
  float scale;
};

// G lanes per row, a 16-byte pack each, ROWS rows per group in flight: the
// token of each row is a load that its table row waits for. bfloat16, 8 x 16384
// rows of 1024 out of 50000: 70 to 75 us, 4.9 to 5.2 TB/s (1 row per group 89 us, 4 rows
// 74 us beside 70).
constexpr int kLookupRows = 2;

template <typename T, int G, int ROWS, bool NARROW>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupArgs a) {
  constexpr int E = kPack<T>;
  constexpr int kGroups = kThreads / G;
  const int64_t n = blockIdx.z;
  const Pack<T, NARROW> pack(int64_t(blockIdx.y) * G + threadIdx.x % G, a.D);
  if (!pack.any) return;
  const int64_t first = int64_t(blockIdx.x) * (kGroups * ROWS) + threadIdx.x / G;
  const T* weight = static_cast<const T*>(a.weight.data) + n * a.weight.stride_n;
  T* out = static_cast<T*>(a.out.data) + n * a.out.stride_n;
  int64_t token[ROWS];
  Vec<T, E> row[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    token[i] = index_at(a.tokens, n, std::min(first + i * kGroups, a.B - 1));
  }
  // Without branches between them; a row of no token is loaded as the first.
  for (Vec<T, E>& r : row) r = Vec<T, E>{};
  if (a.V > 0) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool known = token[i] >= 0 && token[i] < a.V;
      row[i] = pack.load_from(weight + (known ? token[i] : 0) * a.weight.stride_b);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t b = first + i * kGroups;
    const bool known = token[i] >= 0 && token[i] < a.V;
    const Vec<T, E> scaled = narrow<T, E>(widen<T, E>(row[i]) * a.scale);
    if (b < a.B) pack.stream_to(out + b * a.out.stride_b, known ? scaled : Vec<T, E>{});
  }
}

template <typename T, int G, int ROWS, bool NARROW>
int launch_lookup(const LookupArgs& a, int64_t N, hipStream_t stream) {
  const int64_t packs = ceil_div(a.D, kPack<T>);
  const int64_t x = ceil_div(a.B, kThreads / G * ROWS), y = ceil_div(packs, G);
  if (x > kMaxBlocks || y > 65535) return kInvalid;
  const dim3 grid(static_cast<uint32_t>(x), static_cast<uint32_t>(y), static_cast<uint32_t>(N));
  hipLaunchKernelGGL((lookup_kernel<T, G, ROWS, NARROW>), grid, dim3(kThreads), 0, stream, a);
  return launched();
}

// ---------------------------------------------------------------------------
// Gradient: the sorted token list
// ---------------------------------------------------------------------------
// The list's order is by token, then position. Tokens outside [0, V) become V
// and sort to the end.
constexpr int kSortThreadsLog2 = 10;
constexpr int kSortThreads = 1 << kSortThreadsLog2;
constexpr int kDigitLog2 = 8;  // bits of a token per pass, at most
constexpr int kDigits = 1 << kDigitLog2;
constexpr int kFan = 16;  // runs joined per launch
constexpr int kFanLog2 = 4;

// A table row's witness is a position of its token. Only rows with tokens get
// one; what the others hold is whatever the workspace held, and is told from a
// witness by looking the token up.
struct SortArgs {
  ts_index tokens;
  int32_t* token;     // (lists, B), sorted tile by tile
  int32_t* position;  // (lists, B)
  int32_t* witness;   // (lists, V)
  int64_t B, V;
  int bits;        // of a token
  int digit_log2;  // of them per pass
};

// Orders what a wavefront's lanes write to LDS before what they read next.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// List n's tokens at first, first + step, ...: COUNT loads together. Past the
// list's end (B >= 1): its last.
template <int COUNT>
__device__ __forceinline__ void load_tokens(const ts_index& t, int64_t n, int64_t first, int step,
                                            int64_t B, int64_t (&token)[COUNT]) {
  const auto load_all = [&](auto kind) {
    const auto* from = static_cast<const decltype(kind)*>(t.data) + n * t.stride_n;
    decltype(kind) got[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) got[i] = from[std::min(first + i * step, B - 1) * t.stride_b];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) token[i] = got[i];
  };
  if (t.bits == 64) {
    load_all(int64_t{});
  } else {
    load_all(int32_t{});
  }
}

// Sorts one tile of one list, R words per thread, by passes over the tokens'
// digits from the lowest, each of which keeps the order of the pass before. A
// word is a token above its place in the tile: 32 bits where the tokens leave
// room. In a pass, lanes with the same digit find each other by one ballot per
// bit; a word's place is the number of words with lower digits, of those with
// its own in earlier wavefronts, in this one's earlier words and in its earlier
// lanes. What bounds it is latency, of two trips to memory and of the passes: 2 x
// 4096 of 32000 tokens, two passes, 8.6 us; 4 x 16 tiles of 131072 tokens, three
// passes, 11 us. Four words per thread instead of one spare a launch that merges
// (2000 tokens x 8, 500 rows: 17 us, 27 us with 1024-word tiles).
template <typename Word, int R_LOG2>
__global__ __launch_bounds__(kSortThreads) void sort_kernel(SortArgs a) {
  constexpr int R = 1 << R_LOG2, kTileLog2 = kSortThreadsLog2 + R_LOG2, kTile = 1 << kTileLog2;
  constexpr int kWaves = kSortThreads / kWave;
  __shared__ Word buf[kSortThreads * R];
  __shared__ int count[kWaves][kDigits];  // of each wavefront's words
  __shared__ int start[kDigits];
  __shared__ int total[kDigits / kWave];
  const int64_t list = blockIdx.y;
  const int64_t begin = int64_t(blockIdx.x) * kTile;
  const int n = static_cast<int>(std::min<int64_t>(kTile, a.B - begin));
  const int t = threadIdx.x, lane = t % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(t / kWave), waves = blockDim.x / kWave;
  const int mine = wave * kWave * R + lane;  // the thread's words: every kWave-th from here
  int64_t token[R];
  load_tokens<R>(a.tokens, list, begin + mine, kWave, a.B, token);
  Word w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int at = mine + r * kWave;
    if (token[r] < 0 || token[r] >= a.V) token[r] = a.V;
    w[r] = at < n ? Word(token[r]) << kTileLog2 | at : ~Word(0);  // past the end: last
    // Tokens at several positions: any of them will do.
    if (at < n && token[r] < a.V) {
      a.witness[list * a.V + token[r]] = static_cast<int32_t>(begin + at);
    }
  }
  for (int low = 0; low < a.bits; low += a.digit_log2) {
    const int width = std::min(a.digit_log2, a.bits - low), digits = 1 << width;
    for (int d = lane; d < digits; d += kWave) count[wave][d] = 0;
    int digit[R], rank[R];
    uint32_t same_lo[R], same_hi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      digit[r] = static_cast<int>(w[r] >> (kTileLog2 + low)) & (digits - 1);
      same_lo[r] = same_hi[r] = ~0u;
    }
    for (int b = 0; b < width; ++b) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int bit = __builtin_amdgcn_sbfe(digit[r], b, 1);  // 0 or -1
        const uint64_t set = __ballot(bit != 0);
        same_lo[r] &= ~(static_cast<uint32_t>(set) ^ bit);
        same_hi[r] &= ~(static_cast<uint32_t>(set >> 32) ^ bit);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int before =
          __builtin_amdgcn_mbcnt_hi(same_hi[r], __builtin_amdgcn_mbcnt_lo(same_lo[r], 0));
      const int all = __builtin_popcount(same_lo[r]) + __builtin_popcount(same_hi[r]);
      wave_fence();
      const int earlier = count[wave][digit[r]];
      wave_fence();
      if (before == 0) count[wave][digit[r]] = earlier + all;
      rank[r] = earlier + before;
    }
    __syncthreads();
    int all = 0, through = 0;
    if (t < digits) {
      for (int v = 0; v < waves; ++v) {
        const int here = count[v][t];
        count[v][t] = all;
        all += here;
      }
    }
    if (t < kDigits) {
      through = all;
#pragma unroll
      for (int step = 1; step < kWave; step *= 2) {
        const int lower = __shfl_up(through, step, kWave);
        if (lane >= step) through += lower;
      }
      if (lane == kWave - 1) total[wave] = through;
    }
    __syncthreads();
    if (t < digits) {
      for (int v = 0; v < wave; ++v) through += total[v];
      start[t] = through - all;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      buf[start[digit[r]] + count[wave][digit[r]] + rank[r]] = w[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = buf[mine + r * kWave];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int at = mine + r * kWave;
    if (at < n) {
      a.token[list * a.B + begin + at] = static_cast<int32_t>(w[r] >> kTileLog2);
      a.position[list * a.B + begin + at] =
          static_cast<int32_t>(begin + static_cast<int64_t>(w[r] & (kTile - 1)));
    }
  }
}

struct ZeroArgs {
  ts_rows weight_grad;
  ts_index tokens;
  const int32_t* witness;
  int64_t witness_stride;  // per replica: 0 where the tokens are shared
  int64_t B, V, D;
  int64_t first, end;  // of the units (kZeroRows rows for each group of a workgroup)
  int64_t units;       // per replica
};

// A group of G lanes zeroes those without tokens of its kZeroRows rows: bound by
// writing (float32 8 x 32000 x 512, 3266 of them with tokens: 82 us for 471 MB
// behind a merge).
template <typename T, int G, bool NARROW>
__device__ __forceinline__ void zero_rows(const ZeroArgs& a, int64_t unit) {
  constexpr int E = kPack<T>;
  constexpr int kGroups = kThreads / G;
  constexpr int kZeroRows = G < 16 ? G : 16;
  const int64_t n = unit / a.units;
  const int64_t first = (unit % a.units * kGroups + threadIdx.x / G) * kZeroRows;
  const int lane = threadIdx.x % G;
  // Lane i of the group looks at its i-th row.
  const int64_t mine = first + lane % kZeroRows;
  bool named = true;
  if (mine < a.V) {
    const int32_t at = a.witness[n * a.witness_stride + mine];
    named = at >= 0 && at < a.B && index_at(a.tokens, n, at) == mine;
  }
  const uint64_t all = __ballot(named) >> (threadIdx.x % kWave - lane);
  const bool past = past_caches<T, G>(a.weight_grad);
  T* out = static_cast<T*>(a.weight_grad.data) + n * a.weight_grad.stride_n;
#pragma unroll
  for (int i = 0; i < kZeroRows; ++i) {
    if ((all >> i & 1) != 0) continue;
    T* row = out + (first + i) * a.weight_grad.stride_b;
    for (int64_t at = lane; at * E < a.D; at += G) {
      Pack<T, NARROW>(at, a.D).put_to(row, Vec<T, E>{}, past);
    }
  }
}

struct MergeArgs {
  const int32_t* from_token;
  const int32_t* from_position;
  int32_t* to_token;
  int32_t* to_position;
  int64_t lists, B;
  int run_log2;  // length of the sorted runs (each list's last may be shorter)
};

// Joins each FAN neighbouring runs into one: an entry's place is the sum of its
// ranks in all of them, where equal tokens of earlier runs come before it and
// of later ones behind. What bounds it is the number of loads. A wavefront's 64
// entries are neighbours in their run, so first its lanes find, one each, the
// ranks of the first and the last of them in every run, and every entry
// searches only between those, in all runs in step, so that FAN loads are in
// flight. 8340 tokens, 3 runs: 12 us; 28901 tokens, 8 runs: 16 us, 19 us as 16 runs.
template <int FAN>
__device__ __forceinline__ void merge_runs(const MergeArgs& a, int64_t list, int64_t block) {
  const int64_t first = (block * kThreads + threadIdx.x) / kWave * kWave;
  if (first >= a.B) return;
  const int lane = threadIdx.x % kWave;
  const int64_t last = std::min(a.B, first + kWave) - 1;
  const int64_t i = std::min(first + lane, last);
  const int64_t length = int64_t(1) << a.run_log2;
  const int64_t group = i >> (a.run_log2 + kFanLog2) << (a.run_log2 + kFanLog2);
  const int64_t there = std::min(a.B - group, length * kFan);
  const int32_t* runs = a.from_token + list * a.B + group;
  const int own = __builtin_amdgcn_readfirstlane(static_cast<int>((i - group) >> a.run_log2));
  const int token = runs[i - group];

  // Lane r: the first entry's rank in run r; lane FAN + r: the last entry's.
  int bound = 0;
  {
    const int run = lane % FAN;
    const int target = runs[(lane < FAN ? first : last) - group] + (run < own ? 1 : 0);
    const int32_t* entries = runs + run * length;
    // Eighths at a time: a lane's seven probes are in flight together, and their
    // latency is what this costs. The rank is in [bound, bound + left].
    int left = static_cast<int>(
        std::max<int64_t>(0, std::min(length, there - run * length)));
    while (left > 0) {
      const int part = (left + 7) / 8;
      int below = 0;
#pragma unroll
      for (int k = 1; k < 8; ++k) {
        if (k * part <= left && entries[bound + k * part - 1] < target) ++below;
      }
      bound += below * part;
      left = (below + 1) * part <= left && below < 7 ? part - 1 : left - below * part;
    }
    if (run == own) bound = 0;
  }
  int below[FAN], end[FAN], widest = 0;
#pragma unroll
  for (int r = 0; r < FAN; ++r) {
    below[r] = __builtin_amdgcn_readlane(bound, r);
    end[r] = __builtin_amdgcn_readlane(bound, FAN + r);
    widest = std::max(widest, end[r] - below[r]);
  }
  // The largest power of two that is not above the widest range; 0 for none.
  for (int step = widest > 0 ? 1 << (31 - __builtin_clz(widest)) : 0; step > 0; step >>= 1) {
    int probe[FAN];
#pragma unroll
    for (int r = 0; r < FAN; ++r) {
      // Past the range's end: some entry of the group, not looked at.
      probe[r] = runs[std::min(r * length + below[r] + step - 1, there - 1)];
    }
#pragma unroll
    for (int r = 0; r < FAN; ++r) {
      if (below[r] + step <= end[r] && probe[r] < token + (r < own ? 1 : 0)) below[r] += step;
    }
  }
  if (first + lane > last) return;
  int64_t rank = (i - group) & (length - 1);
#pragma unroll
  for (int r = 0; r < FAN; ++r) rank += below[r];
  a.to_token[list * a.B + group + rank] = token;
  a.to_position[list * a.B + group + rank] = a.from_position[list * a.B + i];
}

// The first workgroups merge, the others zero.
template <typename T, int G, bool NARROW, int FAN>
__global__ __launch_bounds__(kThreads) void merge_kernel(MergeArgs a, ZeroArgs z) {
  const int64_t block = blockIdx.x, each = (a.B + kThreads - 1) / kThreads;
  if (block < a.lists * each) {
    merge_runs<FAN>(a, block / each, block % each);
  } else if (z.first + block - a.lists * each < z.end) {
    zero_rows<T, G, NARROW>(z, z.first + block - a.lists * each);
  }
}

struct SumArgs {
  ts_rows weight_grad, grad;
  const int32_t* token;     // the sorted list
  const int32_t* position;
  float* parts;  // (N, chunks, 2, D): a chunk's share of the run that began
                 // before it, and of the one that goes on after it
  int64_t list_stride;  // per replica: 0 where the tokens are shared
  int64_t N, B, V, D;
  int64_t chunks, slices;
  int64_t sum_blocks;  // per replica
  int chunk;
  float scale;
  bool accumulate;
};

template <typename T, int G, bool NARROW>
__device__ __forceinline__ void write_row(const SumArgs& a, const Pack<T, NARROW>& pack, T* out,
                                          int token, Vec<float, kPack<T>> sum) {
  T* row = out + int64_t(token) * a.weight_grad.stride_b;
  if (a.accumulate) {
    pack.add_to(row, sum * a.scale);
  } else {
    pack.put_to(row, narrow<T, kPack<T>>(sum * a.scale), past_caches<T, G>(a.weight_grad));
  }
}

// A group of G lanes sums one chunk's columns of G packs. With a wavefront per
// group everything but the columns is uniform, and the list is read with scalar
// loads. Bound by reading the rows: bfloat16 4 x 65536 x 1024 145 us, 4.7 TB/s with
// the table's rows written; 8 rows are in flight per group.
template <typename T, int G, bool NARROW>
__device__ __forceinline__ void sum_chunk(const SumArgs& a, int64_t n, int64_t unit) {
  constexpr int E = kPack<T>;
  constexpr int kAhead = 8;
  const int64_t chunk = unit / a.slices;
  const Pack<T, NARROW> pack(unit % a.slices * G + threadIdx.x % G, a.D);
  if (chunk >= a.chunks || !pack.any) return;
  const int32_t* tokens = a.token + n * a.list_stride;
  const int32_t* positions = a.position + n * a.list_stride;
  const T* grad = static_cast<const T*>(a.grad.data) + n * a.grad.stride_n;
  T* out = static_cast<T*>(a.weight_grad.data) + n * a.weight_grad.stride_n;
  float* parts = a.parts + ((n * a.chunks + chunk) * 2) * a.D;
  const int64_t begin = chunk * a.chunk;
  const int64_t end = std::min(a.B, begin + a.chunk);
  const int before = begin > 0 ? tokens[begin - 1] : -1;
  const int after = end < a.B ? tokens[end] : -1;
  int token = tokens[begin];
  Vec<float, E> sum = {};
  for (int64_t at = begin; at < end && token < a.V; at += kAhead) {
    int named[kAhead];
    int64_t place[kAhead];
    Vec<T, E> row[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      named[i] = tokens[std::min(at + i, end - 1)];
      place[i] = positions[std::min(at + i, end - 1)];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      row[i] = pack.stream_from(grad + place[i] * a.grad.stride_b);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (at + i >= end) break;
      if (named[i] != token) {  // the run ends inside the chunk
        if (token == before) {
          pack.store_to(parts, sum);
        } else {
          write_row<T, G, NARROW>(a, pack, out, token, sum);
        }
        sum = Vec<float, E>{};
        token = named[i];
        if (token >= a.V) break;
      }
      sum += widen<T, E>(row[i]);
    }
  }
  if (token >= a.V) return;
  if (token == before) {
    pack.store_to(parts, sum);
  } else if (token == after) {
    pack.store_to(parts + a.D, sum);
  } else {
    write_row<T, G, NARROW>(a, pack, out, token, sum);
  }
}

template <typename T, int G, bool NARROW>
__global__ __launch_bounds__(kThreads) void sum_kernel(SumArgs a, ZeroArgs z) {
  constexpr int kGroups = kThreads / G;
  int group = threadIdx.x / G;
  if constexpr (G == kWave) group = __builtin_amdgcn_readfirstlane(group);
  const int64_t block = blockIdx.x;
  if (block < a.N * a.sum_blocks) {
    sum_chunk<T, G, NARROW>(a, block / a.sum_blocks, block % a.sum_blocks * kGroups + group);
  } else if (z.first + block - a.N * a.sum_blocks < z.end) {
    zero_rows<T, G, NARROW>(z, z.first + block - a.N * a.sum_blocks);
  }
}

// One workgroup for each end of a chunk: where the run there goes on into the
// next chunk and began in this one, it adds up that run's parts. G lanes hold a
// row; each of the workgroup's groups adds an equal share of the parts, in
// order, then the shares are added by halves. Bound by latency, where one token
// is a large part of the list, and by the workgroups that find nothing to add:
// 8 x 128 chunks of 512 float32 4.7 us, 4 x 1024 of 1024 10 us. Some ends to a
// workgroup, or one to a wavefront, were no faster.
template <typename T, int G, bool NARROW>
__global__ __launch_bounds__(kThreads) void join_kernel(SumArgs a) {
  constexpr int E = kPack<T>;
  constexpr int kGroups = kThreads / G;
  constexpr int kAhead = 4;
  __shared__ Vec<float, E> share[kGroups][G];
  const uint32_t slices = static_cast<uint32_t>(a.slices);
  const int64_t n = blockIdx.y, chunk = blockIdx.x / slices, slice = blockIdx.x % slices;
  const int32_t* tokens = a.token + n * a.list_stride;
  const int64_t begin = chunk * a.chunk, end = begin + a.chunk;  // not the last chunk
  const int token = tokens[end];
  if (token >= a.V || tokens[end - 1] != token ||
      (begin > 0 && tokens[begin - 1] == token)) {
    return;
  }
  // The chunks after this one that begin with the run: 64 looked at at once.
  int64_t more = 0;
  for (;;) {
    const int64_t next = chunk + 1 + more + threadIdx.x % kWave;
    const uint64_t same =
        __ballot(next < a.chunks && tokens[next * a.chunk] == token);
    if (same != ~uint64_t(0)) {
      more += __builtin_ctzll(~same);
      break;
    }
    more += kWave;
  }
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int64_t count = more + 1;
  const int64_t each = (count + kGroups - 1) / kGroups;
  const int64_t to = std::min(count, each * (group + 1));
  const float* parts = a.parts + ((n * a.chunks + chunk) * 2) * a.D;
  T* out = static_cast<T*>(a.weight_grad.data) + n * a.weight_grad.stride_n;
  const Pack<T, NARROW> pack(slice * G + lane, a.D);
  Vec<float, E> sum = {};
  if (pack.any) {
    for (int64_t k0 = each * group; k0 < to; k0 += kAhead) {
      Vec<float, E> part[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t k = std::min(k0 + i, to - 1);
        part[i] = pack.load_from(parts + (2 * k + (k == 0 ? 1 : 0)) * a.D);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k0 + i < to) sum += part[i];
      }
    }
  }
  share[group][lane] = sum;
#pragma unroll
  for (int half = kGroups / 2; half > 0; half /= 2) {
    __syncthreads();
    if (group < half) share[group][lane] += share[group + half][lane];
  }
  if (group == 0 && pack.any) write_row<T, G, NARROW>(a, pack, out, token, share[0][lane]);
}

// ---------------------------------------------------------------------------
// Gradient of few tokens
// ---------------------------------------------------------------------------
constexpr int kDirectTokens = 256;
constexpr int64_t kDirectBlocks = 1024;

struct DirectArgs {
  ts_rows weight_grad, grad;
  ts_index tokens;
  int64_t B, V, D;
  int rows;  // of the table, per group
  float scale;
  bool accumulate;
};

// Every wavefront holds all the tokens, kWave to a register, and compares them
// with its own rows: a row's positions are the bits of the comparison, in
// order. One launch, where sorting takes three: float32 5 x 127 tokens x 33, 1003
// rows, 4.2 us, 16 us sorted.
template <typename T, int G, bool NARROW>
__global__ __launch_bounds__(kThreads) void direct_kernel(DirectArgs a) {
  constexpr int E = kPack<T>;
  constexpr int kGroups = kThreads / G, kInWave = kWave / G;
  constexpr int kWords = kDirectTokens / kWave;
  constexpr int kAhead = 4;
  const int64_t n = blockIdx.y;
  const int lane = threadIdx.x % kWave, group = lane / G;
  int64_t id[kWords] = {};
  if (a.B > 0) load_tokens<kWords>(a.tokens, n, lane, kWave, a.B, id);
  int token[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    const bool known = j * kWave + lane < a.B && id[j] >= 0 && id[j] < a.V;
    token[j] = known ? static_cast<int>(id[j]) : -1;
  }
  const T* grad = static_cast<const T*>(a.grad.data) + n * a.grad.stride_n;
  T* out = static_cast<T*>(a.weight_grad.data) + n * a.weight_grad.stride_n;
  const bool past = past_caches<T, G>(a.weight_grad);
  for (int i = 0; i < a.rows; ++i) {
    // The wavefront's rows lie together, one to a group; a workgroup's lie apart,
    // as the rows with many tokens are mostly neighbours.
    const int64_t first = (int64_t(i) * gridDim.x + blockIdx.x) * kGroups +
                          threadIdx.x / kWave * kInWave;
    // Most rows have no token.
    bool any = false;
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      any |= static_cast<uint64_t>(token[j] - first) < kInWave;
    }
    uint64_t at[kWords] = {};
    if (__ballot(any) != 0) {
#pragma unroll
      for (int g = 0; g < kInWave; ++g) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          const uint64_t same = __ballot(token[j] == static_cast<int>(first) + g);
          if (group == g) at[j] = same;
        }
      }
    }
    const int64_t v = first + group;
    if (v >= a.V) continue;
    bool named = false;
#pragma unroll
    for (int j = 0; j < kWords; ++j) named |= at[j] != 0;
    if (a.accumulate && !named) continue;
    for (int64_t p = lane % G; p * E < a.D; p += G) {
      const Pack<T, NARROW> pack(p, a.D);
      Vec<float, E> sum = {};
      if (named) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          uint64_t left = at[j];
          while (left != 0) {
            Vec<T, E> row[kAhead];  // behind the last position: that again, not added
            bool there[kAhead];
            int64_t b = 0;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              there[k] = left != 0;
              b = there[k] ? j * kWave + __builtin_ctzll(left) : b;
              left &= left - 1;
              row[k] = pack.load_from(grad + b * a.grad.stride_b);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              if (there[k]) sum += widen<T, E>(row[k]);
            }
          }
        }
      }
      T* to = out + v * a.weight_grad.stride_b;
      if (a.accumulate) {
        pack.add_to(to, sum * a.scale);
      } else {
        pack.put_to(to, narrow<T, E>(sum * a.scale), past);
      }
    }
  }
}

// How a gradient call is cut up and what its workspace holds.
struct GradPlan {
  bool direct;
  int64_t lists, tiles, slices, chunks;
  int lanes, chunk, merges, tile_log2;
  size_t list0, list1, witness, parts, bytes;
};

size_t rounded(int64_t bytes) { return static_cast<size_t>((bytes + 255) / 256 * 256); }

// Entries per chunk: 64 where that makes wavefronts enough for a quarter of the
// chip's, fewer, down to one batch of loads, where not (more chunks are more
// parts to join). bfloat16, 65536 tokens x 256: 8 entries 65 us, 32 entries 55
// us; float32, 8 x 8192 x 512: 16 entries 145 us, 64 entries 143 us; float32, 5 x
// 127 x 33 through here: 64 entries 31 us, 16 entries 16 us.
int chunk_for(int64_t N, int64_t B, int64_t slices, int lanes) {
  int chunk = 64;
  while (chunk > 8 && N * ceil_div(B, chunk) * slices * lanes / kWave < 2048) chunk /= 2;
  return chunk;
}

// Bits of the tokens, of V too, which stands for those outside the table.
int bits_of(int64_t V) { return V > 0 ? 64 - __builtin_clzll(static_cast<uint64_t>(V)) : 0; }

constexpr double kMostZeros = 384e6;  // bytes

GradPlan plan_of(int64_t width, int64_t N, int64_t B, int64_t V, int64_t D, bool shared) {
  GradPlan p{};
  const int64_t packs = ceil_div(D, 16 / width);
  p.lanes = std::max(4, std::min(kWave, pow2_at_least(packs)));
  p.direct = B <= kDirectTokens;
  if (p.direct) return p;
  p.lists = shared ? 1 : N;
  // Words per thread of a tile: one, four or, where that spares the list a merge
  // that the zeros would not hide, eight (5 x 6019 shared tokens x 24 float16 over
  // 49088 rows: 28 us, 36 us with a merge; float32 19 x 5000 x 608 over 3218 rows, 149
  // MB: 101 us, 105 us; 8 x 8192 shared x 512 over 32000 rows, 524 MB: 149 us, 145 us).
  const bool eight = B > 4 * kSortThreads && B <= 8 * kSortThreads &&
                     bits_of(V) + kSortThreadsLog2 + 3 <= 32 &&
                     double(N) * double(V) * double(D * width) <= kMostZeros;
  p.tile_log2 = kSortThreadsLog2 + (B <= kSortThreads ? 0 : eight ? 3 : 2);
  p.tiles = ceil_div(B, int64_t(1) << p.tile_log2);
  for (int64_t runs = p.tiles; runs > 1; runs = ceil_div(runs, kFan)) ++p.merges;
  p.slices = ceil_div(packs, p.lanes);
  p.chunk = chunk_for(N, B, p.slices, p.lanes);
  p.chunks = ceil_div(B, p.chunk);
  size_t at = 0;
  const auto take = [&at](int64_t bytes) {
    const size_t here = at;
    at += rounded(bytes);
    return here;
  };
  p.list0 = take(p.lists * B * 8);
  p.list1 = p.merges > 0 ? take(p.lists * B * 8) : p.list0;
  p.witness = take(p.lists * V * 4);
  p.parts = take(p.chunks > 1 ? N * p.chunks * 2 * D * 4 : 0);
  p.bytes = at;
  return p;
}

bool sizes_ok(int64_t N, int64_t B, int64_t V, int64_t D) {
  constexpr int64_t kMost = (int64_t(1) << 31) - 2;
  return N >= 0 && N <= kMaxReplicas && B >= 0 && B <= kMost && V >= 0 && V <= kMost && D >= 0 &&
         D <= kMost;
}

template <typename T, int G, bool NARROW>
int launch_direct(DirectArgs a, int64_t N, hipStream_t stream) {
  // A wavefront's worth of lanes' rows in turn, to look the tokens up less often,
  // but one where that would leave too few workgroups: float16 22 x 55 tokens x 51,
  // 22000 rows: 4 rows 13 us, 1 row 17 us; bfloat16 23 x 4 x 226, 21360 rows: 2 rows 43
  // us, 4 rows 55 us; float32 4 x 130 x 700, 30000 rows: 1 row 78 us, 4 rows 84 us; 5 x
  // 127 x 33, 1003 rows: 1 row 4.2 us, 4 rows 5.4 us.
  a.rows = std::max(1, std::min(4, kWave / G));
  while (a.rows > 1 && N * ceil_div(a.V, kThreads / G * a.rows) < kDirectBlocks) a.rows /= 2;
  while (ceil_div(a.V, kThreads / G * a.rows) > kMaxBlocks) a.rows *= 2;
  const int64_t blocks = ceil_div(a.V, kThreads / G * a.rows);
  hipLaunchKernelGGL((direct_kernel<T, G, NARROW>),
                     dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(N)),
                     dim3(kThreads), 0, stream, a);
  return launched();
}

template <typename T, int G, bool NARROW>
int launch_sorted(const GradPlan& p, SumArgs a, const ts_index& tokens, char* ws,
                  hipStream_t stream) {
  constexpr int64_t kGroups = kThreads / G, kRows = kGroups * (G < 16 ? G : 16);
  const int64_t zero_units = ceil_div(a.V, kRows);
  const int64_t units = a.accumulate ? 0 : a.N * zero_units;
  const auto zeros_before = [&](int merge) {  // of p.merges; without any: none
    return p.merges > 0 ? units * merge / p.merges : 0;
  };
  a.chunks = p.chunks;
  a.slices = p.slices;
  a.chunk = p.chunk;
  a.sum_blocks = ceil_div(p.chunks * p.slices, kGroups);
  const auto merge_blocks = [&](int m) {
    return p.lists * ceil_div(a.B, kThreads) + zeros_before(m + 1) - zeros_before(m);
  };
  const int64_t sum_blocks = a.N * a.sum_blocks + units - zeros_before(p.merges);
  const int64_t joins = (p.chunks - 1) * p.slices;
  // Before the first launch: a call that cannot end must not begin.
  int64_t most = std::max(sum_blocks, joins);
  for (int m = 0; m < p.merges; ++m) most = std::max(most, merge_blocks(m));
  if (most > kMaxBlocks) return kInvalid;

  a.list_stride = p.lists == 1 ? 0 : a.B;
  // A list: all tokens, then all positions.
  auto* from = reinterpret_cast<int32_t*>(ws + p.list0);
  auto* to = reinterpret_cast<int32_t*>(ws + p.list1);
  const int64_t half = p.lists * a.B;
  auto* witness = reinterpret_cast<int32_t*>(ws + p.witness);
  const int bits = bits_of(a.V);
  const int passes = (bits + kDigitLog2 - 1) / kDigitLog2;
  const SortArgs sort{tokens, from, from + half, witness, a.B, a.V, bits,
                      passes > 0 ? (bits + passes - 1) / passes : 1};
  const dim3 tiles(static_cast<uint32_t>(p.tiles), static_cast<uint32_t>(p.lists));
  // A digit has a thread, so kDigits of them at least.
  const int64_t words = int64_t(1) << (p.tile_log2 - kSortThreadsLog2);
  const dim3 sorters(static_cast<uint32_t>(std::max<int64_t>(
      kDigits,
      std::min<int64_t>(kSortThreads, ceil_div(ceil_div(a.B, words), kWave) * kWave))));
  const auto sorts = [&](auto word, auto words_log2) {
    hipLaunchKernelGGL((sort_kernel<decltype(word), decltype(words_log2)::value>), tiles, sorters,
                       0, stream, sort);
  };
  const bool narrow = bits + p.tile_log2 <= 32;
  switch (p.tile_log2 - kSortThreadsLog2) {
    case 0:
      if (narrow) {
        sorts(uint32_t{}, std::integral_constant<int, 0>{});
      } else {
        sorts(uint64_t{}, std::integral_constant<int, 0>{});
      }
      break;
    case 3:  // 32 bits: where 64 are needed the tile would not fit in LDS
      sorts(uint32_t{}, std::integral_constant<int, 3>{});
      break;
    default:
      if (narrow) {
        sorts(uint32_t{}, std::integral_constant<int, 2>{});
      } else {
        sorts(uint64_t{}, std::integral_constant<int, 2>{});
      }
  }
  if (const int err = launched()) return err;

  ZeroArgs zero{};
  zero.weight_grad = a.weight_grad;
  zero.tokens = tokens;
  zero.witness = witness;
  zero.witness_stride = p.lists == 1 ? 0 : a.V;
  zero.B = a.B;
  zero.V = a.V;
  zero.D = a.D;
  zero.units = zero_units;
  int64_t runs = p.tiles;
  for (int m = 0; m < p.merges; ++m, runs = ceil_div(runs, kFan)) {
    const MergeArgs merge{from, from + half, to, to + half, p.lists, a.B,
                          p.tile_log2 + m * kFanLog2};
    zero.first = zeros_before(m);
    zero.end = zeros_before(m + 1);
    const dim3 grid(static_cast<uint32_t>(merge_blocks(m))), block(kThreads);
    if (runs <= 4) {
      hipLaunchKernelGGL((merge_kernel<T, G, NARROW, 4>), grid, block, 0, stream, merge, zero);
    } else if (runs <= 8) {
      hipLaunchKernelGGL((merge_kernel<T, G, NARROW, 8>), grid, block, 0, stream, merge, zero);
    } else {
      hipLaunchKernelGGL((merge_kernel<T, G, NARROW, kFan>), grid, block, 0, stream, merge,
                         zero);
    }
    if (const int err = launched()) return err;
    std::swap(from, to);
  }
  zero.first = zeros_before(p.merges);
  zero.end = units;
  a.token = from;
  a.position = from + half;
  a.parts = reinterpret_cast<float*>(ws + p.parts);
  hipLaunchKernelGGL((sum_kernel<T, G, NARROW>), dim3(static_cast<uint32_t>(sum_blocks)),
                     dim3(kThreads), 0, stream, a, zero);
  if (const int err = launched()) return err;
  if (p.chunks > 1) {
    hipLaunchKernelGGL((join_kernel<T, G, NARROW>),
                       dim3(static_cast<uint32_t>(joins), static_cast<uint32_t>(a.N)),
                       dim3(kThreads), 0, stream, a);
  }
  return launched();
}

int64_t width_of(ts_dtype dtype) { return dtype == TS_FLOAT32 ? 4 : 2; }

bool dtype_ok(ts_dtype dtype) {
  return dtype == TS_FLOAT32 || dtype == TS_FLOAT16 || dtype == TS_BFLOAT16;
}

}  // namespace
}  // namespace lm
}  // namespace churten

using namespace churten::lm;

extern "C" {

int ts_embedding(ts_rows weight, ts_index tokens, ts_rows out, ts_dtype dtype, int64_t N,
                 int64_t B, int64_t V, int64_t D, float scale, void* stream) {
  if (!sizes_ok(N, B, V, D) || !dtype_ok(dtype)) return kInvalid;
  if (N == 0 || B == 0 || D == 0) return 0;
  if (!index_ok(tokens) || out.data == nullptr || (V > 0 && weight.data == nullptr)) {
    return kInvalid;
  }
  const LookupArgs a{weight, out, tokens, B, V, D, scale};
  const auto s = static_cast<hipStream_t>(stream);
  return by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    const int64_t packs = ceil_div(D, kPack<T>);
    if (D < kPack<T>) return launch_lookup<T, 4, 1, true>(a, N, s);
    const bool many = N * B * packs >= int64_t(1) << 19;
    const auto launch = [&](auto g) {
      constexpr int G = decltype(g)::value;
      return many ? launch_lookup<T, G, kLookupRows, false>(a, N, s)
                  : launch_lookup<T, G, 1, false>(a, N, s);
    };
    // Rows of several wavefronts: all of a row by one workgroup at a time.
    if (packs > 2 * kWave) return launch(std::integral_constant<int, 4 * kWave>{});
    if (packs > kWave) return launch(std::integral_constant<int, 2 * kWave>{});
    return by_lanes(static_cast<int>(packs), launch);
  });
}

size_t ts_embedding_grad_workspace(ts_dtype dtype, int64_t N, int64_t B, int64_t V, int64_t D,
                                   int shared_tokens) {
  if (!sizes_ok(N, B, V, D) || !dtype_ok(dtype) || N == 0 || V == 0 || D == 0) return 0;
  return plan_of(width_of(dtype), N, B, V, D, shared_tokens != 0).bytes;
}

int ts_embedding_grad(ts_rows weight_grad, ts_rows grad, ts_index tokens, ts_dtype dtype,
                      int64_t N, int64_t B, int64_t V, int64_t D, float scale, uint32_t flags,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (!sizes_ok(N, B, V, D) || !dtype_ok(dtype) || (flags & ~TS_ACCUMULATE) != 0) {
    return kInvalid;
  }
  if (N == 0 || V == 0 || D == 0) return 0;
  const bool accumulate = (flags & TS_ACCUMULATE) != 0;
  if (accumulate && B == 0) return 0;
  if (weight_grad.data == nullptr ||
      (B > 0 && (grad.data == nullptr || !index_ok(tokens)))) {
    return kInvalid;
  }
  const GradPlan p = plan_of(width_of(dtype), N, B, V, D, tokens.stride_n == 0);
  if (p.bytes > 0 && (workspace == nullptr || workspace_bytes < p.bytes ||
                      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
    return kInvalid;
  }
  SumArgs a{};
  a.weight_grad = weight_grad;
  a.grad = grad;
  a.N = N;
  a.B = B;
  a.V = V;
  a.D = D;
  a.scale = scale;
  a.accumulate = accumulate;
  const DirectArgs few{weight_grad, grad, tokens, B, V, D, 1, scale, accumulate};
  const auto s = static_cast<hipStream_t>(stream);
  auto* ws = static_cast<char*>(workspace);
  return by_dtype(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    return by_lanes(p.lanes, [&](auto lanes) {
      constexpr int G = decltype(lanes)::value;
      if (D < kPack<T>) {
        return p.direct ? launch_direct<T, 4, true>(few, N, s)
                        : launch_sorted<T, 4, true>(p, a, tokens, ws, s);
      }
      return p.direct ? launch_direct<T, G, false>(few, N, s)
                      : launch_sorted<T, G, false>(p, a, tokens, ws, s);
    });
  });
}

}  // extern "C"
