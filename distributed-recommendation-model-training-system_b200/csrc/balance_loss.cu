// balance_loss.cu -- a loss that balances the experts, each expert's count, and the
// logits' gradient (eps_b200_balance_loss, eps_b200_balance_loss_backward).
//
// Mathematics (n counted tokens, k entries each, E experts):
//   p = softmax(l), or s = sigmoid(l) divided by its sum or not
//   counts[e] = entries that are e,  mass[e] = sum_t p[t, e]
//   loss = w E / (k n^2) sum_e counts[e] mass[e]
// The counts take no gradient, so with d[e] = dloss w E / (k n^2) counts[e]
//   softmax:              dl = p (d - sum_e p d)
//   sigmoid, normalised:  dl = s (1 - s) (d - sum_e p d) / sum_e s
//   sigmoid:              dl = s (1 - s) d
// Where p adds up to one a constant may be taken from d without changing the result:
// the mean count goes, so that what is left of nearly equal counts keeps its bits.
//
// Bound: one read of the logits (backward: of the logits and `add`, one write), and one
// exponential an element.  The lanes of a row hold it in registers between its reductions
// while the next rows are copied to shared memory (cp.async), each pack by the lane that
// reads it back; each lane sums its columns over all of its rows.  Blocks leave their sums,
// which a cluster adds up in block order: no float atomics, so results repeat exactly.
//   At these sizes a pass is as long as its chain: launch, first rows (1.5 us), rows (a turn
// of two waits for some 20 dependent steps), the block's sums, and the second launch (4 us).
// 32771 x 256 floats, sigmoid: 16.5 us; 131071 x 96 bf16, half of it padding: 19.7; backward
// of 65521 x 256 bf16 with `add`, half of it padding: 21.9, 59 % of the copy rate for the 84
// MB that it moves (a plain sum of two tensors of that size takes 16.7).  Before rows were
// copied ahead, with twice the instructions a column: 30.3, 37.5 and 25.9.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

// One block an SM, as many threads as the columns of a lane leave registers for.
template <int COLUMNS> constexpr unsigned kThreadsFor = COLUMNS <= 8 ? 1024 : COLUMNS <= 16 ? 512 : 256;
constexpr unsigned kMost = 1024;          // most blocks
constexpr unsigned kFinish = 8, kFinishThreads = 512, kFinishWarps = kFinishThreads / 32;      // blocks that add their sums up

// Rows that a lane copies ahead, of the forward pass and, from two tensors, of the backward
// pass.  Single 16-bit values cannot be copied to shared memory on their own: of those one
// row waits in registers.
template <int BYTES> constexpr unsigned kAheadOf = BYTES == 2 ? 1 : 4;
template <class T, int BYTES> constexpr unsigned kAheadBack = BYTES == 2 ? 1 : sizeof(T) == 4 ? 3 : 4;
struct Rows {
  const void* logits;
  int64_t stride;
  const uint8_t* mask;
  uint32_t tokens, experts, top_k;
  unsigned width;            // lanes of a row
  bool normalise;
  float weight;
};

struct Forward : Rows {
  const int32_t* chosen;
  float* loss;
  int32_t* counts;
  float* mass;
  int32_t* counted;
  uint32_t* sums;            // a block's mass, counts and counted tokens: 2 E + 1 words
};

struct Backward : Rows {
  const int32_t* counts;
  const int32_t* counted;
  const float* dloss;
  const void* add;
  int64_t add_stride;
  void* out;
  int64_t out_stride;
};

// The larger and the smaller of two values; NaN if one is.
__device__ __forceinline__ float most(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float least(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// e^x of N values up to 88.72.  The power of two takes x log2 e rounded to a float, off by
// |x| / 2 units; float logits add back what that lost, x less that power's logarithm.
template <int N, bool FINE>
__device__ __forceinline__ void powers(float (&x)[N]) {
  constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
  if constexpr (FINE) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = most(x[i], -200.f);      // below it is 0 anyway, and an infinity has no rest
  }
  float t[N];
  vmul<N>(t, x, kLog2e);
  if constexpr (FINE) vfma<N>(x, t, -kLn2, x);
#pragma unroll
  for (int i = 0; i < N; ++i) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t[i]));
  if constexpr (FINE) {
    vfma<N>(x, t, x, t);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = t[i];
  }
}

__device__ __forceinline__ float inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / total, 0 where that is 0.
__device__ __forceinline__ float share(float total) { return total == 0.f ? 0.f : inverse(total); }

// Over the lanes of a row, U rows at once.
template <int U>
__device__ __forceinline__ void row_add(float (&v)[U], unsigned width) {
  for (unsigned o = width / 2; o; o /= 2)
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(~0u, v[u], o);
}
template <int U>
__device__ __forceinline__ void row_most(float (&v)[U], unsigned width) {
  for (unsigned o = width / 2; o; o /= 2)
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = fmaxf(v[u], __shfl_xor_sync(~0u, v[u], o));
}

// The sum of a lane's values, two halves at a time.
template <int N>
__device__ __forceinline__ float lane_sum(const float (&v)[N]) {
  if constexpr (N == 1) {
    return v[0];
  } else {
    float half[N / 2 + N % 2];
    vadd<N / 2>(reinterpret_cast<float(&)[N / 2]>(half), reinterpret_cast<const float(&)[N / 2]>(v[0]), reinterpret_cast<const float(&)[N / 2]>(v[N / 2]));
    if constexpr (N % 2) half[N / 2] = v[N - 1];
    return lane_sum<N / 2 + N % 2>(half);
  }
}

// A lane's packs of a row, pack j the V columns from (j * width + lane) * V on, copied ahead
// to shared memory, AHEAD rows of them.
template <class T, int V, int J, unsigned THREADS, unsigned AHEAD>
struct Copies {
  static constexpr unsigned kBytes = V * sizeof(T), kRow = J * THREADS * kBytes, kAll = kBytes == 2 ? 16 : AHEAD * kRow;
  Pack<T, V> waiting[kBytes == 2 ? J : 1];
  unsigned at, here;       // the packs of this lane in its row, a bit each
  // What is behind the last column is `rest` once and for all: no copy reaches it.
  __device__ __forceinline__ Copies(void* shared, unsigned first, unsigned width, unsigned columns, float rest)
      : at(shared_at(shared) + threadIdx.x * kBytes), here(0) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_float<T>(rest);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (first + j * width * V < columns) {
        here |= 1u << j;
      } else if constexpr (kBytes == 2) {
        waiting[j] = r;
      } else {
        for (unsigned k = 0; k < AHEAD; ++k) *reinterpret_cast<Pack<T, V>*>(static_cast<char*>(shared) + k * kRow + (j * THREADS + threadIdx.x) * kBytes) = r;
      }
    }
  }
  __device__ __forceinline__ void copy(unsigned turn, const T* row, unsigned width, bool there) {
    const unsigned to = at + turn % AHEAD * kRow;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (!there || !(here >> j & 1)) continue;
      if constexpr (kBytes == 2) waiting[j] = load_pack<T, V>(row + j * width * V);
      else copy_ahead<(int)kBytes>(to + j * THREADS * kBytes, row + j * width * V, true);
    }
  }
  __device__ __forceinline__ void read(unsigned turn, float (&v)[J * V]) const {
    const unsigned from = at + turn % AHEAD * kRow;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float(&to)[V] = *reinterpret_cast<float(*)[V]>(v + j * V);
      if constexpr (kBytes == 2) widen(waiting[j], to);
      else widen(own_shared<Pack<T, V>>(from + j * THREADS * kBytes), to);
    }
  }
};

// What the scores of sigmoids are divided by, so that the reciprocal keeps them normal floats
// as far down as a float can tell them from 0: e^-x passes 2^127.99 at -88.716, behind which
// they are 0 (the router's are behind 2^128).  It costs no instruction.
constexpr float kUnit = 0.2518f, kLeast = 88.72f;      // kUnit e^kLeast is above 2^126, e^kLeast below 2^128

// The scores of U rows of logits, -inf behind their last columns: their unnormalised p and,
// for sigmoids, 1 - s in rest, both over kUnit.
template <class T, int U, int N, bool SIGMOID>
__device__ __forceinline__ void scores(float (&v)[U][N], float (&rest)[U][SIGMOID ? N : 1], unsigned width) {
  constexpr bool kFine = std::is_same_v<T, float>;
  if constexpr (SIGMOID) {
    // s = 1 / (1 + e), 1 - s = e s with e = e^-x; s is 0 from -kLeast down
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = least(-v[u][i], kLeast);
      powers<N, kFine>(e);
      vfma<N>(v[u], e, +kUnit, +kUnit);
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] = inverse(v[u][i]);
      vmul<N>(rest[u], e, v[u]);
    }
  } else {
    float top[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      top[u] = v[u][0];
#pragma unroll
      for (int i = 1; i < N; ++i) top[u] = fmaxf(top[u], v[u][i]);
    }
    row_most<U>(top, width);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vadd<N>(v[u], v[u], top[u] == -INFINITY ? 0.f : -top[u]);       // a row of -inf alone gives zeros, not NaN
      powers<N, kFine>(v[u]);
    }
  }
}

// The loss of the joint sums.
__device__ __forceinline__ float loss_of(double dot, double n, const Rows& r) {
  return n == 0 ? 0.f : (float)(r.weight * (double)r.experts / (r.top_k * n * n) * dot);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Sums of a block's run of tokens, [tokens * b / blocks, tokens * (b + 1) / blocks); one
// block alone finishes by itself.
template <class T, int V, int J, bool SIGMOID>
__global__ void __launch_bounds__(kThreadsFor<J * V>, 1) balance_forward(Forward f) {
  constexpr unsigned kThreads = kThreadsFor<J * V>;         // at most
  const unsigned threads = blockDim.x, warps = threads / 32;
  constexpr unsigned kAhead = kAheadOf<V * sizeof(T)>;
  extern __shared__ __align__(16) uint32_t shared[];
  using C = Copies<T, V, J, kThreads, kAhead>;
  const unsigned E = f.experts, lane = threadIdx.x % 32, warp = threadIdx.x / 32, width = f.width, first = lane % width * V;
  C copies(shared, first, width, E, -INFINITY);
  float* const mass = reinterpret_cast<float*>(shared + C::kAll / 4);       // [warps][E]
  double* const total = reinterpret_cast<double*>(shared + C::kAll / 4 + (warps * E + 1) / 2 * 2);      // [E]
  uint32_t* const counts = reinterpret_cast<uint32_t*>(total + E);          // [E], and the counted tokens behind them
  asm volatile("griddepcontrol.launch_dependents;");
  const unsigned begin = (uint64_t)f.tokens * blockIdx.x / gridDim.x, end = (uint64_t)f.tokens * (blockIdx.x + 1) / gridDim.x;
  // this lane's rows: `row` is the next to be copied, `there` has a bit for each that is under way
  const unsigned step = warps * (32 / width);
  unsigned row = begin + warp * (32 / width) + lane / width, there = 0;
  const T* from = static_cast<const T*>(f.logits) + (int64_t)row * f.stride + first;
  const int64_t jump = (int64_t)step * f.stride;
  auto mask_of = [&](unsigned r) { return f.mask && r < end ? f.mask[r] : (uint8_t)1; };
  uint8_t mask = mask_of(row);             // asked for a turn before it decides on a copy
  auto copy = [&](unsigned turn) {
    const bool counts = row < end && mask;
    mask = mask_of(row + step);
    copies.copy(turn, from, width, counts);
    copies_end();
    there = there >> 1 | (unsigned)counts << (kAhead - 1);
    row += step;
    from += jump;
  };
#pragma unroll
  for (unsigned i = 0; i < kAhead; ++i) copy(i);
  for (unsigned i = threadIdx.x; i <= E; i += threads) counts[i] = 0;
  __syncthreads();
  // entries and counted tokens; eight entries a thread are asked for at once
  constexpr unsigned kMany = 8;
  for (unsigned i = begin * f.top_k + threadIdx.x; i < end * f.top_k; i += threads * kMany) {
    unsigned e[kMany];
#pragma unroll
    for (unsigned j = 0; j < kMany; ++j) {
      const unsigned k = i + j * threads;
      const bool entry = k < end * f.top_k;
      e[j] = entry ? (unsigned)f.chosen[k] : ~0u;
      if (f.mask && entry && !f.mask[k / f.top_k]) e[j] = ~0u;
    }
#pragma unroll
    for (unsigned j = 0; j < kMany; ++j)
      if (e[j] < E) atomicAdd(&counts[e[j]], 1u);
  }
  if (f.mask) {
    unsigned n = 0;
    for (unsigned t = begin + threadIdx.x; t < end; t += threads) n += f.mask[t] != 0;
    n = __reduce_add_sync(~0u, n);
    if (lane == 0) atomicAdd(&counts[E], n);
  } else if (threadIdx.x == 0) {
    counts[E] = end - begin;
  }
  // mass, two rows a turn, whose chains of reductions run beside each other.  Up to kRun rows of
  // a lane are added in float, over the block too; where it has more, such runs go on in double,
  // so that sums are as exact for many tokens as for few: equal rows are off by kRun / 2 units
  // of 2^-24 and some (a run ends with the block's join: 3e6 x 256 floats 465 us, 2e6 x 1000 bf16
  // 1167 where one run of all rows takes 1110; runs of 32 take 1253)
  constexpr int U = kAhead > 1 ? 2 : 1;
  constexpr unsigned kRun = 64;
  float sum[J * V] = {};
  bool before = false;                     // a run is in total already
  for (unsigned turn = 0, left = end - begin;; left -= kRun * step) {
    const unsigned until = end + kAhead * step - (left > kRun * step ? left - kRun * step : 0);      // what `row` is behind the run
    for (; __any_sync(~0u, row < until); turn += U) {
      bool now[U];
      float v[U][J * V], rest[U][SIGMOID ? J * V : 1], by[U];
      copies_wait<kAhead - U>();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        now[u] = there >> u & 1;
        copies.read(turn + u, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) copy(turn + kAhead + u);
      if (!__any_sync(~0u, now[0] || now[U - 1])) continue;
      scores<T, U, J * V, SIGMOID>(v, rest, width);
      if (!SIGMOID || f.normalise) {
#pragma unroll
        for (int u = 0; u < U; ++u) by[u] = lane_sum<J * V>(v[u]);
        row_add<U>(by, width);
#pragma unroll
        for (int u = 0; u < U; ++u) by[u] = share(by[u]);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) by[u] = kUnit;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (now[u]) vfma<J * V>(sum, v[u], by[u], sum);       // the others' packs hold what was there before
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const unsigned c = first + j * width * V;
      Pack<float, V> s;                    // as a row's, it begins on its size and is all there or not
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s.v[i] = sum[j * V + i];
        for (unsigned o = width; o < 32; o *= 2) s.v[i] += __shfl_xor_sync(~0u, s.v[i], o);
      }
      if (lane < width && c < E) store_pack<float, V>(mass + warp * E + c, s);
    }
    __syncthreads();
    if (left <= kRun * step) break;
    for (unsigned e = threadIdx.x; e < E; e += threads) {
      double all = before ? total[e] : 0;
#pragma unroll 8
      for (unsigned w = 0; w < warps; ++w) all += (double)mass[w * E + e];
      total[e] = all;
    }
    before = true;
#pragma unroll
    for (int i = 0; i < J * V; ++i) sum[i] = 0.f;
    __syncthreads();                       // the next run writes over mass
  }
  if (gridDim.x > 1) {
    uint32_t* const mine = f.sums + (size_t)blockIdx.x * (2 * E + 1);
    for (unsigned e = threadIdx.x; e < E; e += threads) {
      float s = 0.f;
#pragma unroll 8
      for (unsigned w = 0; w < warps; ++w) s += mass[w * E + e];
      if (before) s = (float)(total[e] + s);
      mine[e] = __float_as_uint(s);
      mine[E + e] = counts[e];
    }
    if (threadIdx.x == 0) mine[2 * E] = counts[E];
    return;
  }
  double dot = 0;
  for (unsigned e = threadIdx.x; e < E; e += threads) {
    double s = before ? total[e] : 0;
#pragma unroll 8
    for (unsigned w = 0; w < warps; ++w) s += (double)mass[w * E + e];
    f.mass[e] = (float)s;
    f.counts[e] = (int32_t)counts[e];
    dot += s * counts[e];
  }
  __shared__ double each[32];
  dot = warp_sum(dot);
  if (lane == 0) each[warp] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    dot = 0;
    for (unsigned w = 0; w < warps; ++w) dot += each[w];
    *f.counted = (int32_t)counts[E];
    *f.loss = loss_of(dot, counts[E], f);
  }
}

// Adds the blocks' sums up, one cluster: each of its blocks takes some experts, 32 lanes
// a run of them, its warps the sums in turn.
__global__ void __cluster_dims__(kFinish) __launch_bounds__(kFinishThreads) balance_finish(Forward f, unsigned sums) {
  __shared__ double mass[kFinishWarps][32];
  __shared__ uint32_t counts[kFinishWarps][32];
  __shared__ uint32_t tokens[kFinishWarps];
  __shared__ double mine;
  const unsigned E = f.experts, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double dot = 0;
  for (unsigned e0 = blockIdx.x * 32; e0 < E; e0 += kFinish * 32) {
    const unsigned e = e0 + lane;
    double m = 0;
    uint32_t n = 0;
    if (e < E)
#pragma unroll 10
      for (unsigned b = warp; b < sums; b += kFinishWarps) {
        m += (double)__uint_as_float(f.sums[(size_t)b * (2 * E + 1) + e]);
        n += f.sums[(size_t)b * (2 * E + 1) + E + e];
      }
    mass[warp][lane] = m;
    counts[warp][lane] = n;
    __syncthreads();
    if (warp == 0 && e < E) {
      m = 0;
      n = 0;
      for (unsigned w = 0; w < kFinishWarps; ++w) {
        m += mass[w][lane];
        n += counts[w][lane];
      }
      f.mass[e] = (float)m;
      f.counts[e] = (int32_t)n;
      dot += m * n;
    }
    __syncthreads();
  }
  uint32_t n = 0;
  if (blockIdx.x == 0) {
    for (unsigned b = threadIdx.x; b < sums; b += kFinishThreads) n += f.sums[(size_t)b * (2 * E + 1) + 2 * E];
    n = __reduce_add_sync(~0u, n);
    if (lane == 0) tokens[warp] = n;
  }
  if (warp == 0) {
    dot = warp_sum(dot);
    if (lane == 0) mine = dot;
  }
  cluster_sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    dot = 0;
    for (unsigned r = 0; r < kFinish; ++r) dot += cluster_load(&mine, r);
    n = 0;
    for (unsigned w = 0; w < kFinishWarps; ++w) n += tokens[w];
    *f.counted = (int32_t)n;
    *f.loss = loss_of(dot, n, f);
  }
  cluster_sync();                        // no block leaves while the first reads from it
}

template <class T, int V, int J, bool SIGMOID>
__global__ void __launch_bounds__(kThreadsFor<J * V>, 1) balance_backward(Backward b) {
  constexpr unsigned kThreads = kThreadsFor<J * V>;         // at most
  const unsigned warps = blockDim.x / 32;
  extern __shared__ __align__(16) uint32_t shared[];
  constexpr unsigned kAhead = kAheadBack<T, V * sizeof(T)>;
  using C = Copies<T, V, J, kThreads, kAhead>;
  const unsigned E = b.experts, lane = threadIdx.x % 32, width = b.width, first = lane % width * V;
  const bool shares = !SIGMOID || b.normalise, plus = b.add != nullptr;
  C copies(shared, first, width, E, -INFINITY), extra(plus ? shared + C::kAll / 4 : shared, first, width, plus ? E : ~0u, 0.f);
  // this lane's rows: `row` is the next to be copied, `there` has a bit for each that is under way
  const uint64_t step = (uint64_t)gridDim.x * warps * (32 / width);
  const uint64_t own = (threadIdx.x / 32 * gridDim.x + blockIdx.x) * (32 / width) + lane / width;
  uint64_t row = own;
  unsigned there = 0;
  const T* from = static_cast<const T*>(b.logits) + (int64_t)own * b.stride + first;
  const T* from_add = static_cast<const T*>(b.add) + (int64_t)own * b.add_stride + first;
  T* out = static_cast<T*>(b.out) + (int64_t)own * b.out_stride + first;
  auto mask_of = [&](uint64_t r) { return b.mask && r < b.tokens ? b.mask[r] : (uint8_t)1; };
  uint8_t mask = mask_of(row);             // asked for a turn before it decides on a copy
  auto copy = [&](unsigned turn) {
    const bool counts = row < b.tokens && mask;
    mask = mask_of(row + step);
    copies.copy(turn, from, width, counts);
    if (plus) extra.copy(turn, from_add, width, row < b.tokens);
    copies_end();
    there = there >> 1 | (unsigned)counts << (kAhead - 1);
    row += step;
    from += (int64_t)step * b.stride;
    from_add += (int64_t)step * b.add_stride;
  };
#pragma unroll
  for (unsigned i = 0; i < kAhead; ++i) copy(i);
  // a column's d, less what the mean count gives
  float d[J * V];
  {
    const double n = *b.counted, k = b.top_k;
    const double c = n == 0 ? 0.0 : (b.dloss ? (double)*b.dloss : 1.0) * b.weight * E / (k * n * n);
    const double mean = shares ? k * n / E : 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const unsigned e = first + j * width * V + i;
        d[j * V + i] = e < E ? (float)(c * (b.counts[e] - mean)) : 0.f;
      }
  }
  const uint64_t last = b.tokens + kAhead * step;      // what `row` is behind the last
  for (unsigned turn = 0; __any_sync(~0u, row < last); ++turn) {
    const bool now = there & 1, mine = row < last;
    float score[1][J * V], g[J * V], rest[1][SIGMOID ? J * V : 1];
    float(&v)[J * V] = score[0];
    copies_wait<kAhead - 1>();
    copies.read(turn, v);
    if (plus) {
      extra.read(turn, g);
    } else {
#pragma unroll
      for (int i = 0; i < J * V; ++i) g[i] = 0.f;
    }
    copy(turn + kAhead);
    if (__any_sync(~0u, now)) {
      scores<T, 1, J * V, SIGMOID>(score, rest, width);
      float by = kUnit, dot = 0.f, slope[J * V];
      if (shares) {
        vmul<J * V>(slope, v, d);
        float both[2] = {lane_sum<J * V>(v), lane_sum<J * V>(slope)};
        row_add<2>(both, width);
        by = share(both[0]);
        dot = both[1] * by;
      }
      if (now) {
        if constexpr (SIGMOID) by *= kUnit;      // of rest
        vadd<J * V>(slope, d, -dot);
        vmul<J * V>(v, v, by);
        if constexpr (SIGMOID) vmul<J * V>(v, v, rest[0]);
        vfma<J * V>(g, v, slope, g);
      }
    }
    if (mine) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (copies.here >> j & 1) store_pack<T, V>(out + j * width * V, narrow<T, V>(*reinterpret_cast<const float(*)[V]>(g + j * V)));
    }
    out += (int64_t)step * b.out_stride;
  }
}

// The variants: packs of 16 bytes where every row begins on 16 bytes and ends with a pack,
// of 4 where that holds for 4, single elements else.  Of the packs a lane may have, those that cost a row the
// fewest instructions: some 12 a column of a lane and 100 a turn, for 32 / width rows; but
// four lanes side by side, for 64 bytes in a row (131072 x 16 floats: 12 us against 14).
// More columns than 16 a lane leave few warps and are taken only where a row needs them.
template <class T, int V, class F>
void by_packs(unsigned experts, unsigned* width, F launch) {
  const unsigned packs = (unsigned)ceil_div(experts, V);
  unsigned best = 0, least = ~0u;
  auto ask = [&](unsigned each) {
    unsigned w = 1;
    while (w * each < packs) w *= 2;
    const unsigned cost = w * (12 * each * V + 100);
    if (w <= 32 && w >= std::min(packs, 4u) && (each * V <= 16 || !best) && cost < least) best = each, *width = w, least = cost;
  };
  auto go = [&](auto each) {
    if constexpr (decltype(each)::value * V <= 32)
      if (best == decltype(each)::value) launch(each);
  };
  if constexpr (V == 8) {
    for (unsigned e : {1u, 2u, 4u}) ask(e);
  } else if constexpr (V == 4) {
    for (unsigned e : {1u, 2u, 3u, 4u, 8u}) ask(e);
  } else {
    for (unsigned e : {1u, 2u, 4u, 8u, 16u, 32u})
      if (!best) ask(e);                     // small packs: as many lanes side by side as there are
  }
  go(std::integral_constant<int, 1>{});
  go(std::integral_constant<int, 2>{});
  if constexpr (V == 4) go(std::integral_constant<int, 3>{});
  go(std::integral_constant<int, 4>{});
  if constexpr (V < 8) go(std::integral_constant<int, 8>{});
  if constexpr (V <= 2) go(std::integral_constant<int, 16>{});
  if constexpr (V == 1) go(std::integral_constant<int, 32>{});
}

template <class T, class F>
void by_pack(size_t bytes, F run) {
  if (bytes == 16) run(std::integral_constant<int, 16 / sizeof(T)>{});
  else if (bytes == 4) run(std::integral_constant<int, 4 / sizeof(T)>{});
  else if constexpr (sizeof(T) == 2) run(std::integral_constant<int, 1>{});
}

template <class T>
void forward(Forward f, size_t pack, bool sigmoid, unsigned grid, int device, cudaStream_t stream) {
  auto run = [&](auto v) {
    constexpr int V = decltype(v)::value;
    by_packs<T, V>(f.experts, &f.width, [&](auto j) {
      constexpr int J = decltype(j)::value;
      constexpr unsigned kThreads = kThreadsFor<J * V>;
      // a block alone has as many warps as its tokens need
      const unsigned threads = grid > 1 ? kThreads : std::min<unsigned>(kThreads, std::max<unsigned>(4, (unsigned)ceil_div(f.tokens, 32 / f.width)) * 32);
      const size_t bytes = Copies<T, V, J, kThreads, kAheadOf<V * sizeof(T)>>::kAll + (round_up(threads / 32 * f.experts, 2) + 3 * (size_t)f.experts + 1) * 4;
      auto go = [&](auto s) {
        constexpr bool S = decltype(s)::value;
        room<balance_forward<T, V, J, S>>(device);
        balance_forward<T, V, J, S><<<grid, threads, bytes, stream>>>(f);
      };
      sigmoid ? go(std::true_type{}) : go(std::false_type{});
    });
  };
  by_pack<T>(pack, run);
  check(cudaGetLastError(), "balance_forward");
  if (grid == 1) return;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = kFinish;
  config.blockDim = kFinishThreads;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  check(cudaLaunchKernelEx(&config, balance_finish, f, grid), "balance_finish");
}

template <class T>
void backward(Backward b, size_t pack, bool sigmoid, int device, cudaStream_t stream) {
  auto run = [&](auto v) {
    constexpr int V = decltype(v)::value;
    by_packs<T, V>(b.experts, &b.width, [&](auto j) {
      constexpr int J = decltype(j)::value;
      constexpr unsigned kThreads = kThreadsFor<J * V>;
      const size_t bytes = Copies<T, V, J, kThreads, kAheadBack<T, V * sizeof(T)>>::kAll * (b.add ? 2 : 1);
      const uint64_t turns = ceil_div(b.tokens, 32 / b.width);      // of a warp
      const unsigned grid = (unsigned)std::min<uint64_t>(turns, sm_count(device));
      const unsigned threads = (unsigned)std::min<uint64_t>(kThreads / 32, ceil_div(turns, grid)) * 32;
      auto go = [&](auto s) {
        constexpr bool S = decltype(s)::value;
        room<balance_backward<T, V, J, S>>(device);
        balance_backward<T, V, J, S><<<grid, threads, bytes, stream>>>(b);
      };
      sigmoid ? go(std::true_type{}) : go(std::false_type{});
    });
  };
  by_pack<T>(pack, run);
  check(cudaGetLastError(), "balance_backward");
}

// Blocks of the forward pass: one for a small batch, which then needs no second launch
// (16384 values 6.4 us against 7.3; 32768 7.9 against 7.3), else some 8192 values each (131072
// values 7.8 us; with 2048 each 8.4, with 32768 9.8).
unsigned forward_blocks(uint64_t tokens, uint32_t experts, unsigned sms) {
  const uint64_t values = tokens * experts;
  return values <= 16384 ? 1 : (unsigned)std::min<uint64_t>(ceil_div(values, 8192), std::min(sms, kMost));
}

// The largest packs that every row of these tensors (not NULL) begins on and ends with.
struct Place {
  const void* p;
  int64_t stride;
};
size_t pack_bytes(std::initializer_list<Place> places, uint64_t columns, size_t size) {
  for (size_t n : {(size_t)16, (size_t)4}) {
    bool all = columns * size % n == 0;
    for (const Place& q : places) all = all && (!q.p || (aligned(q.p, n) && q.stride * (int64_t)size % (int64_t)n == 0));
    if (all) return n;
  }
  return size;
}

Rows checked(const EpsB200BalanceLoss* a) {
  need(a, "null balance argument");
  need(known_type(a->type), "unknown element type");
  need(a->score == EPS_B200_SCORE_SOFTMAX || a->score == EPS_B200_SCORE_SIGMOID, "unknown score");
  need(a->experts > 0 && a->experts <= EPS_B200_ROUTE_EXPERTS, "1 to 1024 experts");
  need(a->top_k > 0 && a->top_k <= EPS_B200_ROUTE_TOP_K, "top_k is 1 to 32");
  need(a->tokens < (1ull << 31) && a->tokens * a->top_k < (1ull << 31), "tokens * top_k must be below 2^31");
  need(std::isfinite(a->weight), "the weight must be finite");
  need(a->logits || !a->tokens, "null logits");
  need(aligned(a->logits, size_of(a->type)), "logits are not aligned to their type");
  Rows r{};
  r.logits = a->logits;
  r.stride = a->logits_stride;
  r.mask = a->mask;
  r.tokens = (uint32_t)a->tokens;
  r.experts = a->experts;
  r.top_k = a->top_k;
  r.normalise = a->normalise != 0;
  r.weight = a->weight;
  return r;
}

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_balance_loss_workspace(uint64_t tokens, uint32_t experts) {
  const unsigned blocks = forward_blocks(tokens, experts, kMost);
  return blocks == 1 ? 0 : (uint64_t)blocks * (2 * (uint64_t)experts + 1) * 4;
}

int eps_b200_balance_loss(const EpsB200BalanceLoss* a, const int32_t* chosen, float* loss, int32_t* counts, float* mass, int32_t* counted,
                          void* workspace, uint64_t workspace_bytes, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Forward f{};
    static_cast<Rows&>(f) = checked(a);
    need(loss && counts && mass && counted, "null balance output");
    need(chosen || !a->tokens, "null chosen experts");
    need(words(chosen, loss, counts, mass, counted), "experts and outputs are 4-byte aligned");
    const uint64_t space = eps_b200_balance_loss_workspace(a->tokens, a->experts);
    need(!space || (workspace && aligned(workspace, 4) && workspace_bytes >= space), "the balance loss's workspace is too small");
    f.chosen = chosen;
    f.loss = loss;
    f.counts = counts;
    f.mass = mass;
    f.counted = counted;
    f.sums = static_cast<uint32_t*>(workspace);
    OnDevice on(a->device);
    const size_t size = size_of(a->type);
    const size_t pack = pack_bytes({{a->logits, a->logits_stride}}, a->experts, size);
    const unsigned grid = forward_blocks(a->tokens, a->experts, sm_count(a->device));
    const auto s = static_cast<cudaStream_t>(stream);
    const bool sigmoid = a->score == EPS_B200_SCORE_SIGMOID;
    if (a->type == EPS_B200_F32) forward<float>(f, pack, sigmoid, grid, a->device, s);
    else if (a->type == EPS_B200_BF16) forward<bf16>(f, pack, sigmoid, grid, a->device, s);
    else forward<f16>(f, pack, sigmoid, grid, a->device, s);
  });
}

int eps_b200_balance_loss_backward(const EpsB200BalanceLoss* a, const int32_t* counts, const int32_t* counted, const float* dloss,
                                   const void* add, int64_t add_stride, void* dlogits, int64_t dlogits_stride, void* stream,
                                   EpsB200Status* status) {
  return guard(status, [&] {
    Backward b{};
    static_cast<Rows&>(b) = checked(a);
    need(counts && counted, "null counts");
    need(dlogits || !a->tokens, "null dlogits");
    need(words(counts, counted, dloss), "counts and dloss are 4-byte aligned");
    need(aligned(add, size_of(a->type)) && aligned(dlogits, size_of(a->type)), "a gradient is not aligned to its type");
    if (!a->tokens) return;
    b.counts = counts;
    b.counted = counted;
    b.dloss = dloss;
    b.add = add;
    b.add_stride = add_stride;
    b.out = dlogits;
    b.out_stride = dlogits_stride;
    // A lane reads its packs of a row before it writes them: what lies at the same place may be the same
    // tensor.  Elsewhere a row would be written before another lane has read it.
    const size_t size = size_of(a->type);
    const Matrix to{dlogits, dlogits_stride, a->experts};
    need(a->tokens == 1 || dlogits_stride >= (int64_t)a->experts || dlogits_stride <= -(int64_t)a->experts, "rows of dlogits overlap");
    auto apart = [&](const void* p, int64_t stride) {
      return !p || (p == dlogits && (a->tokens == 1 || stride == dlogits_stride)) || !overlap(to, {p, stride, a->experts}, a->tokens, size);
    };
    need(apart(a->logits, a->logits_stride), "dlogits overlaps logits without being it");
    need(apart(add, add_stride), "dlogits overlaps add without being it");
    OnDevice on(a->device);
    const size_t pack = pack_bytes({{a->logits, a->logits_stride}, {dlogits, dlogits_stride}, {add, add_stride}}, a->experts, size);
    const auto s = static_cast<cudaStream_t>(stream);
    const bool sigmoid = a->score == EPS_B200_SCORE_SIGMOID;
    if (a->type == EPS_B200_F32) backward<float>(b, pack, sigmoid, a->device, s);
    else if (a->type == EPS_B200_BF16) backward<bf16>(b, pack, sigmoid, a->device, s);
    else backward<f16>(b, pack, sigmoid, a->device, s);
  });
}

}  // extern "C"
