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
// exponential an element.  The lanes of a row (the fewest, a power of two, whose packs
// cover it) hold it in registers between its reductions and the next row is under way
// meanwhile; each lane sums its columns over all of its rows.  Blocks leave their sums,
// which a cluster adds up in block order: no float atomics, so results repeat exactly.
#include <algorithm>
#include <cmath>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

constexpr unsigned kThreads = 256, kWarps = kThreads / 32;
// Blocks an SM, by the columns of a lane: what their registers leave room for.
constexpr unsigned blocks_an_sm(int columns) { return columns <= 8 ? 4 : columns <= 16 ? 2 : 1; }
constexpr unsigned kTogether = 4;         // blocks whose sums are added before they leave them
constexpr unsigned kMost = 1024;          // most blocks
constexpr unsigned kFinish = 8, kFinishThreads = 512, kFinishWarps = kFinishThreads / 32;      // blocks that add up what is left

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
  uint32_t* sums;            // a cluster's mass, counts and counted tokens: 2 E + 1 words
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

// e^x for x <= 88; 0 below -200, and NaN stays.  The power of two takes x log2 e rounded
// to a float, off by |x| / 2 units; float logits add back what that lost (the product's
// error by a fused multiply-add, and the rest of log2 e).
template <bool FINE>
__device__ __forceinline__ float power(float x) {
  constexpr float kLog2e = 1.44269502f, kRest = 1.92596303e-8f, kLn2 = 0.693147182f;   // log2 e in two parts; ln 2
  x = x < -200.f ? -200.f : x;
  const float t = x * kLog2e;
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  if constexpr (FINE) r = fmaf(r, fmaf(x, kRest, fmaf(x, kLog2e, -t)) * kLn2, r);
  return r;
}

__device__ __forceinline__ float inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / total, 0 where that is 0.
__device__ __forceinline__ float share(float total) { return total == 0.f ? 0.f : inverse(total); }

__device__ __forceinline__ float row_add(float v, unsigned width) {
  for (unsigned o = width / 2; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// A lane's packs of a row: pack j covers the V columns from (j * width + lane) * V on.
template <class T, int V, int J>
struct Held {
  Pack<T, V> p[J];
  __device__ __forceinline__ void load(const T* row, unsigned first, unsigned width, unsigned columns, bool there) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const unsigned c = first + j * width * V;
      if (there && c < columns) p[j] = load_once<T, V>(row + c);
    }
  }
};

// The scores of a row: its unnormalised p in v and, for sigmoids, 1 - s in rest.  What is
// behind the last column, or in a row that is not there, is 0.
template <class T, int V, int J, bool SIGMOID>
__device__ __forceinline__ void scores(const Held<T, V, J>& h, unsigned first, unsigned width, unsigned columns, bool there, float (&v)[J * V],
                                       float (&rest)[SIGMOID ? J * V : 1]) {
  constexpr bool kFine = std::is_same_v<T, float>;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (there && first + j * width * V < columns) {
      widen(h.p[j], *reinterpret_cast<float(*)[V]>(v + j * V));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j * V + i] = -INFINITY;
    }
  }
  if constexpr (SIGMOID) {
#pragma unroll
    for (int i = 0; i < J * V; ++i) {
      const bool low = v[i] < -87.f;          // s would leave the normal floats: 0
      const float e = low ? 1.f : power<kFine>(-v[i]);
      const float s = inverse(1.f + e);
      rest[i] = e * s;
      v[i] = low ? 0.f : s;
    }
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < J * V; ++i) top = fmaxf(top, v[i]);
    for (unsigned o = width / 2; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float less = top == -INFINITY ? 0.f : top;       // a row of -inf alone gives zeros, not NaN
#pragma unroll
    for (int i = 0; i < J * V; ++i) v[i] = power<kFine>(v[i] - less);
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

// Sums of a block's run of tokens, [tokens * b / blocks, tokens * (b + 1) / blocks), added
// over a cluster; one block alone finishes by itself.
template <class T, int V, int J, bool SIGMOID>
__global__ void __launch_bounds__(kThreads, blocks_an_sm(J * V)) balance_forward(Forward f) {
  extern __shared__ uint32_t shared[];
  const unsigned E = f.experts, lane = threadIdx.x % 32, warp = threadIdx.x / 32, width = f.width;
  float* const mass = reinterpret_cast<float*>(shared);       // [kWarps][E]
  uint32_t* const counts = shared + kWarps * E;                 // [E], and the counted tokens behind them
  asm volatile("griddepcontrol.launch_dependents;");
  const unsigned begin = (uint64_t)f.tokens * blockIdx.x / gridDim.x, end = (uint64_t)f.tokens * (blockIdx.x + 1) / gridDim.x;
  const unsigned step = kWarps * (32 / width), first = lane % width * V;
  const T* const logits = static_cast<const T*>(f.logits);
  Held<T, V, J> now, next;
  unsigned row = begin + warp * (32 / width) + lane / width;
  bool there = row < end && (!f.mask || f.mask[row]);
  now.load(logits + (int64_t)row * f.stride, first, width, E, there);
  for (unsigned i = threadIdx.x; i <= E; i += kThreads) counts[i] = 0;
  __syncthreads();
  // entries and counted tokens
  for (unsigned i = begin * f.top_k + threadIdx.x; i < end * f.top_k; i += kThreads) {
    const unsigned e = (unsigned)f.chosen[i];
    if (e < E && (!f.mask || f.mask[i / f.top_k])) atomicAdd(&counts[e], 1u);
  }
  if (f.mask) {
    unsigned n = 0;
    for (unsigned t = begin + threadIdx.x; t < end; t += kThreads) n += f.mask[t] != 0;
    n = __reduce_add_sync(~0u, n);
    if (lane == 0) atomicAdd(&counts[E], n);
  } else if (threadIdx.x == 0) {
    counts[E] = end - begin;
  }
  // mass
  float sum[J * V] = {};
  while (__any_sync(~0u, row < end)) {
    const unsigned after = row + step;
    const bool more = after < end && (!f.mask || f.mask[after]);
    next.load(logits + (int64_t)after * f.stride, first, width, E, more);
    float v[J * V], rest[SIGMOID ? J * V : 1];
    scores<T, V, J, SIGMOID>(now, first, width, E, there, v, rest);
    float by = 1.f;
    if (!SIGMOID || f.normalise) {
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < J * V; ++i) total += v[i];
      by = share(row_add(total, width));
    }
#pragma unroll
    for (int i = 0; i < J * V; ++i) sum[i] = fmaf(v[i], by, sum[i]);
    now = next;
    there = more;
    row = after;
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const unsigned c = first + j * width * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = sum[j * V + i];
      for (unsigned o = width; o < 32; o *= 2) s += __shfl_xor_sync(~0u, s, o);
      if (lane < width && c + i < E) mass[warp * E + c + i] = s;
    }
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (unsigned e = threadIdx.x; e < E; e += kThreads) {
      float s = 0.f;
#pragma unroll
      for (unsigned w = 0; w < kWarps; ++w) s += mass[w * E + e];
      mass[e] = s;
    }
    cluster_sync();
    uint32_t* const mine = f.sums + (size_t)(blockIdx.x / kTogether) * (2 * E + 1);
    for (unsigned e = threadIdx.x * kTogether + cluster_rank(); e <= E; e += kThreads * kTogether) {
      float s = 0.f;
      uint32_t n = 0;
#pragma unroll
      for (unsigned r = 0; r < kTogether; ++r) {
        if (e < E) s += cluster_load(mass + e, r);
        n += cluster_load(counts + e, r);
      }
      if (e < E) mine[e] = __float_as_uint(s);
      mine[E + e] = n;
    }
    cluster_sync();                      // no block leaves while another reads from it
    return;
  }
  double dot = 0;
  for (unsigned e = threadIdx.x; e < E; e += kThreads) {
    double s = 0;
#pragma unroll
    for (unsigned w = 0; w < kWarps; ++w) s += (double)mass[w * E + e];
    f.mass[e] = (float)s;
    f.counts[e] = (int32_t)counts[e];
    dot += s * counts[e];
  }
  __shared__ double each[kWarps];
  dot = warp_sum(dot);
  if (lane == 0) each[warp] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    dot = 0;
    for (unsigned w = 0; w < kWarps; ++w) dot += each[w];
    *f.counted = (int32_t)counts[E];
    *f.loss = loss_of(dot, counts[E], f);
  }
}

// Adds the clusters' sums up, one cluster: each of its blocks takes some experts, 32 lanes
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
#pragma unroll 5
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
__global__ void __launch_bounds__(kThreads, blocks_an_sm(J * V)) balance_backward(Backward b) {
  const unsigned E = b.experts, lane = threadIdx.x % 32, width = b.width, first = lane % width * V;
  const bool shares = !SIGMOID || b.normalise;
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
  const unsigned slots = gridDim.x * kWarps * (32 / width);
  const T* const logits = static_cast<const T*>(b.logits);
  const T* const add = static_cast<const T*>(b.add);
  T* const out = static_cast<T*>(b.out);
  Held<T, V, J> now, next, more, also;
  uint64_t row = (uint64_t)(blockIdx.x * kWarps + threadIdx.x / 32) * (32 / width) + lane / width;
  bool there = row < b.tokens && (!b.mask || b.mask[row]);
  now.load(logits + (int64_t)row * b.stride, first, width, E, there);
  if (add) more.load(add + (int64_t)row * b.add_stride, first, width, E, row < b.tokens);
  while (__any_sync(~0u, row < b.tokens)) {
    const uint64_t after = row + slots;
    const bool then = after < b.tokens && (!b.mask || b.mask[after]);
    next.load(logits + (int64_t)after * b.stride, first, width, E, then);
    if (add) also.load(add + (int64_t)after * b.add_stride, first, width, E, after < b.tokens);
    float v[J * V], rest[SIGMOID ? J * V : 1];
    scores<T, V, J, SIGMOID>(now, first, width, E, there, v, rest);
    float by = 1.f, dot = 0.f;
    if (shares) {
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < J * V; ++i) {
        total += v[i];
        dot = fmaf(v[i], d[i], dot);
      }
      by = share(row_add(total, width));
      dot = row_add(dot, width) * by;
    }
    if (row < b.tokens) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const unsigned c = first + j * width * V;
        if (c >= E) continue;
        float g[V], plus[V];
        if (add) {
          widen(more.p[j], plus);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) plus[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int q = j * V + i;
          float p = v[q] * by;
          if constexpr (SIGMOID) p *= rest[q];
          g[i] = there ? fmaf(p, d[q] - dot, plus[i]) : plus[i];
        }
        store_pack<T, V>(out + (int64_t)row * b.out_stride + c, narrow<T, V>(g));
      }
    }
    now = next;
    more = also;
    there = then;
    row = after;
  }
}

// The variants: whole packs of 16 bytes where every row begins on 16 bytes and ends with
// a pack, single elements else; as many packs a lane as the row needs.
template <class T, int V, class F>
void by_packs(unsigned experts, unsigned* width, F launch) {
  const unsigned packs = (unsigned)ceil_div(experts, V);
  *width = 1;
  while (*width < 32 && *width < packs) *width *= 2;
  const unsigned each = (unsigned)ceil_div(packs, *width);
  if (each <= 1) launch(std::integral_constant<int, 1>{});
  else if (each <= 2) launch(std::integral_constant<int, 2>{});
  else if (each <= 4) launch(std::integral_constant<int, 4>{});
  else if constexpr (V <= 4) {
    if (each <= 8) launch(std::integral_constant<int, 8>{});
    else if constexpr (V == 1) {
      if (each <= 16) launch(std::integral_constant<int, 16>{});
      else launch(std::integral_constant<int, 32>{});
    }
  }
}

template <class T>
void forward(Forward f, bool wide, bool sigmoid, unsigned grid, int device, cudaStream_t stream) {
  const size_t bytes = (kWarps * (size_t)f.experts + f.experts + 1) * 4;
  auto run = [&](auto v) {
    constexpr int V = decltype(v)::value;
    by_packs<T, V>(f.experts, &f.width, [&](auto j) {
      constexpr int J = decltype(j)::value;
      auto go = [&](auto s) {
        constexpr bool S = decltype(s)::value;
        room<balance_forward<T, V, J, S>>(device);
        cudaLaunchAttribute together{};
        together.id = cudaLaunchAttributeClusterDimension;
        together.val.clusterDim.x = grid == 1 ? 1 : kTogether;
        together.val.clusterDim.y = together.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = grid;
        config.blockDim = kThreads;
        config.dynamicSmemBytes = bytes;
        config.stream = stream;
        config.attrs = &together;
        config.numAttrs = 1;
        check(cudaLaunchKernelEx(&config, balance_forward<T, V, J, S>, f), "balance_forward");
      };
      sigmoid ? go(std::true_type{}) : go(std::false_type{});
    });
  };
  wide ? run(std::integral_constant<int, 16 / sizeof(T)>{}) : run(std::integral_constant<int, 1>{});
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
  check(cudaLaunchKernelEx(&config, balance_finish, f, grid / kTogether), "balance_finish");
}

template <class T>
void backward(Backward b, bool wide, bool sigmoid, int device, cudaStream_t stream) {
  auto run = [&](auto v) {
    constexpr int V = decltype(v)::value;
    by_packs<T, V>(b.experts, &b.width, [&](auto j) {
      constexpr int J = decltype(j)::value;
      const unsigned rows = kWarps * (32 / b.width);
      const unsigned grid = (unsigned)std::min<uint64_t>(ceil_div(b.tokens, rows), sm_count(device) * blocks_an_sm(J * V));
      if (sigmoid) balance_backward<T, V, J, true><<<grid, kThreads, 0, stream>>>(b);
      else balance_backward<T, V, J, false><<<grid, kThreads, 0, stream>>>(b);
    });
  };
  wide ? run(std::integral_constant<int, 16 / sizeof(T)>{}) : run(std::integral_constant<int, 1>{});
  check(cudaGetLastError(), "balance_backward");
}

// Blocks of the forward pass: some 8192 values each, so that a small batch takes one;
// more come in clusters.
unsigned forward_blocks(uint64_t tokens, uint32_t experts, unsigned sms) {
  const uint64_t n = ceil_div(tokens * experts, 8192);
  return n <= 1 ? 1 : (unsigned)std::min<uint64_t>(round_up(n, kTogether), std::min(sms * 4, kMost) / kTogether * kTogether);
}

bool wide_rows(const void* p, int64_t stride, size_t size) { return aligned(p, 16) && stride * (int64_t)size % 16 == 0; }

Rows checked(const EpsB200BalanceLoss* a) {
  need(a, "null balance argument");
  need(known_type(a->type), "unknown element type");
  need(a->score == EPS_B200_SCORE_SOFTMAX || a->score == EPS_B200_SCORE_SIGMOID, "unknown score");
  need(a->experts > 0 && a->experts <= EPS_B200_ROUTE_EXPERTS, "1 to 1024 experts");
  need(a->top_k > 0 && a->top_k <= EPS_B200_ROUTE_TOP_K, "top_k is 1 to 32");
  need(a->tokens < (1ull << 31) && a->tokens * a->top_k < (1ull << 31), "tokens * top_k must be below 2^31");
  need(std::isfinite(a->weight), "the weight must be finite");
  need(a->logits || !a->tokens, "null logits");
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
  return blocks == 1 ? 0 : (uint64_t)blocks / kTogether * (2 * (uint64_t)experts + 1) * 4;
}

int eps_b200_balance_loss(const EpsB200BalanceLoss* a, const int32_t* chosen, float* loss, int32_t* counts, float* mass, int32_t* counted,
                          void* workspace, uint64_t workspace_bytes, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Forward f{};
    static_cast<Rows&>(f) = checked(a);
    need(loss && counts && mass && counted, "null balance output");
    need(chosen || !a->tokens, "null chosen experts");
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
    const bool wide = wide_rows(a->logits, a->logits_stride, size) && a->experts * size % 16 == 0;
    const unsigned grid = forward_blocks(a->tokens, a->experts, sm_count(a->device));
    const auto s = static_cast<cudaStream_t>(stream);
    const bool sigmoid = a->score == EPS_B200_SCORE_SIGMOID;
    if (a->type == EPS_B200_F32) forward<float>(f, wide, sigmoid, grid, a->device, s);
    else if (a->type == EPS_B200_BF16) forward<bf16>(f, wide, sigmoid, grid, a->device, s);
    else forward<f16>(f, wide, sigmoid, grid, a->device, s);
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
    if (!a->tokens) return;
    b.counts = counts;
    b.counted = counted;
    b.dloss = dloss;
    b.add = add;
    b.add_stride = add_stride;
    b.out = dlogits;
    b.out_stride = dlogits_stride;
    OnDevice on(a->device);
    const size_t size = size_of(a->type);
    const bool wide = wide_rows(a->logits, a->logits_stride, size) && wide_rows(dlogits, dlogits_stride, size) &&
                      (!add || wide_rows(add, add_stride, size)) && a->experts * size % 16 == 0;
    const auto s = static_cast<cudaStream_t>(stream);
    const bool sigmoid = a->score == EPS_B200_SCORE_SIGMOID;
    if (a->type == EPS_B200_F32) backward<float>(b, wide, sigmoid, a->device, s);
    else if (a->type == EPS_B200_BF16) backward<bf16>(b, wide, sigmoid, a->device, s);
    else backward<f16>(b, wide, sigmoid, a->device, s);
  });
}

}  // extern "C"
