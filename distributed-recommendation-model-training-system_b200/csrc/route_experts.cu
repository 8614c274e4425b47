// route_experts.cu -- routing of tokens to experts (eps_b200_route_experts,
// eps_b200_route_experts_backward).
//
// Mathematics: s = softmax(l) or 1 / (1 + exp(-l)); key = s + bias; the best groups
// by the sum of their two best keys; the k best keys in them; w = s / sum(s) * scale.
// Backward, over the chosen c with d = dw * scale:
//   ds_c = (d_c - sum_j d_j s_j / S) / S   (renormalised, S = sum_j s_j; else d_c)
//   softmax: dl_e = s_e (ds_e - sum_c ds_c s_c),   sigmoid: dl_e = ds_e s_e (1 - s_e)
//
// The ranking is made of correctly rounded additions and divisions of expf values,
// and the softmax's sum is taken in 64 bits, so that it does not hang on the order
// of its terms: equal inputs rank equally wherever they are computed this way.
//
// A warp owns a token; lane l holds experts l * EPL .. l * EPL + EPL - 1.  Ranking is
// on unsigned images of the keys (`image`), so one warp instruction finds the best
// key and the lowest lane that holds it owns the lowest index.
//
// The sort by expert is a counting sort in three steps.  A tile is the tokens of one
// block; each of its warps counts its own run of consecutive tokens, whose experts
// are distinct within a token, so counting needs no atomics and an entry's count
// before its own increment is its rank in the run.  The block adds up its warps'
// counts; route_scan turns tile counts into starts; route_place writes.  One tile
// does all of it in the first launch.
#include <cfloat>
#include <cmath>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

constexpr unsigned kWarps = 8;             // of a tile
constexpr unsigned kRun = 16;              // tokens of a warp's run
constexpr unsigned kTile = kWarps * kRun;

struct Route {
  const void* logits;
  int64_t stride;
  const float* bias;
  int32_t* chosen;
  float* weights;
  int32_t *order, *position, *offsets;
  uint32_t* counts;                        // [tiles][experts]
  uint16_t* ranks;                         // [tokens * top_k]
  uint64_t tokens;
  unsigned experts, top_k, groups, top_groups, per_group, tiles;
  int softmax, renormalise, wide;
  float scale;
  const int32_t* given;                    // backward: chosen, dweights -> dlogits
  const float* dweights;
  void* dlogits;
  int64_t dstride;
};

// Orders like the floats, -FLT_MAX and above; 0 is below every image.  NaN and
// -inf take the place of the lowest finite value.
__device__ __forceinline__ unsigned image(float key) {
  if (!(key >= -FLT_MAX)) key = -FLT_MAX;
  const unsigned u = __float_as_uint(key + 0.f);     // -0 is 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o /= 2) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

template <class T, int EPL>
__device__ __forceinline__ void load_logits(const Route& a, const T* row, unsigned lane, float (&x)[EPL]) {
  const unsigned e0 = lane * EPL;
  if (a.wide && e0 + EPL <= a.experts) {
    constexpr int W = EPL * sizeof(T) > 16 ? 16 / sizeof(T) : EPL;
#pragma unroll
    for (int i = 0; i < EPL; i += W) {
      const Pack<T, W> k = load_once<T, W>(row + e0 + i);
#pragma unroll
      for (int j = 0; j < W; ++j) x[i + j] = to_float(k.v[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = e0 + i < a.experts ? to_float(row[e0 + i]) : -INFINITY;
  }
}

// The scores of a token; lanes past the experts hold 0.
template <int EPL>
__device__ __forceinline__ void score(const Route& a, float (&x)[EPL]) {
  if (!a.softmax) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = __fdiv_rn(1.f, __fadd_rn(1.f, expf(-x[i])));
    return;
  }
  float top = x[0];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    top = fmaxf(top, x[i]);
    nan |= x[i] != x[i];
  }
  top = warp_max(top);
  nan = __any_sync(~0u, nan);
  if (nan) top = NAN;
  double sum = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    x[i] = top == -INFINITY ? 0.f : expf(__fsub_rn(x[i], top));
    sum += (double)x[i];
  }
#pragma unroll
  for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
  const float total = (float)sum;
#pragma unroll
  for (int i = 0; i < EPL; ++i) x[i] = total == 0.f ? 0.f : __fdiv_rn(x[i], total);
}

// Shared memory of a warp: the images of its keys, then its groups' scores.
struct Scratch {
  unsigned* keys;      // [experts]
  float* groups;       // [groups]
};

// Clears the images of experts outside the best groups.
template <int EPL>
__device__ __forceinline__ void keep_groups(const Route& a, const float (&p)[EPL], unsigned (&key)[EPL], unsigned lane, const Scratch& s) {
  const unsigned e0 = lane * EPL;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (e0 + i < a.experts) s.keys[e0 + i] = key[i];
  __syncwarp();
  auto value = [](unsigned u) { return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u); };
  for (unsigned g = lane; g < a.groups; g += 32) {
    unsigned first = 0, second = 0;
    for (unsigned i = 0; i < a.per_group; ++i) {
      const unsigned k = s.keys[g * a.per_group + i];
      second = max(second, min(first, k));
      first = max(first, k);
    }
    s.groups[g] = a.per_group > 1 ? __fadd_rn(value(first), value(second)) : value(first);
  }
  __syncwarp();
  // a group stays if fewer than top_groups come before it
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    if (e0 + i >= a.experts) continue;
    const unsigned g = (e0 + i) / a.per_group;
    const float mine = s.groups[g];
    unsigned before = 0;
    for (unsigned o = 0; o < a.groups; ++o) {
      const float v = s.groups[o];
      before += v > mine || (v == mine && o < g);
    }
    if (before >= a.top_groups) key[i] = 0;
  }
  __syncwarp();
}

template <class T, int EPL>
__global__ void __launch_bounds__(kWarps * 32) route_tokens(const Route a) {
  extern __shared__ unsigned char raw[];
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  // [kWarps][experts] counts, then each warp's scratch
  uint16_t* const counts = reinterpret_cast<uint16_t*>(raw);
  unsigned char* const rest = raw + (kWarps * a.experts * 2 + 15) / 16 * 16 + warp * ((a.experts + a.groups) * 4);
  const Scratch s{reinterpret_cast<unsigned*>(rest), reinterpret_cast<float*>(rest) + a.experts};
  uint16_t* const count = counts + warp * a.experts;
  const bool sorting = a.order != nullptr;
  if (sorting)
    for (unsigned e = lane; e < a.experts; e += 32) count[e] = 0;
  __syncwarp();

  const uint64_t tile = (uint64_t)blockIdx.x * kTile;
  for (unsigned r = 0; r < kRun; ++r) {
    const uint64_t token = tile + warp * kRun + r;
    if (token >= a.tokens) break;
    float p[EPL];
    load_logits<T, EPL>(a, static_cast<const T*>(a.logits) + token * a.stride, lane, p);
    score<EPL>(a, p);
    unsigned key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const unsigned e = lane * EPL + i;
      key[i] = e < a.experts ? image(a.bias ? __fadd_rn(p[i], a.bias[e]) : p[i]) : 0;
    }
    if (a.groups > 1 && a.top_groups < a.groups) keep_groups<EPL>(a, p, key, lane, s);

    int expert = 0;          // of slot `lane`
    float weight = 0.f;
    for (unsigned k = 0; k < a.top_k; ++k) {
      unsigned best = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) best = max(best, key[i]);
      const unsigned top = __reduce_max_sync(~0u, best);
      const unsigned owner = __ffs(__ballot_sync(~0u, best == top)) - 1;
      int at = 0;
      float w = 0.f;
      if (lane == owner) {
        bool found = false;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (!found && key[i] == top) {
            found = true;
            at = lane * EPL + i;
            w = p[i];
            key[i] = 0;
          }
      }
      at = __shfl_sync(~0u, at, owner);
      w = __shfl_sync(~0u, w, owner);
      if (lane == k) { expert = at; weight = w; }
    }
    float total = 0.f;
    if (a.renormalise) {
      total = weight;
#pragma unroll
      for (int o = 16; o; o /= 2) total += __shfl_xor_sync(~0u, total, o);
      weight = total == 0.f ? 0.f : __fdiv_rn(weight, total);
    }
    if (lane < a.top_k) {
      const uint64_t entry = token * a.top_k + lane;
      a.chosen[entry] = expert;
      a.weights[entry] = weight * a.scale;
      if (sorting) a.ranks[entry] = count[expert]++;
    }
    __syncwarp();
  }
  if (!sorting) return;
  __syncthreads();
  // warps' counts to starts within the tile; the tile's totals
  unsigned* const total = reinterpret_cast<unsigned*>(raw + (kWarps * a.experts * 2 + 15) / 16 * 16);   // the scratch, no longer used
  for (unsigned e = threadIdx.x; e < a.experts; e += blockDim.x) {
    unsigned before = 0;
#pragma unroll
    for (unsigned w = 0; w < kWarps; ++w) {
      const unsigned n = counts[w * a.experts + e];
      counts[w * a.experts + e] = (uint16_t)before;
      before += n;
    }
    if (a.tiles > 1) a.counts[(uint64_t)blockIdx.x * a.experts + e] = before;
    else total[e] = before;
  }
  __syncthreads();
  if (a.tiles == 1) {
    if (warp == 0) {          // the experts' starts
      unsigned carry = 0;
      for (unsigned e0 = 0; e0 < a.experts; e0 += 32) {
        const unsigned n = e0 + lane < a.experts ? total[e0 + lane] : 0;
        unsigned sum = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const unsigned up = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += up;
        }
        if (e0 + lane < a.experts) {
          total[e0 + lane] = carry + sum - n;
          a.offsets[e0 + lane] = (int32_t)(carry + sum - n);
        }
        carry += __shfl_sync(~0u, sum, 31);
      }
      if (lane == 0) a.offsets[a.experts] = (int32_t)carry;
    }
    __syncthreads();
  }
  const uint64_t first = tile * a.top_k, last = min(tile + kTile, a.tokens) * a.top_k;
  for (uint64_t i = first + threadIdx.x; i < last; i += blockDim.x) {
    const unsigned w = (unsigned)((i - first) / (kRun * a.top_k));
    const unsigned e = (unsigned)a.chosen[i];
    const unsigned in_tile = counts[w * a.experts + e] + a.ranks[i];
    if (a.tiles > 1) {
      a.ranks[i] = (uint16_t)in_tile;
    } else {
      const unsigned at = total[e] + in_tile;
      a.position[i] = (int32_t)at;
      a.order[at] = (int32_t)i;
    }
  }
}

// counts[tile][e] -> entries of expert e before the tile; offsets.  One block; each
// thread owns one expert at a time.
__global__ void __launch_bounds__(1024) route_scan(const Route a) {
  __shared__ unsigned sums[32];
  unsigned carry = 0;
  for (unsigned e0 = 0; e0 < a.experts; e0 += blockDim.x) {
    const unsigned e = e0 + threadIdx.x;
    unsigned n = 0;
    if (e < a.experts)
      for (unsigned t = 0; t < a.tiles; ++t) {
        const unsigned c = a.counts[(uint64_t)t * a.experts + e];
        a.counts[(uint64_t)t * a.experts + e] = n;
        n += c;
      }
    unsigned sum = n;
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned up = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    unsigned before = carry, all = 0;
    for (unsigned w = 0; w < blockDim.x / 32; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    if (e < a.experts) a.offsets[e] = (int32_t)(before + sum - n);
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.offsets[a.experts] = (int32_t)carry;
}

__global__ void __launch_bounds__(256) route_place(const Route a) {
  const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.tokens * a.top_k) return;
  const uint64_t tile = i / ((uint64_t)kTile * a.top_k);
  const unsigned e = (unsigned)a.chosen[i];
  const unsigned at = (unsigned)a.offsets[e] + a.counts[tile * a.experts + e] + a.ranks[i];
  a.position[i] = (int32_t)at;
  a.order[at] = (int32_t)i;
}

template <class T, int EPL>
__global__ void __launch_bounds__(kWarps * 32) route_gradient(const Route a) {
  extern __shared__ unsigned char raw[];
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float* const ds = reinterpret_cast<float*>(raw) + warp * a.experts;
  const uint64_t token = (uint64_t)blockIdx.x * kWarps + warp;
  if (token >= a.tokens) return;
  float p[EPL];
  load_logits<T, EPL>(a, static_cast<const T*>(a.logits) + token * a.stride, lane, p);
  score<EPL>(a, p);
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (lane * EPL + i < a.experts) ds[lane * EPL + i] = p[i];
  __syncwarp();
  int expert = -1;
  float d = 0.f, s = 0.f;
  if (lane < a.top_k) {
    expert = a.given[token * a.top_k + lane];
    if (expert < 0 || (unsigned)expert >= a.experts) expert = -1;
    if (expert >= 0) {
      d = a.dweights[token * a.top_k + lane] * a.scale;
      s = ds[expert];
    }
  }
  auto sum = [](float v) {
#pragma unroll
    for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    return v;
  };
  if (a.renormalise) {
    const float total = sum(s);
    const float mean = sum(d * s) / total;
    d = total == 0.f || expert < 0 ? 0.f : (d - mean) / total;
  }
  const float dot = a.softmax ? sum(d * s) : 0.f;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (lane * EPL + i < a.experts) ds[lane * EPL + i] = 0.f;
  __syncwarp();
  if (expert >= 0) atomicAdd(ds + expert, d);      // distinct experts: no order to depend on
  __syncwarp();
  T* const out = static_cast<T*>(a.dlogits) + token * a.dstride;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const unsigned e = lane * EPL + i;
    if (e >= a.experts) continue;
    const float g = a.softmax ? p[i] * (ds[e] - dot) : ds[e] * p[i] * (1.f - p[i]);
    out[e] = from_float<T>(g);
  }
}

Route checked(const EpsB200RouteExperts* a) {
  need(a, "null routing arguments");
  need(known_type(a->type), "unknown element type");
  need(a->score == EPS_B200_SCORE_SOFTMAX || a->score == EPS_B200_SCORE_SIGMOID, "unknown score");
  need(a->experts > 0 && a->experts <= EPS_B200_ROUTE_EXPERTS, "experts out of range");
  need(a->groups > 0 && a->experts % a->groups == 0, "groups must divide the experts");
  need(a->top_groups > 0 && a->top_groups <= a->groups, "top_groups out of range");
  need(a->top_k > 0 && a->top_k <= EPS_B200_ROUTE_TOP_K, "top_k out of range");
  need(a->top_k <= a->experts / a->groups * a->top_groups, "more experts a token than its groups hold");
  need(a->tokens < (1ull << 31) && a->tokens * a->top_k < (1ull << 31), "too many tokens");
  need(a->scale == a->scale, "the scale is not a number");
  need(!a->tokens || a->logits, "null logits");
  Route r{};
  r.logits = a->logits;
  r.stride = a->logits_stride;
  r.tokens = a->tokens;
  r.experts = a->experts;
  r.top_k = a->top_k;
  r.groups = a->groups;
  r.top_groups = a->top_groups;
  r.per_group = a->experts / a->groups;
  r.tiles = (unsigned)ceil_div(a->tokens, kTile);
  r.softmax = a->score == EPS_B200_SCORE_SOFTMAX;
  r.renormalise = a->renormalise != 0;
  r.scale = a->scale;
  return r;
}

template <class F>
void by_type(int type, F f) {
  if (type == EPS_B200_F32) f(float{});
  else if (type == EPS_B200_BF16) f(bf16{});
  else f(f16{});
}

// Experts a lane: the power of two that covers them.
template <class F>
void by_experts(unsigned experts, F f) {
  if (experts <= 32) f(std::integral_constant<int, 1>{});
  else if (experts <= 64) f(std::integral_constant<int, 2>{});
  else if (experts <= 128) f(std::integral_constant<int, 4>{});
  else if (experts <= 256) f(std::integral_constant<int, 8>{});
  else if (experts <= 512) f(std::integral_constant<int, 16>{});
  else f(std::integral_constant<int, 32>{});
}

// Whether every lane's experts can be read 16 bytes (or its own few) at a time.
bool lanes_wide(const void* p, int64_t stride, unsigned experts, int type) {
  unsigned per = 1;
  while (per * 32 < experts) per *= 2;
  const size_t bytes = per * size_of(type) > 16 ? 16 : per * size_of(type);
  return aligned(p, bytes) && stride * (int64_t)size_of(type) % (int64_t)bytes == 0;
}

template <class K>
void room(K kernel, size_t bytes) {
  if (bytes > 48 * 1024)
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "cudaFuncSetAttribute");
}

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_route_experts_workspace(uint64_t tokens, uint32_t experts, uint32_t top_k) {
  return round_up(tokens * top_k * 2, 16) + ceil_div(tokens, kTile) * experts * 4;
}

int eps_b200_route_experts(const EpsB200RouteExperts* a, const float* bias, int32_t* chosen, float* weights,
                           int32_t* order, int32_t* position, int32_t* offsets, void* workspace,
                           uint64_t workspace_bytes, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Route r = checked(a);
    need(!r.tokens || (chosen && weights), "null output");
    need((order != nullptr) == (position != nullptr) && (order != nullptr) == (offsets != nullptr),
         "order, position and offsets come together");
    OnDevice on(a->device);
    const auto st = static_cast<cudaStream_t>(stream);
    if (!r.tokens) {
      if (offsets) check(cudaMemsetAsync(offsets, 0, (r.experts + 1) * 4, st), "cudaMemsetAsync");
      return;
    }
    if (order) {
      need(workspace && workspace_bytes >= eps_b200_route_experts_workspace(r.tokens, r.experts, r.top_k) &&
               aligned(workspace, 16), "routing workspace too small or not 16-byte aligned");
      r.ranks = static_cast<uint16_t*>(workspace);
      r.counts = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + round_up(r.tokens * r.top_k * 2, 16));
    }
    r.bias = bias;
    r.chosen = chosen;
    r.weights = weights;
    r.order = order;
    r.position = position;
    r.offsets = offsets;
    r.wide = lanes_wide(r.logits, r.stride, r.experts, a->type);
    const size_t shared = (kWarps * r.experts * 2 + 15) / 16 * 16 + kWarps * (r.experts + r.groups) * 4;
    by_type(a->type, [&](auto t) {
      by_experts(r.experts, [&](auto epl) {
        auto* kernel = route_tokens<decltype(t), decltype(epl)::value>;
        room(kernel, shared);
        kernel<<<r.tiles, kWarps * 32, shared, st>>>(r);
      });
    });
    check(cudaGetLastError(), "route_experts");
    if (order && r.tiles > 1) {
      route_scan<<<1, 1024, 0, st>>>(r);
      check(cudaGetLastError(), "route_scan");
      route_place<<<(unsigned)ceil_div(r.tokens * r.top_k, 256), 256, 0, st>>>(r);
      check(cudaGetLastError(), "route_place");
    }
  });
}

int eps_b200_route_experts_backward(const EpsB200RouteExperts* a, const int32_t* chosen, const float* dweights,
                                    void* dlogits, int64_t dlogits_stride, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Route r = checked(a);
    need(!r.tokens || (chosen && dweights && dlogits), "null gradient or output");
    if (!r.tokens) return;
    OnDevice on(a->device);
    r.given = chosen;
    r.dweights = dweights;
    r.dlogits = dlogits;
    r.dstride = dlogits_stride;
    r.wide = lanes_wide(r.logits, r.stride, r.experts, a->type);
    const size_t shared = kWarps * r.experts * 4;
    by_type(a->type, [&](auto t) {
      by_experts(r.experts, [&](auto epl) {
        auto* kernel = route_gradient<decltype(t), decltype(epl)::value>;
        room(kernel, shared);
        kernel<<<(unsigned)ceil_div(r.tokens, kWarps), kWarps * 32, shared, static_cast<cudaStream_t>(stream)>>>(r);
      });
    });
    check(cudaGetLastError(), "route_experts_backward");
  });
}

}  // extern "C"
