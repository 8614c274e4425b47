// route_experts.cu -- routing of tokens to experts (eps_b200_route_experts,
// eps_b200_route_experts_backward).
//
// Mathematics: s = softmax(l) or 1 / (1 + exp(-l)); key = s + bias; the best groups
// by the sum of their two best keys; the k best keys in them; w = s / sum(s) * scale.
// A masked expert (l = -inf) has the lowest key there is: its bias does not bring it back.
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
// key and the lowest lane that holds it owns the lowest index.  What bounds it is the
// number of instructions a token takes (the logits of a batch are a few megabytes):
// every lane sorts its own few keys once, and then only offers the best it has left (in
// registers up to 8 keys a lane; the 16 or 32 of more than 256 experts lie in local memory).
// Measured at 32771 x 256 floats, top 8 of the best 4 of 8 groups: 46 us (850
// instructions a token; 132 with the best key searched anew each time and groups scored
// lane by lane), 6 to scan the tiles and 5 to place; the gradient at 32771 x 96 bf16 19.
//
// The sort by expert is a counting sort in three steps.  A tile is the tokens of one
// block; each of its warps counts its own run of consecutive tokens, whose experts
// are distinct within a token, so counting needs no atomics and an entry's count
// before its own increment is its rank in the run.  The block adds up its warps'
// counts; route_scan turns tile counts into starts within an expert; route_place adds
// the experts' starts and writes.  One tile does all of it in the first launch.
#include <cfloat>
#include <cmath>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

constexpr unsigned kWarps = 8;             // of a tile
constexpr unsigned kRun = 8;               // tokens of a warp's run, where there are several tiles
constexpr unsigned kTile = kWarps * kRun;

struct Route {
  const void* logits;
  int64_t stride;
  const float* bias;
  int32_t* chosen;
  float* weights;
  int32_t *order, *position, *offsets;
  uint32_t* counts;                        // [tiles][experts]; at the end, the experts' totals
  uint16_t* ranks;                         // [tokens * top_k]
  uint64_t tokens;
  unsigned experts, top_k, groups, top_groups, per_group, tiles, run;
  int softmax, renormalise, wide, wide_out;
  float scale;
  const int32_t* given;                    // backward: chosen, dweights -> dlogits
  const float* dweights;
  void* dlogits;
  int64_t dstride;
};

// Orders like the floats, infinities too; 0 is below every one that is not NaN.
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned u = __float_as_uint(v + 0.f);       // -0 is 0
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

// Orders like the floats, -FLT_MAX and above; 0 is below every image.  NaN and
// -inf take the place of the lowest finite value.
__device__ __forceinline__ unsigned image(float key) {
  return ordered(key >= -FLT_MAX ? key : -FLT_MAX);
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

// The sum of n over the lanes up to this one.
__device__ __forceinline__ unsigned inclusive(unsigned n, unsigned lane) {
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned up = __shfl_up_sync(~0u, n, o);
    if (lane >= o) n += up;
  }
  return n;
}

// The scores of a token; lanes past the experts hold 0.
// RANKED: with the operations that the ranking is defined by.  The gradient, which ranks
// nothing, multiplies by the reciprocal of a sum in 32 bits: one rounding more a score.
template <int EPL, bool RANKED>
__device__ __forceinline__ void score(const Route& a, float (&x)[EPL]) {
  if (!a.softmax) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = __fadd_rn(1.f, expf(-x[i]));
    reciprocals<EPL>(x);
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
  std::conditional_t<RANKED, double, float> sum = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    x[i] = top == -INFINITY ? 0.f : expf(__fsub_rn(x[i], top));
    sum += x[i];
  }
#pragma unroll
  for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
  const float total = (float)sum;
  if constexpr (RANKED) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = total == 0.f ? 0.f : __fdiv_rn(x[i], total);
  } else {
    const float by = total == 0.f ? 0.f : __fdiv_rn(1.f, total);
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] *= by;
  }
}

// Shared memory of a warp: its counts, its token's scores and sorted keys, and, for
// groups that lanes do not divide evenly, the keys by expert and the groups' scores.
struct Scratch {
  uint16_t* count;     // [experts]
  int* chosen;         // [32]
  float* score;        // [32 * EPL]
  uint64_t* sorted;    // [32][EPL + 2]: an odd number of 16-byte words a lane meets all banks
  unsigned* keys;      // [experts]
  float* groups;       // [groups]
};

__host__ __device__ __forceinline__ unsigned scratch_bytes(unsigned experts, unsigned per_lane, unsigned groups, bool spread) {
  return ((experts * 2 + 15) / 16 * 16 + 128 + 32 * per_lane * 4 + 32 * (per_lane + 2) * 8 + (spread ? (experts + groups) * 4 : 0) + 15) / 16 * 16;
}

// Descending (K. Batcher's odd-even merge sort), N a power of two.
template <int N>
__device__ __forceinline__ void sort(uint64_t (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint64_t a = v[i + j], b = v[i + j + k];
            v[i + j] = a > b ? a : b;
            v[i + j + k] = a > b ? b : a;
          }
}

__device__ __forceinline__ float image_value(unsigned u) { return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u); }

// Whether every group is a run of whole lanes, a power of two of them.
__host__ __device__ __forceinline__ bool lanes_divide(unsigned per_group, unsigned per_lane) {
  const unsigned lanes = per_group / per_lane;
  return per_group % per_lane == 0 && (lanes & (lanes - 1)) == 0;
}

// Clears the images of experts outside the best groups: a group stays if fewer than
// top_groups come before it.
template <int EPL>
__device__ __forceinline__ void keep_groups(const Route& a, unsigned (&key)[EPL], unsigned lane, const Scratch& s) {
  const unsigned e0 = lane * EPL;
  if (lanes_divide(a.per_group, EPL)) {
    unsigned first = 0, second = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      second = max(second, min(first, key[i]));
      first = max(first, key[i]);
    }
    const unsigned lanes = a.per_group / EPL;
    for (unsigned o = 1; o < lanes; o *= 2) {
      const unsigned f = __shfl_xor_sync(~0u, first, o), g = __shfl_xor_sync(~0u, second, o);
      second = max(max(second, g), min(first, f));
      first = max(first, f);
    }
    const float mine = a.per_group > 1 ? __fadd_rn(image_value(first), image_value(second)) : image_value(first);
    // the best of what is left, top_groups times; a group is where its first lane is
    unsigned left = e0 < a.experts ? ordered(mine) : 0, kept = 0;
    for (unsigned k = 0; k < a.top_groups; ++k) {
      const unsigned top = __reduce_max_sync(~0u, left);
      const unsigned first_lane = __ffs(__ballot_sync(~0u, left == top)) - 1;
      const unsigned me = (lane ^ first_lane) < lanes;      // same group: the lanes' upper bits agree
      left = me ? 0 : left;
      kept |= me;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = kept ? key[i] : 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (e0 + i < a.experts) s.keys[e0 + i] = key[i];
  __syncwarp();
  for (unsigned g = lane; g < a.groups; g += 32) {
    unsigned first = 0, second = 0;
    for (unsigned i = 0; i < a.per_group; ++i) {
      const unsigned k = s.keys[g * a.per_group + i];
      second = max(second, min(first, k));
      first = max(first, k);
    }
    s.groups[g] = a.per_group > 1 ? __fadd_rn(image_value(first), image_value(second)) : image_value(first);
  }
  __syncwarp();
  for (unsigned g = lane; g < a.groups; g += 32) {
    const float mine = s.groups[g];
    unsigned before = 0;
    for (unsigned o = 0; o < a.groups; ++o) {
      const float v = s.groups[o];
      before += v > mine || (v == mine && o < g);
    }
    s.keys[g] = before < a.top_groups;      // the keys are in registers
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (e0 + i < a.experts && !s.keys[(e0 + i) / a.per_group]) key[i] = 0;
  __syncwarp();
}

template <class T, int EPL>
__global__ void __launch_bounds__(kWarps * 32, EPL <= 8 ? 4 : EPL == 16 ? 2 : 1) route_tokens(const Route a) {
  extern __shared__ __align__(16) unsigned char raw[];
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const bool grouped = a.groups > 1 && a.top_groups < a.groups;
  const unsigned each = scratch_bytes(a.experts, EPL, a.groups, grouped && !lanes_divide(a.per_group, EPL));
  unsigned char* const p0 = raw + warp * each;
  unsigned char* const p1 = p0 + (a.experts * 2 + 15) / 16 * 16;
  unsigned char* const p2 = p1 + 128 + 32 * EPL * 4;
  unsigned char* const p3 = p2 + 32 * (EPL + 2) * 8;
  const Scratch s{reinterpret_cast<uint16_t*>(p0), reinterpret_cast<int*>(p1), reinterpret_cast<float*>(p1 + 128), reinterpret_cast<uint64_t*>(p2),
                  reinterpret_cast<unsigned*>(p3), reinterpret_cast<float*>(p3) + a.experts};
  const bool sorting = a.order != nullptr;
  uint16_t* const ranks = reinterpret_cast<uint16_t*>(raw + kWarps * each + a.experts * 4);     // of the tile's entries in their warp's run
  if (sorting)
    for (unsigned e = lane; e < a.experts; e += 32) s.count[e] = 0;
  float bias[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i)       // behind the last expert: a key that every expert's comes before
    bias[i] = lane * EPL + i >= a.experts ? -INFINITY : a.bias ? a.bias[lane * EPL + i] : 0.f;
  __syncwarp();

  const uint64_t tile = (uint64_t)blockIdx.x * kTile, begin = tile + warp * a.run, end = min(begin + a.run, a.tokens);
  const T* const logits = static_cast<const T*>(a.logits);
  float next[EPL];
  if (begin < end) load_logits<T, EPL>(a, logits + begin * a.stride, lane, next);
  for (uint64_t token = begin; token < end; ++token) {
    float p[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] = next[i];
    if (token + 1 < end) load_logits<T, EPL>(a, logits + (token + 1) * a.stride, lane, next);
    float lowest = p[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) lowest = fminf(lowest, p[i]);
    unsigned masked = 0;                // bit i: the lane's expert i is masked
    if (lowest == -INFINITY) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) masked |= (unsigned)(p[i] == -INFINITY) << i;
    }
    score<EPL, true>(a, p);
    unsigned key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = image(__fadd_rn(p[i], bias[i]));
    if (masked) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) key[i] = masked >> i & 1 ? image(-INFINITY) : key[i];
    }
    if (grouped) keep_groups<EPL>(a, key, lane, s);

    // by key, and the lower index of equal keys first
    uint64_t order[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) order[i] = (uint64_t)key[i] << 32 | (unsigned)~(lane * EPL + i);
    sort<EPL>(order);
    uint64_t* const mine = s.sorted + lane * (EPL + 2);
    if constexpr (EPL >= 4) {
#pragma unroll
      for (int i = 0; i < EPL; i += 2) *reinterpret_cast<ulonglong2*>(mine + i) = make_ulonglong2(order[i], order[i + 1]);
#pragma unroll
      for (int i = 0; i < EPL; i += 4) *reinterpret_cast<float4*>(s.score + lane * EPL + i) = make_float4(p[i], p[i + 1], p[i + 2], p[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        mine[i] = order[i];
        s.score[lane * EPL + i] = p[i];
      }
    }
    mine[EPL] = 0;
    unsigned taken = 0;
    uint64_t best = order[0];
    for (unsigned k = 0; k < a.top_k; ++k) {
      const unsigned top = __reduce_max_sync(~0u, (unsigned)(best >> 32));
      const unsigned owner = __ffs(__ballot_sync(~0u, (unsigned)(best >> 32) == top)) - 1;
      if (lane == owner) s.chosen[k] = (int)~(unsigned)best;
      taken += lane == owner;
      best = mine[taken];
    }
    __syncwarp();
    const int expert = lane < a.top_k ? s.chosen[lane] : 0;
    float weight = lane < a.top_k ? s.score[expert] : 0.f;
    __syncwarp();
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
      if (sorting) ranks[entry - tile * a.top_k] = s.count[expert]++;
    }
    __syncwarp();
  }
  if (!sorting) return;
  __syncthreads();
  // warps' counts to starts within the tile; the tile's totals
  unsigned* const total = reinterpret_cast<unsigned*>(raw + kWarps * each);
  for (unsigned e = threadIdx.x; e < a.experts; e += blockDim.x) {
    unsigned before = 0;
#pragma unroll
    for (unsigned w = 0; w < kWarps; ++w) {
      uint16_t* const c = reinterpret_cast<uint16_t*>(raw + w * each) + e;
      const unsigned n = *c;
      *c = (uint16_t)before;
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
        const unsigned sum = inclusive(n, lane);
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
    const unsigned w = (unsigned)(i - first) / (a.run * a.top_k);
    const unsigned e = (unsigned)a.chosen[i];
    const unsigned in_tile = reinterpret_cast<const uint16_t*>(raw + w * each)[e] + ranks[i - first];
    if (a.tiles > 1) {
      a.ranks[i] = (uint16_t)in_tile;
    } else {
      const unsigned at = total[e] + in_tile;
      a.position[i] = (int32_t)at;
      a.order[at] = (int32_t)i;
    }
  }
}

// counts[tile][e] -> entries of expert e in the tiles before; counts[tiles][e] = all of
// them.  A block has 32 experts, a warp of it a run of tiles, read twice.
constexpr unsigned kScanWarps = 32;
__global__ void __launch_bounds__(32 * kScanWarps) route_scan(const Route a) {
  __shared__ unsigned sums[kScanWarps][33];
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32, e = blockIdx.x * 32 + lane;
  const unsigned run = (a.tiles + kScanWarps - 1) / kScanWarps, first = warp * run, last = min(first + run, a.tiles);
  unsigned n = 0;
  if (e < a.experts) {
#pragma unroll 8
    for (unsigned t = first; t < last; ++t) n += a.counts[(uint64_t)t * a.experts + e];
  }
  sums[warp][lane] = n;
  __syncthreads();
  const unsigned mine = sums[lane][warp], sum = inclusive(mine, lane);     // lane: run of tiles, warp: expert
  sums[lane][warp] = sum - mine;
  if (lane == 31 && blockIdx.x * 32 + warp < a.experts) a.counts[(uint64_t)a.tiles * a.experts + blockIdx.x * 32 + warp] = sum;
  __syncthreads();
  if (e >= a.experts) return;
  unsigned before = sums[warp][lane];
#pragma unroll 8
  for (unsigned t = first; t < last; ++t) {
    unsigned* const c = a.counts + (uint64_t)t * a.experts + e;
    const unsigned here = *c;
    *c = before;
    before += here;
  }
}

// Every block sums the experts' totals to starts for itself; the first writes them.
__global__ void __launch_bounds__(256) route_place(const Route a) {
  __shared__ unsigned starts[EPS_B200_ROUTE_EXPERTS];
  __shared__ unsigned sums[8];
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const unsigned* const totals = a.counts + (uint64_t)a.tiles * a.experts;
  unsigned carry = 0;
  for (unsigned e0 = 0; e0 < a.experts; e0 += 256) {
    const unsigned e = e0 + threadIdx.x, n = e < a.experts ? totals[e] : 0, sum = inclusive(n, lane);
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    unsigned before = carry, all = 0;
#pragma unroll
    for (unsigned w = 0; w < 8; ++w) {
      before += w < warp ? sums[w] : 0;
      all += sums[w];
    }
    if (e < a.experts) starts[e] = before + sum - n;
    carry += all;
    __syncthreads();
  }
  if (blockIdx.x == 0) {
    for (unsigned e = threadIdx.x; e < a.experts; e += 256) a.offsets[e] = (int32_t)starts[e];
    if (threadIdx.x == 0) a.offsets[a.experts] = (int32_t)carry;
  }
  const uint64_t entries = a.tokens * a.top_k;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (uint64_t)gridDim.x * 256) {
    const unsigned tile = (unsigned)i / (kTile * a.top_k);
    const unsigned e = (unsigned)a.chosen[i];
    const unsigned at = starts[e] + a.counts[(uint64_t)tile * a.experts + e] + a.ranks[i];
    a.position[i] = (int32_t)at;
    a.order[at] = (int32_t)i;
  }
}

// A warp walks tokens, the next one's logits under way.
template <class T, int EPL>
__global__ void __launch_bounds__(kWarps * 32) route_gradient(const Route a) {
  extern __shared__ __align__(16) unsigned char raw[];
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float* const ds = reinterpret_cast<float*>(raw) + warp * 32 * EPL;      // zeros but while a token's chosen are in it
#pragma unroll
  for (int i = 0; i < EPL; ++i) ds[i * 32 + lane] = 0.f;
  const uint64_t stride = (uint64_t)gridDim.x * kWarps;
  uint64_t token = (uint64_t)blockIdx.x * kWarps + warp;
  const T* const logits = static_cast<const T*>(a.logits);
  float next[EPL];
  if (token < a.tokens) load_logits<T, EPL>(a, logits + token * a.stride, lane, next);
  auto sum = [](float v) {
#pragma unroll
    for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    return v;
  };
  for (; token < a.tokens; token += stride) {
    float p[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] = next[i];
    int expert = -1;
    float d = 0.f;
    if (lane < a.top_k) {
      expert = a.given[token * a.top_k + lane];
      d = a.dweights[token * a.top_k + lane] * a.scale;
      if ((unsigned)expert >= a.experts) expert = -1;
    }
    if (token + stride < a.tokens) load_logits<T, EPL>(a, logits + (token + stride) * a.stride, lane, next);
    score<EPL, false>(a, p);
    // the chosen's scores, by way of the lanes that hold them
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float v = __shfl_sync(~0u, p[i], expert < 0 ? 0 : expert / EPL);
      if (expert >= 0 && expert % EPL == i) s = v;
    }
    if (expert < 0) d = 0.f;
    if (a.renormalise) {
      const float total = sum(s), mean = sum(d * s);
      const float by = total == 0.f ? 0.f : __fdiv_rn(1.f, total);
      d = expert < 0 ? 0.f : (d - mean * by) * by;
    }
    const float dot = a.softmax ? sum(d * s) : 0.f;
    if (expert >= 0) atomicAdd(ds + expert, d);      // distinct experts: no order to depend on
    __syncwarp();
    float g[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) g[i] = ds[lane * EPL + i];
    __syncwarp();
    if (expert >= 0) ds[expert] = 0.f;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < EPL; ++i) g[i] = a.softmax ? p[i] * (g[i] - dot) : g[i] * p[i] * (1.f - p[i]);
    T* const out = static_cast<T*>(a.dlogits) + token * a.dstride + lane * EPL;
    if (a.wide_out && (lane + 1) * EPL <= a.experts) {
      constexpr int W = EPL * sizeof(T) > 16 ? 16 / sizeof(T) : EPL;
#pragma unroll
      for (int i = 0; i < EPL; i += W) store_pack<T, W>(out + i, narrow<T, W>(reinterpret_cast<const float(&)[W]>(g[i])));
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (lane * EPL + i < a.experts) out[i] = from_float<T>(g[i]);
    }
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
  r.run = r.tiles > 1 ? kRun : (unsigned)ceil_div(a->tokens, kWarps);
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

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_route_experts_workspace(uint64_t tokens, uint32_t experts, uint32_t top_k) {
  if (tokens <= kTile) return 0;
  return round_up(tokens * top_k * 2, 16) + (ceil_div(tokens, kTile) + 1) * experts * 4;
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
    if (order && r.tiles > 1) {
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
    by_type(a->type, [&](auto t) {
      by_experts(r.experts, [&](auto epl) {
        const bool spread = r.groups > 1 && r.top_groups < r.groups && !lanes_divide(r.per_group, decltype(epl)::value);
        const size_t shared = kWarps * scratch_bytes(r.experts, decltype(epl)::value, r.groups, spread) + r.experts * 4 + (order ? kTile * r.top_k * 2 : 0);
        constexpr auto kernel = route_tokens<decltype(t), decltype(epl)::value>;
        room<kernel>(a->device);
        kernel<<<r.tiles, kWarps * 32, shared, st>>>(r);
      });
    });
    check(cudaGetLastError(), "route_experts");
    if (order && r.tiles > 1) {
      route_scan<<<(unsigned)ceil_div(r.experts, 32), 32 * kScanWarps, 0, st>>>(r);
      check(cudaGetLastError(), "route_scan");
      const uint64_t most = (uint64_t)sm_count(a->device) * 8, all = ceil_div(r.tokens * r.top_k, 256);
      route_place<<<(unsigned)(all < most ? all : most), 256, 0, st>>>(r);
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
    r.wide_out = lanes_wide(dlogits, dlogits_stride, r.experts, a->type);
    const uint64_t most = (uint64_t)sm_count(a->device) * 8, all = ceil_div(r.tokens, kWarps);
    by_type(a->type, [&](auto t) {
      by_experts(r.experts, [&](auto epl) {
        constexpr auto kernel = route_gradient<decltype(t), decltype(epl)::value>;
        const size_t shared = kWarps * 32 * decltype(epl)::value * 4;
        room<kernel>(a->device);
        kernel<<<(unsigned)(all < most ? all : most), kWarps * 32, shared, static_cast<cudaStream_t>(stream)>>>(r);
      });
    });
    check(cudaGetLastError(), "route_experts_backward");
  });
}

}  // extern "C"
