// gradient_norm.cu -- the norm over many gradients, its clip factor, clipping in place
// (eps_b200_gradient_norm).
//
// Mathematics:
//   norm = |u| sqrt(sum g^2) or |u| max |g|,  scale = u min(1, max_norm / norm),  g <- g scale
// The squares of one 16-byte load are added in float and go on in double.  Where a
// float could not hold that sum (it overflows, or its terms vanish) the squares are
// taken in double, so the norm is right over the whole range of the type.  A maximum
// is taken over the bits of |g|, where NaN is above infinity and is not lost.
//
// Bound: one read of every gradient; to clip, a read and a write more, from the last span
// back, where L2 still has what was read last.  A plan lists spans of 16 KB, each with its
// address, so one launch walks tensors of any size and type.  Blocks leave one sum each
// and the next launch adds them, in the same order in every block: no atomics, so results
// repeat exactly.  That launch begins while the first still runs and waits for its end
// (programmatic dependent launch), which saves 0.9 us.
//   1.5e8 bf16 measured: 49.7 us, 92 % of the copy rate.  2e8 floats clipped in place: 383
// us, 2.4 GB at 96 %.  1.3e6 floats clipped: 6.9 us.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <vector>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

constexpr unsigned kSpan = 16384;       // bytes of a span
constexpr unsigned kThreads = 256;
constexpr unsigned kBlocksEach = 8;     // blocks an SM
constexpr unsigned kMost = 2048;         // most blocks that leave a sum

struct Span {
  void* at;             // 16-byte aligned but for a tensor's first
  uint32_t elements;
  int32_t type;
};
static_assert(sizeof(Span) == 16, "one load");

// What a block gathers: a sum of squares, or the bits of a magnitude.
template <int KIND> struct Gather;
template <> struct Gather<EPS_B200_GRADIENT_L2> {
  using V = double;
  static __device__ __forceinline__ V join(V a, V b) { return a + b; }
  template <int N> static __device__ __forceinline__ void take(V& v, const float (&x)[N]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
    if (s >= 0x1p-90f && s <= 0x1p120f) {     // a square that vanishes is below 2^-149, no unit of such a sum
      v += (double)s;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v = fma((double)x[i], (double)x[i], v);
    }
  }
  static __device__ __forceinline__ double norm(V v) { return sqrt(v); }
};
template <> struct Gather<EPS_B200_GRADIENT_MAX> {
  using V = uint32_t;
  static __device__ __forceinline__ V join(V a, V b) { return max(a, b); }
  template <int N> static __device__ __forceinline__ void take(V& v, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v = max(v, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  }
  static __device__ __forceinline__ double norm(V v) { return (double)__uint_as_float(v); }
};

struct Call {
  const Span* spans;
  unsigned count;
  const float* gradient_scale;
  double max_norm;
  EpsB200GradientResult* result;
  double* sums;            // one 8-byte value a block
};

// Calls vector(p) for each whole 16 bytes of a span and single(p) for each element before
// or behind them.
template <class T, class F, class G>
__device__ __forceinline__ void walk(T* p, unsigned n, F vector, G single) {
  constexpr unsigned V = 16 / sizeof(T);
  const unsigned t = threadIdx.x, threads = blockDim.x;
  const unsigned head = min(n, (unsigned)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (unsigned)sizeof(T));
  const unsigned packs = (n - head) / V;
  T* const body = p + head;
  if (packs == kSpan / 16 && threads == kThreads) {
#pragma unroll
    for (unsigned j = 0; j < kSpan / 16 / kThreads; ++j) vector(body + (j * kThreads + t) * V);
  } else {
    for (unsigned j = t; j < packs; j += threads) vector(body + j * V);
  }
  const unsigned rest = n - head - packs * V;
  if (t < head) single(p + t);
  if (t < rest) single(body + packs * V + t);
}

template <int KIND, class T>
__device__ __forceinline__ void gather_span(const Span& s, typename Gather<KIND>::V& v) {
  constexpr int V = 16 / sizeof(T);
  walk(static_cast<T*>(s.at), s.elements,
       [&](const T* p) {
         float x[V];
         widen(load_pack<T, V>(p), x);
         Gather<KIND>::take(v, x);
       },
       [&](const T* p) {
         const float x[1] = {to_float(*p)};
         Gather<KIND>::take(v, x);
       });
}

template <class T>
__device__ __forceinline__ void clip_span(const Span& s, float scale) {
  constexpr int V = 16 / sizeof(T);
  walk(static_cast<T*>(s.at), s.elements,
       [&](T* p) {
         float x[V];
         widen(load_once<T, V>(p), x);
#pragma unroll
         for (int i = 0; i < V; ++i) x[i] *= scale;
         store_pack<T, V>(p, narrow<T, V>(x));
       },
       [&](T* p) { *p = from_float<T>(to_float(*p) * scale); });
}

// A block's value, the same in every thread.
template <int KIND>
__device__ __forceinline__ typename Gather<KIND>::V block_join(typename Gather<KIND>::V v) {
  using G = Gather<KIND>;
  __shared__ typename G::V each[32];
#pragma unroll
  for (int o = 16; o; o /= 2) v = G::join(v, __shfl_xor_sync(~0u, v, o));
  if (threadIdx.x % 32 == 0) each[threadIdx.x / 32] = v;
  __syncthreads();
  v = each[0];
  for (unsigned w = 1; w < blockDim.x / 32; ++w) v = G::join(v, each[w]);
  return v;
}

template <int KIND>
__device__ __forceinline__ typename Gather<KIND>::V gather_spans(const Call& c) {
  typename Gather<KIND>::V v = 0;
  for (unsigned i = blockIdx.x; i < c.count; i += gridDim.x) {
    const Span s = c.spans[i];
    if (s.type == EPS_B200_F32) gather_span<KIND, float>(s, v);
    else if (s.type == EPS_B200_BF16) gather_span<KIND, bf16>(s, v);
    else gather_span<KIND, f16>(s, v);
  }
  return block_join<KIND>(v);
}

// The result of the joint value; the factor that gradients take (1 where they stay).
__device__ __forceinline__ float conclude(const Call& c, double raw, bool write) {
  const double u = c.gradient_scale ? (double)*c.gradient_scale : 1.0;
  const double norm = raw * fabs(u);
  EpsB200GradientResult r;
  r.norm = (float)norm;
  r.skip = !(r.norm <= FLT_MAX);
  r.scale = r.skip ? 0.f : (float)(norm > c.max_norm ? u * (c.max_norm / norm) : u);
  if (write && threadIdx.x == 0) *c.result = r;
  return r.skip ? 1.f : r.scale;
}

__device__ __forceinline__ void clip_spans(const Call& c, float scale) {
  if (scale == 1.f) return;               // every gradient is its own product
  // from the last span on: what the sums read last is still in L2
  for (unsigned j = blockIdx.x; j < c.count; j += gridDim.x) {
    const Span s = c.spans[c.count - 1 - j];
    if (s.type == EPS_B200_F32) clip_span<float>(s, scale);
    else if (s.type == EPS_B200_BF16) clip_span<bf16>(s, scale);
    else clip_span<f16>(s, scale);
  }
}

template <int KIND>
__global__ void __launch_bounds__(kThreads, kBlocksEach) gradient_gather(Call c) {
  asm volatile("griddepcontrol.launch_dependents;");
  const auto v = gather_spans<KIND>(c);
  if (threadIdx.x == 0) reinterpret_cast<typename Gather<KIND>::V*>(c.sums)[blockIdx.x] = v;
}

template <int KIND, bool CLIP>
__global__ void __launch_bounds__(kThreads, kBlocksEach) gradient_finish(Call c, unsigned sums) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  typename Gather<KIND>::V v = 0;
  for (unsigned i = threadIdx.x; i < sums; i += blockDim.x)
    v = Gather<KIND>::join(v, reinterpret_cast<const typename Gather<KIND>::V*>(c.sums)[i]);
  const float scale = conclude(c, Gather<KIND>::norm(block_join<KIND>(v)), blockIdx.x == 0);
  if constexpr (CLIP) clip_spans(c, scale);
}

// Few spans: one cluster, whose blocks read each other's values, in one launch.  That takes
// the GPU 4.2 us for 8 spans and 4.5 for 16, against 3.2 and 3.4 in two launches, and the
// host 11 us a call against 16, however many they are.  A call takes as long as the host
// there; at 32 spans (5.9 us of the GPU against 3.4) the GPU's loss is half of the host's
// gain, and it grows with the spans.
constexpr unsigned kCluster = 8, kClusterThreads = 1024, kClusterSpans = 16;
template <int KIND, bool CLIP>
__global__ void __cluster_dims__(kCluster) __launch_bounds__(kClusterThreads) gradient_few(Call c) {
  using V = typename Gather<KIND>::V;
  __shared__ V mine;
  const V v = gather_spans<KIND>(c);
  if (threadIdx.x == 0) mine = v;
  cluster_sync();
  V all = 0;
#pragma unroll
  for (unsigned r = 0; r < kCluster; ++r) all = Gather<KIND>::join(all, cluster_load(&mine, r));
  cluster_sync();                        // no block leaves while another reads from it
  const float scale = conclude(c, Gather<KIND>::norm(all), blockIdx.x == 0);
  if constexpr (CLIP) clip_spans(c, scale);
}

template <int KIND, bool CLIP>
void launch(const Call& c, int device, cudaStream_t stream) {
  if (c.count <= kClusterSpans) {
    gradient_few<KIND, CLIP><<<kCluster, kClusterThreads, 0, stream>>>(c);
    check(cudaGetLastError(), "gradient_few");
    return;
  }
  const unsigned most = std::min(sm_count(device) * kBlocksEach, kMost), grid = std::min(c.count, most);
  gradient_gather<KIND><<<grid, kThreads, 0, stream>>>(c);
  check(cudaGetLastError(), "gradient_gather");
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = CLIP ? grid : 1;
  config.blockDim = kThreads;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  check(cudaLaunchKernelEx(&config, gradient_finish<KIND, CLIP>, c, grid), "gradient_finish");
}

// Elements of the spans of a tensor: the first takes what lies before the first aligned
// address too.
struct Cut {
  uint64_t first, each;
  explicit Cut(const EpsB200Gradient& t) {
    const uint64_t size = size_of(t.type);
    each = kSpan / size;
    first = each + (16 - reinterpret_cast<uintptr_t>(t.gradient) % 16) % 16 / size;
  }
  uint64_t count(uint64_t n) const { return !n ? 0 : n <= first ? 1 : 1 + ceil_div(n - first, each); }
};

uint64_t spans_of(const EpsB200Gradient* t, uint64_t count) {
  uint64_t n = 0;
  for (uint64_t i = 0; i < count; ++i)
    if (known_type(t[i].type)) n += Cut(t[i]).count(t[i].elements);
  return n;
}

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_gradient_norm_plan_bytes(const EpsB200Gradient* tensors, uint64_t count) {
  return tensors ? spans_of(tensors, count) * sizeof(Span) : 0;
}

int eps_b200_gradient_norm_plan(const EpsB200Gradient* tensors, uint64_t count, void* plan, uint64_t plan_bytes,
                                uint64_t* blocks_out, EpsB200Status* status) {
  return guard(status, [&] {
    need(tensors && blocks_out && count, "null gradient plan argument");
    std::vector<std::pair<uintptr_t, uintptr_t>> places;
    for (uint64_t i = 0; i < count; ++i) {
      const EpsB200Gradient& t = tensors[i];
      need(known_type(t.type), "unknown element type");
      need(t.elements < (1ull << 44), "too many elements");
      if (!t.elements) continue;
      const uintptr_t a = reinterpret_cast<uintptr_t>(t.gradient);
      need(a, "null gradient");
      need(a % size_of(t.type) == 0, "a gradient is not aligned to its type");
      need(a + t.elements * size_of(t.type) > a, "a gradient ends behind the last address");
      places.emplace_back(a, a + t.elements * size_of(t.type));
    }
    std::sort(places.begin(), places.end());
    for (size_t i = 1; i < places.size(); ++i) need(places[i - 1].second <= places[i].first, "gradients overlap");
    const uint64_t spans = spans_of(tensors, count);
    need(spans < (1ull << 31), "too many elements for one norm");
    need(plan_bytes >= spans * sizeof(Span) && (plan || !spans), "the gradient plan needs more room");
    Span* to = static_cast<Span*>(plan);
    for (uint64_t i = 0; i < count; ++i) {
      const EpsB200Gradient& t = tensors[i];
      const Cut cut(t);
      for (uint64_t at = 0, n; at < t.elements; at += n) {
        n = std::min(at ? cut.each : cut.first, t.elements - at);
        *to++ = Span{static_cast<char*>(t.gradient) + at * size_of(t.type), (uint32_t)n, t.type};
      }
    }
    *blocks_out = spans;
  });
}

uint64_t eps_b200_gradient_norm_workspace(uint64_t blocks) {
  return blocks <= kClusterSpans ? 0 : std::min<uint64_t>(blocks, kMost) * sizeof(double);
}

int eps_b200_gradient_norm(const EpsB200GradientNorm* a, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    need(a && a->result, "null gradient norm argument");
    need(a->kind == EPS_B200_GRADIENT_L2 || a->kind == EPS_B200_GRADIENT_MAX, "unknown norm");
    need(a->clip == 0 || a->clip == 1, "clip is 0 or 1");
    need(a->max_norm >= 0, "max_norm is 0 or more");            // and no NaN
    need(a->blocks < (1ull << 31), "too many elements for one norm");
    need(!a->blocks || (a->plan && aligned(a->plan, 16)), "a plan is 16-byte aligned");
    need(words(a->gradient_scale, a->result), "gradient_scale and result are 4-byte aligned");
    const uint64_t space = eps_b200_gradient_norm_workspace(a->blocks);
    need(!space || (a->workspace && aligned(a->workspace, 8) && a->workspace_bytes >= space), "the norm's workspace is too small");
    // every block reads the factor, after the first launch left its sums and while one block writes the result
    auto apart = [](const void* p, uint64_t n, const void* q, uint64_t m) {
      const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
      return !p || !q || a + n <= b || b + m <= a;
    };
    need(apart(a->gradient_scale, sizeof(float), a->result, sizeof(EpsB200GradientResult)), "gradient_scale is a part of result");
    need(apart(a->gradient_scale, sizeof(float), a->workspace, space), "gradient_scale is a part of the workspace");
    OnDevice on(a->device);
    Call c{static_cast<const Span*>(a->plan), (unsigned)a->blocks, a->gradient_scale, a->max_norm, a->result, static_cast<double*>(a->workspace)};
    const auto s = static_cast<cudaStream_t>(stream);
    if (a->kind == EPS_B200_GRADIENT_L2)
      a->clip ? launch<EPS_B200_GRADIENT_L2, true>(c, a->device, s) : launch<EPS_B200_GRADIENT_L2, false>(c, a->device, s);
    else a->clip ? launch<EPS_B200_GRADIENT_MAX, true>(c, a->device, s) : launch<EPS_B200_GRADIENT_MAX, false>(c, a->device, s);
  });
}

}  // extern "C"
