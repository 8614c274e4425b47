// int8_product.cu -- matrix products in 8-bit integers with a scale for each token
// and channel, rows grouped by expert (eps_b200_int8_quantize, eps_b200_int8_product,
// eps_b200_int8_linear).
//
// Mathematics: q[r, k] = round-half-even(x[r, k] * (127 * (1 / amax_r))), scale_r = amax_r / 127;
//   out[r, n] = (sum_k q[r, k] w[e, n, k]) * (scale_r * weight_scale[e, n]) + bias[e, n]
// with the sum exact in 32-bit integers (inner <= 131072: 127 * 127 * 131072 < 2^31).
#include <cmath>
#include <type_traits>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

struct Quantize {
  const void* x;
  int64_t stride;
  uint64_t x_rows, count;
  unsigned inner, padded, divisor;
  const int32_t* rows;
  int8_t* q;
  float* scale;
  int wide;
};

// One block a row, two passes over it: the largest magnitude, then the values (the
// second read comes from L1 or L2).
template <class T>
__global__ void __launch_bounds__(256) quantize_rows(const Quantize a) {
  __shared__ unsigned tops[8];
  const uint64_t r = blockIdx.x;
  const int64_t from = a.rows ? a.rows[r] / (int64_t)a.divisor : (int64_t)r;
  const bool known = (!a.rows || a.rows[r] >= 0) && (uint64_t)from < a.x_rows;
  const T* const x = static_cast<const T*>(a.x) + (known ? from : 0) * a.stride;
  constexpr int V = 16 / sizeof(T);
  unsigned top = 0;
  if (known) {
    if (a.wide) {
      for (unsigned k = threadIdx.x * V; k < a.inner; k += 256 * V) {
        const Pack<T, V> p = load_pack<T, V>(x + k);
#pragma unroll
        for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(to_float(p.v[j])) & 0x7FFFFFFFu);
      }
    } else {
      for (unsigned k = threadIdx.x; k < a.inner; k += 256) top = max(top, __float_as_uint(to_float(x[k])) & 0x7FFFFFFFu);
    }
  }
  top = __reduce_max_sync(~0u, top);
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, tops[w]);
  const float amax = __uint_as_float(top);
  const bool finite = known && top < 0x7F800000u;
  const float by = finite && amax >= 0x1p-120f ? __fmul_rn(127.f, __fdiv_rn(1.f, amax)) : 0.f;
  if (threadIdx.x == 0) a.scale[r] = !finite ? NAN : by == 0.f ? 0.f : __fdiv_rn(amax, 127.f);
  int8_t* const q = a.q + r * a.padded;
  auto round = [by](float v) { return by == 0.f ? 0 : __float2int_rn(__fmul_rn(v, by)); };
  for (unsigned k = threadIdx.x * 4; k < a.padded; k += 256 * 4) {
    unsigned word = 0;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j)
      if (k + j < a.inner) word |= ((unsigned)round(to_float(x[k + j])) & 0xFFu) << 8 * j;
    *reinterpret_cast<unsigned*>(q + k) = word;
  }
}

struct Product {
  const int8_t *q, *weight;
  const float *scale, *weight_scale, *bias;
  const int32_t* offsets;
  void* out;
  unsigned rows, experts, channels, padded;
};

struct Tile { unsigned expert, row, rows; };   // rows == 0: there is no such tile

// The index-th tile of `tile_rows` rows, expert after expert; called by a whole warp.
__device__ __forceinline__ Tile locate(const Product& a, unsigned tile_rows, unsigned index) {
  if (!a.offsets) {
    const unsigned row = index * tile_rows;
    return {0, row, row < a.rows ? min(tile_rows, a.rows - row) : 0};
  }
  const unsigned lane = threadIdx.x % 32;
  unsigned before = 0;
  for (unsigned e0 = 0; e0 < a.experts; e0 += 32) {
    unsigned begin = 0, end = 0;
    if (e0 + lane < a.experts) {
      begin = (unsigned)min(max(a.offsets[e0 + lane], 0), (int)a.rows);
      end = (unsigned)min(max(a.offsets[e0 + lane + 1], 0), (int)a.rows);
    }
    const unsigned n = end > begin ? (end - begin + tile_rows - 1) / tile_rows : 0;
    unsigned sum = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned up = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += up;
    }
    const unsigned here = __ballot_sync(~0u, index - before < sum);
    if (here) {
      const int owner = __ffs(here) - 1;
      const unsigned row = begin + (index - before - (sum - n)) * tile_rows;
      const unsigned rows = min(tile_rows, end - row);
      return {e0 + owner, __shfl_sync(~0u, row, owner), __shfl_sync(~0u, rows, owner)};
    }
    before += __shfl_sync(~0u, sum, 31);
  }
  return {0, 0, 0};
}

// A warp a channel, RT rows at once, the weights streamed past them.
template <class T, int RT>
__global__ void __launch_bounds__(256) product_rows(const Product a, unsigned channel_blocks) {
  const unsigned lane = threadIdx.x % 32;
  const Tile t = locate(a, RT, blockIdx.x / channel_blocks);
  const unsigned n = blockIdx.x % channel_blocks * 8 + threadIdx.x / 32;
  if (!t.rows || n >= a.channels) return;
  const int8_t* const w = a.weight + ((uint64_t)t.expert * a.channels + n) * a.padded;
  const int8_t* const q = a.q + (uint64_t)t.row * a.padded;
  int acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = 0;
  for (unsigned k = lane * 16; k < a.padded; k += 512) {
    const int4 x = *reinterpret_cast<const int4*>(w + k);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (r >= t.rows) continue;
      const int4 y = *reinterpret_cast<const int4*>(q + (uint64_t)r * a.padded + k);
      acc[r] = __dp4a(x.x, y.x, __dp4a(x.y, y.y, __dp4a(x.z, y.z, __dp4a(x.w, y.w, acc[r]))));
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int sum = __reduce_add_sync(~0u, acc[r]);
    if (lane == r && r < t.rows) {
      const uint64_t c = (uint64_t)t.expert * a.channels + n;
      float v = (float)sum * (a.scale[t.row + r] * a.weight_scale[c]);
      if (a.bias) v += a.bias[c];
      static_cast<T*>(a.out)[(uint64_t)(t.row + r) * a.channels + n] = from_float<T>(v);
    }
  }
}

template <class F>
void by_type(int type, F f) {
  if (type == EPS_B200_F32) f(float{});
  else if (type == EPS_B200_BF16) f(bf16{});
  else f(f16{});
}

void quantize(int type, const Quantize& a, cudaStream_t stream) {
  need(a.count < (1ull << 31), "too many rows");
  by_type(type, [&](auto t) { quantize_rows<decltype(t)><<<(unsigned)a.count, 256, 0, stream>>>(a); });
  check(cudaGetLastError(), "int8_quantize");
}

void product(int type, const Product& a, cudaStream_t stream) {
  const unsigned channel_blocks = (unsigned)ceil_div(a.channels, 8);
  const uint64_t tiles = ceil_div(a.rows, 8) + (a.offsets ? a.experts - 1 : 0);
  need(tiles * channel_blocks < (1ull << 31), "too many rows");
  by_type(type, [&](auto t) {
    product_rows<decltype(t), 8><<<(unsigned)(tiles * channel_blocks), 256, 0, stream>>>(a, channel_blocks);
  });
  check(cudaGetLastError(), "int8_product");
}

Quantize quantize_args(int type, const void* x, int64_t x_stride, uint64_t x_rows, unsigned inner, const int32_t* rows,
                       unsigned divisor, uint64_t count, int8_t* q, float* scale) {
  need(known_type(type), "unknown element type");
  need(inner > 0 && inner <= EPS_B200_INT8_INNER, "inner size out of range");
  need(rows ? divisor > 0 : count <= x_rows, "more rows than x has");
  need(!count || (q && scale && (x || !x_rows)), "null input or output");
  need(aligned(q, 16), "q must be 16-byte aligned");
  return Quantize{x, x_stride, x_rows, count, inner, (unsigned)eps_b200_int8_stride(inner), divisor, rows, q, scale,
                  aligned(x, 16) && x_stride * (int64_t)size_of(type) % 16 == 0 && inner * size_of(type) % 16 == 0};
}

Product product_args(const EpsB200Int8Product* a) {
  need(a, "null product arguments");
  need(known_type(a->type), "unknown element type");
  need(a->experts > 0 && a->experts < (1u << 20) && a->channels > 0 && a->channels < (1u << 28), "experts or channels out of range");
  need(a->inner > 0 && a->inner <= EPS_B200_INT8_INNER, "inner size out of range");
  need(a->rows < (1ull << 31), "too many rows");
  need(a->offsets || a->experts == 1, "several experts need offsets");
  need(a->weight && a->weight_scale && (a->out || !a->rows), "null weight or output");
  need(aligned(a->weight, 16) && aligned(a->out, 16) && aligned(a->workspace, 16), "weight, out and workspace must be 16-byte aligned");
  Product p{};
  p.weight = a->weight;
  p.weight_scale = a->weight_scale;
  p.bias = a->bias;
  p.offsets = a->offsets;
  p.out = a->out;
  p.rows = (unsigned)a->rows;
  p.experts = a->experts;
  p.channels = a->channels;
  p.padded = (unsigned)eps_b200_int8_stride(a->inner);
  return p;
}

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_int8_stride(uint32_t inner) { return round_up(inner, 16); }

int eps_b200_int8_quantize(int32_t device, int32_t type, const void* x, int64_t x_stride, uint64_t x_rows,
                           uint32_t inner, const int32_t* rows, uint32_t rows_divisor, uint64_t count, int8_t* q,
                           float* scale, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    const Quantize a = quantize_args(type, x, x_stride, x_rows, inner, rows, rows_divisor, count, q, scale);
    if (!count) return;
    OnDevice on(device);
    quantize(type, a, static_cast<cudaStream_t>(stream));
  });
}

uint64_t eps_b200_int8_product_workspace(uint64_t rows, uint32_t experts, uint32_t channels, uint32_t inner) {
  (void)experts;
  (void)channels;
  return rows * eps_b200_int8_stride(inner) + round_up(rows * 4, 16);
}

int eps_b200_int8_product(const EpsB200Int8Product* a, const int8_t* q, const float* scale, void* stream,
                          EpsB200Status* status) {
  return guard(status, [&] {
    Product p = product_args(a);
    need(!p.rows || (q && scale), "null input");
    need(aligned(q, 16), "q must be 16-byte aligned");
    if (!p.rows) return;
    p.q = q;
    p.scale = scale;
    OnDevice on(a->device);
    product(a->type, p, static_cast<cudaStream_t>(stream));
  });
}

int eps_b200_int8_linear(const EpsB200Int8Product* a, const void* x, int64_t x_stride, uint64_t x_rows,
                         const int32_t* rows, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Product p = product_args(a);
    if (!p.rows) return;
    need(a->workspace && a->workspace_bytes >= eps_b200_int8_product_workspace(a->rows, a->experts, a->channels, a->inner),
         "int8 workspace too small");
    auto* q = static_cast<int8_t*>(a->workspace);
    auto* scale = reinterpret_cast<float*>(q + (uint64_t)p.rows * p.padded);
    const Quantize z = quantize_args(a->type, x, x_stride, x_rows, a->inner, rows, a->rows_divisor, a->rows, q, scale);
    p.q = q;
    p.scale = scale;
    OnDevice on(a->device);
    const auto st = static_cast<cudaStream_t>(stream);
    quantize(a->type, z, st);
    product(a->type, p, st);
  });
}

}  // extern "C"
