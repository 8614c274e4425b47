// int8_product.cu -- matrix products in 8-bit integers with a scale for each token
// and channel, rows grouped by expert (eps_b200_int8_quantize, eps_b200_int8_product,
// eps_b200_int8_linear).
//
// Mathematics: q[r, k] = round-half-even(x[r, k] * (127 * (1 / amax_r))), scale_r = amax_r / 127;
//   out[r, n] = (sum_k q[r, k] w[e, n, k]) * (scale_r * weight_scale[e, n]) + bias[e, n]
// with the sum exact in 32-bit integers (inner <= 131072: 127 * 127 * 131072 < 2^31).
#include <cuda.h>

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

// ------------------------------------------------ the tensor cores' product
//
// A tile is 128 channels x BN rows of one expert: D[channel, row] = W q^T, so the
// channels lie on the lanes of tensor memory and a store of a warp covers 32
// neighbouring channels of one output row.  Both operands are K-major int8, 128
// bytes of inner size a stage, brought by TMA with the 128-byte swizzle that the
// matrix instruction reads; out-of-range rows and bytes arrive as zeros, and rows of
// the next expert or channel group, which a ragged tile also covers, are not stored.
//
// One block an SM walks the tiles: warp 0 fills the stages, warp 1 issues
// tcgen05.mma (kind::i8, 32-bit sums in tensor memory), warps 4..7 scale, round and
// store the tile before while the next is being summed (two halves of tensor memory).
constexpr int kMmaThreads = 256;
constexpr unsigned kStageK = 128;          // bytes of inner size a stage
constexpr unsigned kTileM = 128;           // channels of a tile

template <int BN>
struct MmaShape {
  static constexpr unsigned stage_bytes = (kTileM + BN) * kStageK;
  static constexpr unsigned stages = 196608 / stage_bytes < 8 ? 196608 / stage_bytes : 8;
  static constexpr unsigned shared = stages * stage_bytes + 1024;      // and room to align
  static constexpr unsigned columns = 2 * BN;                          // of tensor memory
};

__device__ __forceinline__ void tma_load(void* to, const CUtensorMap* map, uint64_t* barrier, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(shared_at(to)), "l"(map), "r"(shared_at(barrier)), "r"(x), "r"(y) : "memory");
}

// Shared-memory descriptor of a K-major operand in the 128-byte swizzle: rows of 128
// bytes, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(const void* p) {
  return (uint64_t)(shared_at(p) >> 4 & 0x3FFF) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

template <int BN>
__device__ __forceinline__ void mma_i8(unsigned d, uint64_t a, uint64_t b, bool accumulate) {
  // 32-bit signed sums, signed 8-bit operands, both K-major, N = BN, M = 128
  constexpr unsigned shape = 2u << 4 | 1u << 7 | 1u << 10 | (unsigned)(BN / 8) << 17 | (kTileM / 16) << 24;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((unsigned)accumulate) : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t* barrier) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_at(barrier)) : "memory");
}

// 32 lanes x 32 columns of tensor memory: lane l of the warp gets its 32 columns.
__device__ __forceinline__ void tensor_load(unsigned address, int (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(address));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <class T, int BN>
__global__ void __launch_bounds__(kMmaThreads, 1)
    product_tiles(const Product a, const __grid_constant__ CUtensorMap weights, const __grid_constant__ CUtensorMap rows,
                  unsigned channel_tiles) {
  using Shape = MmaShape<BN>;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[Shape::stages], empty[Shape::stages], summed[2], drained[2];
  __shared__ unsigned tensor_base;
  unsigned char* const stages = raw + (1024 - shared_at(raw) % 1024) % 1024;
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (unsigned s = 0; s < Shape::stages; ++s) {
      barrier_init(full + s, 1);
      barrier_init(empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(summed + s, 1);
      barrier_init(drained + s, 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&weights) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&rows) : "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_at(&tensor_base)),
                 "r"(Shape::columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned base = tensor_base;
  const unsigned steps = (a.padded + kStageK - 1) / kStageK;

  if (warp == 0) {
    unsigned stage = 0, phase = 0, filled = 0;
    bool ok = true;
    for (unsigned t = blockIdx.x; ok; t += gridDim.x) {
      const Tile tile = locate(a, BN, t / channel_tiles);
      if (!tile.rows) break;
      if (lane == 0) {
        const int y = (int)(tile.expert * a.channels + t % channel_tiles * kTileM);
        for (unsigned k = 0; k < steps; ++k) {
          if (!(ok = barrier_wait(empty + stage, phase ^ 1))) break;
          unsigned char* const p = stages + stage * Shape::stage_bytes;
          barrier_expect(full + stage, Shape::stage_bytes);
          tma_load(p, &weights, full + stage, (int)(k * kStageK), y);
          tma_load(p + kTileM * kStageK, &rows, full + stage, (int)(k * kStageK), (int)tile.row);
          if (++filled > Shape::stages) filled = Shape::stages;
          if (++stage == Shape::stages) { stage = 0; phase ^= 1; }
        }
      }
      ok = __shfl_sync(~0u, ok, 0);
    }
    // no block ends with copies into its shared memory in flight
    if (lane == 0 && !ok)
      for (unsigned n = 0; n < filled; ++n) {
        stage = stage ? stage - 1 : Shape::stages - 1;
        if (stage == Shape::stages - 1) phase ^= 1;
        barrier_wait(full + stage, phase);
      }
  } else if (warp == 1) {
    unsigned stage = 0, phase = 0, half = 0, turn = 0;
    bool ok = true;
    for (unsigned t = blockIdx.x; ok; t += gridDim.x) {
      if (!locate(a, BN, t / channel_tiles).rows) break;
      if (lane == 0) {
        ok = barrier_wait(drained + half, turn ^ 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (unsigned k = 0; ok && k < steps; ++k) {
          if (!(ok = barrier_wait(full + stage, phase))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned char* const p = stages + stage * Shape::stage_bytes;
          const uint64_t w = operand(p), q = operand(p + kTileM * kStageK);
#pragma unroll
          for (unsigned i = 0; i < kStageK / 32; ++i) mma_i8<BN>(base + half * BN, w + 2 * i, q + 2 * i, k || i);
          mma_commit(empty + stage);
          if (++stage == Shape::stages) { stage = 0; phase ^= 1; }
        }
        if (ok) mma_commit(summed + half);
      }
      ok = __shfl_sync(~0u, ok, 0);
      half ^= 1;
      turn ^= half == 0;
    }
  } else if (warp >= 4) {
    unsigned half = 0, turn = 0;
    bool ok = true;
    for (unsigned t = blockIdx.x; ok; t += gridDim.x) {
      const Tile tile = locate(a, BN, t / channel_tiles);
      if (!tile.rows) break;
      const unsigned n = t % channel_tiles * kTileM + (warp - 4) * 32 + lane;
      const uint64_t c = (uint64_t)tile.expert * a.channels + n;
      const bool in = n < a.channels;
      const float ws = in ? a.weight_scale[c] : 0.f, b = in && a.bias ? a.bias[c] : 0.f;
      ok = __all_sync(~0u, barrier_wait(summed + half, turn));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      T* const out = static_cast<T*>(a.out) + (uint64_t)tile.row * a.channels + n;
#pragma unroll 1
      for (unsigned r0 = 0; r0 < tile.rows; r0 += 32) {
        int v[32];
        tensor_load(base + half * BN + r0 + ((warp - 4) * 32 << 16), v);
        const float mine = r0 + lane < tile.rows ? a.scale[tile.row + r0 + lane] : 0.f;
#pragma unroll
        for (unsigned j = 0; j < 32; ++j) {
          const float s = __shfl_sync(~0u, mine, j);
          const float value = ok ? fmaf((float)v[j], s * ws, b) : NAN;
          if (in && r0 + j < tile.rows) out[(uint64_t)(r0 + j) * a.channels] = from_float<T>(value);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(drained + half);
      half ^= 1;
      turn ^= half == 0;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(Shape::columns) : "memory");
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

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, asked for once.
Encode encoder() {
  static const Encode found = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!found) throw Fail(EPS_B200_UNAVAILABLE, "the driver offers no cuTensorMapEncodeTiled");
  return found;
}

// A matrix of `rows` rows of `padded` bytes in boxes of box_rows x 128 bytes.
CUtensorMap tensor_map(const void* p, uint64_t rows, unsigned padded, unsigned box_rows) {
  CUtensorMap m;
  const cuuint64_t dims[2] = {padded, rows}, strides[1] = {padded};
  const cuuint32_t box[2] = {kStageK, box_rows}, step[2] = {1, 1};
  const CUresult r = encoder()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, step,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Fail(EPS_B200_RUN_FAILED, "cuTensorMapEncodeTiled failed");
  return m;
}

// Upper bound of the tiles of `tile_rows` rows that the groups make.
uint64_t tile_bound(const Product& a, unsigned tile_rows) {
  const uint64_t extra = a.offsets ? (a.experts < a.rows ? a.experts : a.rows) - 1 : 0;
  return ceil_div(a.rows, tile_rows) + extra;
}

template <int BN>
void tiles(int type, const Product& a, unsigned sms, cudaStream_t stream) {
  using Shape = MmaShape<BN>;
  const CUtensorMap w = tensor_map(a.weight, (uint64_t)a.experts * a.channels, a.padded, kTileM);
  const CUtensorMap q = tensor_map(a.q, a.rows, a.padded, BN);
  const unsigned channel_tiles = (unsigned)ceil_div(a.channels, kTileM);
  const uint64_t most = tile_bound(a, BN) * channel_tiles;
  need(most < (1ull << 31), "too many rows");
  by_type(type, [&](auto t) {
    auto* kernel = product_tiles<decltype(t), BN>;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape::shared), "cudaFuncSetAttribute");
    kernel<<<(unsigned)(most < sms ? most : sms), kMmaThreads, Shape::shared, stream>>>(a, w, q, channel_tiles);
  });
  check(cudaGetLastError(), "int8_product");
}

void product(int type, const Product& a, unsigned sms, cudaStream_t stream) {
  const uint64_t each = ceil_div(a.rows, a.experts);      // rows of an expert, on average
  if (a.rows > 8 && each > 2) {
    need((uint64_t)a.experts * a.channels < (1ull << 31), "too many channels");
    if (each > 128) tiles<256>(type, a, sms, stream);
    else if (each > 64) tiles<128>(type, a, sms, stream);
    else if (each > 32) tiles<64>(type, a, sms, stream);
    else tiles<32>(type, a, sms, stream);
    return;
  }
  const unsigned channel_blocks = (unsigned)ceil_div(a.channels, 8);
  const uint64_t most = tile_bound(a, 8) * channel_blocks;
  need(most < (1ull << 31), "too many rows");
  by_type(type, [&](auto t) { product_rows<decltype(t), 8><<<(unsigned)most, 256, 0, stream>>>(a, channel_blocks); });
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
    product(a->type, p, sm_count(a->device), static_cast<cudaStream_t>(stream));
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
    product(a->type, p, sm_count(a->device), st);
  });
}

}  // extern "C"
