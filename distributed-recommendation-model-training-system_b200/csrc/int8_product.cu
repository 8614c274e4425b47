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

// The factor and the scale of a row whose largest magnitude has these bits.
__device__ __forceinline__ void factors(unsigned top, bool known, float* by, float* scale) {
  const float amax = __uint_as_float(top);
  const bool finite = known && top < 0x7F800000u;
  *by = finite && amax >= 0x1p-120f ? __fmul_rn(127.f, __fdiv_rn(1.f, amax)) : 0.f;
  *scale = !finite ? NAN : *by == 0.f ? 0.f : __fdiv_rn(amax, 127.f);
}

// by == 0: nothing but zeros comes out, also of NaN and infinity.
__device__ __forceinline__ unsigned quantized(float v, float by) {
  return by == 0.f ? 0u : (unsigned)__float2int_rn(__fmul_rn(v, by)) & 0xFFu;
}

// Row r's place in x; `known` is false where `rows` points outside.
template <class T>
__device__ __forceinline__ const T* source_row(const Quantize& a, uint64_t r, bool* known) {
  const int64_t index = a.rows ? a.rows[r] : (int64_t)r, from = a.rows ? index / (int64_t)a.divisor : index;
  *known = index >= 0 && (uint64_t)from < a.x_rows;
  return static_cast<const T*>(a.x) + (*known ? from : 0) * a.stride;
}

// A block a row.  Rows of up to NIT packs of 16 bytes a thread stay in registers
// between the search for the largest magnitude and the rounding: one pass over memory,
// which is what bounds it (8189 x 4096 bf16: 19 us, 5.3 TB/s; 33 when rows were read
// twice).  NIT == 0 reads a row of any kind twice.
constexpr unsigned kQuantizeThreads = 128;
template <class T, int NIT>
__global__ void __launch_bounds__(kQuantizeThreads) quantize_rows(const Quantize a) {
  __shared__ unsigned tops[kQuantizeThreads / 32];
  constexpr int V = 16 / sizeof(T), kHeld = NIT ? NIT : 1;
  const uint64_t r = blockIdx.x;
  bool known;
  const T* const x = source_row<T>(a, r, &known);
  unsigned top = 0;
  auto look = [&](float v) { top = max(top, __float_as_uint(v) & 0x7FFFFFFFu); };
  Pack<T, V> held[kHeld];
  if constexpr (NIT > 0) {
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const unsigned k = (i * kQuantizeThreads + threadIdx.x) * V;
      held[i] = Pack<T, V>{};
      if (known && k < a.inner) held[i] = load_once<T, V>(x + k);
    }
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float v[V];
      widen(held[i], v);
#pragma unroll
      for (int j = 0; j < V; ++j) look(v[j]);
    }
  } else if (known) {
    for (unsigned k = threadIdx.x; k < a.inner; k += kQuantizeThreads) look(to_float(x[k]));
  }
  top = __reduce_max_sync(~0u, top);
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (unsigned w = 0; w < kQuantizeThreads / 32; ++w) top = max(top, tops[w]);
  float by, scale;
  factors(top, known, &by, &scale);
  if (threadIdx.x == 0) a.scale[r] = scale;
  int8_t* const q = a.q + r * a.padded;
  if constexpr (NIT > 0) {
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const unsigned k = (i * kQuantizeThreads + threadIdx.x) * V;
      if (k >= a.padded) continue;           // behind `inner` the packs hold zeros
      float v[V];
      widen(held[i], v);
      unsigned words[V / 4];
#pragma unroll
      for (int w = 0; w < V / 4; ++w)
        words[w] = quantized(v[4 * w], by) | quantized(v[4 * w + 1], by) << 8 | quantized(v[4 * w + 2], by) << 16 | quantized(v[4 * w + 3], by) << 24;
      if constexpr (V == 8) *reinterpret_cast<uint2*>(q + k) = make_uint2(words[0], words[1]);
      else *reinterpret_cast<unsigned*>(q + k) = words[0];
    }
  } else {
    for (unsigned k = threadIdx.x * 4; k < a.padded; k += kQuantizeThreads * 4) {
      unsigned word = 0;
#pragma unroll
      for (unsigned j = 0; j < 4; ++j)
        if (k + j < a.inner) word |= quantized(to_float(x[k + j]), by) << 8 * j;
      *reinterpret_cast<unsigned*>(q + k) = word;
    }
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

// Expert e's run of rows, clamped to what there is.
__device__ __forceinline__ void run_of(const Product& a, unsigned e, unsigned* begin, unsigned* end) {
  *begin = (unsigned)min(max(a.offsets[e], 0), (int)a.rows);
  *end = (unsigned)min(max(a.offsets[e + 1], 0), (int)a.rows);
}

__device__ __forceinline__ unsigned tiles_of(const Product& a, unsigned e, unsigned tile_rows) {
  unsigned begin, end;
  run_of(a, e, &begin, &end);
  return end > begin ? (end - begin + tile_rows - 1) / tile_rows : 0;
}

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
    if (e0 + lane < a.experts) run_of(a, e0 + lane, &begin, &end);
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

// Few rows: the weights' bytes are all there is.  A warp has a channel, asks for its
// first weights, and while they come the block quantizes its RT rows into shared
// memory for all its warps (every block does that again: the rows are a few kilobytes
// in L2, and a launch before this one would take longer).  1 x 4096 x 4096 takes 8.9 us,
// 13 with a launch of its own to quantize, against a floor of 2.6: what is left is the
// wait for the row before anything can be summed.
constexpr unsigned kRowsThreads = 512, kRowsAhead = 8;
template <class T, int RT, bool QUANTIZE>
__global__ void __launch_bounds__(kRowsThreads) product_rows(const Product a, const Quantize z, unsigned channel_blocks) {
  extern __shared__ __align__(16) int8_t staged[];      // QUANTIZE: [RT][padded]
  __shared__ unsigned tops[kRowsThreads / 32];
  __shared__ float scales[RT];
  constexpr int kV = 16 / sizeof(T);
  const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Tile t = locate(a, RT, blockIdx.x / channel_blocks);
  if (!t.rows) return;
  const unsigned n = blockIdx.x % channel_blocks * (kRowsThreads / 32) + warp;
  const bool in = n < a.channels;
  const int8_t* const w = a.weight + ((uint64_t)t.expert * a.channels + (in ? n : 0)) * a.padded;
  int4 ahead[kRowsAhead];
#pragma unroll
  for (unsigned i = 0; i < kRowsAhead; ++i) {
    const unsigned k = (i * 32 + lane) * 16;
    ahead[i] = make_int4(0, 0, 0, 0);
    if (in && k < a.padded) ahead[i] = __ldcs(reinterpret_cast<const int4*>(w + k));
  }
  float scale[RT];
  if constexpr (QUANTIZE) {
    // the block's warps share the rows: all rows are read at once
    constexpr unsigned kEach = kRowsThreads / RT;
    const unsigned r = threadIdx.x / kEach, thread = threadIdx.x % kEach;
    bool known = false;
    const T* const x = r < t.rows ? source_row<T>(z, t.row + r, &known) : nullptr;
    unsigned top = 0;
    if (known && z.wide) {
#pragma unroll 4
      for (unsigned k = thread * kV; k < z.inner; k += kEach * kV) {
        float v[kV];
        widen(load_pack<T, kV>(x + k), v);
#pragma unroll
        for (int j = 0; j < kV; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      }
    } else if (known) {
#pragma unroll 4
      for (unsigned k = thread; k < z.inner; k += kEach) top = max(top, __float_as_uint(to_float(x[k])) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(~0u, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (unsigned i = 0; i < kEach / 32; ++i) top = max(top, tops[r * (kEach / 32) + i]);
    float by, mine;
    factors(top, known, &by, &mine);
    if (thread == 0) scales[r] = mine;
    int8_t* const s = staged + r * a.padded;
    if (known && z.wide) {
      for (unsigned k = thread * kV; k < a.padded; k += kEach * kV) {
        float v[kV] = {};
        if (k < z.inner) widen(load_pack<T, kV>(x + k), v);
#pragma unroll
        for (int j = 0; j < kV; j += 4)
          *reinterpret_cast<unsigned*>(s + k + j) =
              quantized(v[j], by) | quantized(v[j + 1], by) << 8 | quantized(v[j + 2], by) << 16 | quantized(v[j + 3], by) << 24;
      }
    } else if (r < t.rows) {
      for (unsigned k = thread; k < a.padded; k += kEach) s[k] = known && k < z.inner ? (int8_t)quantized(to_float(x[k]), by) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i) scale[i] = scales[i];
  } else {
#pragma unroll
    for (int r = 0; r < RT; ++r) scale[r] = r < t.rows ? a.scale[t.row + r] : 0.f;
  }
  if (!in) return;
  const int8_t* const q = QUANTIZE ? staged : a.q + (uint64_t)t.row * a.padded;
  int acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = 0;
  for (unsigned k0 = 0; k0 < a.padded; k0 += kRowsAhead * 512) {
#pragma unroll
    for (unsigned i = 0; i < kRowsAhead; ++i) {
      const unsigned k = k0 + (i * 32 + lane) * 16;
      if (k >= a.padded) break;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r >= t.rows) continue;
        const int4 y = *reinterpret_cast<const int4*>(q + (uint64_t)r * a.padded + k);
        acc[r] = __dp4a(ahead[i].x, y.x, __dp4a(ahead[i].y, y.y, __dp4a(ahead[i].z, y.z, __dp4a(ahead[i].w, y.w, acc[r]))));
      }
      const unsigned next = k + kRowsAhead * 512;
      if (next < a.padded) ahead[i] = __ldcs(reinterpret_cast<const int4*>(w + next));
    }
  }
  const uint64_t c = (uint64_t)t.expert * a.channels + n;
  const float ws = a.weight_scale[c], b = a.bias ? a.bias[c] : 0.f;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int sum = __reduce_add_sync(~0u, acc[r]);
    if (lane == 0 && r < t.rows)
      static_cast<T*>(a.out)[(uint64_t)(t.row + r) * a.channels + n] = from_float<T>(fmaf((float)sum, scale[r] * ws, b));
  }
}

// ------------------------------------------------ the tensor cores' product
//
// A tile is 128 channels x BN rows of one expert: D[channel, row] = W q^T, so the
// channels lie on the lanes of tensor memory and a store of a warp covers 32
// neighbouring channels of one output row.  Both operands are K-major int8, brought by
// TMA in spans of 128 bytes of inner size with the 128-byte swizzle that the matrix
// instruction reads; a stage is one span, or two for tiles of up to 128 rows, since a
// stage's hand-over between the warps takes as long (some 430 cycles) whatever it holds
// (200 rows x 4096 x 4096: 15.6 us with one span a stage, 14.2 with two, 15.5 with four,
// which leave too few stages);
// out-of-range rows and bytes arrive as zeros, and rows of
// the next expert or channel group, which a ragged tile also covers, are not stored.
//
// One block an SM walks the tiles: warp 0 fills the stages, warp 1 issues
// tcgen05.mma (kind::i8, 32-bit sums in tensor memory), warps 4..11 scale, round and
// store the tile before while the next is being summed (two halves of tensor memory).
//
// What bounds it: a large product (8189 x 8192 x 4096: 175 us alone, 3.15e15 operations a
// second; some 220 one after another, where the power cap holds it) by the hand-over of its stages and by what the SMs bring in, 48 KB for every
// 512 cycles of matrix instructions, 18 TB/s over the GPU out of L2; a pair of SMs on one
// tile would take a third off that.  Four warps storing instead of eight took 225 us (and eight 179):
// the next tile but one waited for them.
constexpr int kMmaThreads = 384;            // four warps that feed, eight that store
constexpr unsigned kSpan = 128;            // bytes of inner size that one swizzled copy covers
constexpr unsigned kTileM = 128;           // channels of a tile

template <int BN>
struct MmaShape {
  static constexpr unsigned spans = BN < 256 ? 2 : 1;                  // of a stage: see above
  static constexpr unsigned span_bytes = (kTileM + BN) * kSpan;        // of both operands
  static constexpr unsigned stage_bytes = spans * span_bytes;
  static constexpr unsigned stages = 196608 / stage_bytes < 8 ? 196608 / stage_bytes : 8;
  static constexpr unsigned shared = stages * stage_bytes + 1024;      // and room to align
  static constexpr unsigned columns = 2 * BN;                          // of tensor memory
};

// The same for a whole warp, which stays together.
// `b` is a shared address.
__device__ __forceinline__ bool warp_wait(unsigned b, unsigned parity) {
  uint64_t start = 0;
  for (unsigned tries = 1;; ++tries) {
    unsigned done;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(b), "r"(parity) : "memory");
    if (__all_sync(~0u, done)) return true;
    if (tries % 256 == 0) {
      const uint64_t now = nanoseconds();
      if (!start) start = now;
      else if (__any_sync(~0u, now - start > 2000000000ull)) return false;
    }
  }
}

// One lane of a warp that is together, always the same.
__device__ __forceinline__ bool elected() {
  unsigned one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one;
}

__device__ __forceinline__ void expect(unsigned barrier, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}

__device__ __forceinline__ void tma_load(unsigned to, const CUtensorMap* map, unsigned barrier, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(to), "l"(map), "r"(barrier), "r"(x), "r"(y) : "memory");
}

// Shared-memory descriptor of a K-major operand in the 128-byte swizzle: rows of 128
// bytes, groups of eight rows 1024 bytes apart.  Its upper word is a constant, its
// lower one moves with the address; kept apart they stay in uniform registers.
constexpr unsigned kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ unsigned operand_low(unsigned address) { return (address >> 4 & 0x3FFF) | 1u << 16; }

template <int BN>
__device__ __forceinline__ void mma_i8(unsigned d, unsigned a, unsigned b, bool accumulate) {
  // 32-bit signed sums, signed 8-bit operands, both K-major, N = BN, M = 128
  constexpr unsigned shape = 2u << 4 | 1u << 7 | 1u << 10 | (unsigned)(BN / 8) << 17 | (kTileM / 16) << 24;
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, p;\n}\n"
      ::"r"(d), "r"(a), "r"(b), "r"(shape), "r"((unsigned)accumulate), "r"(kOperandHigh) : "memory");
}

__device__ __forceinline__ void mma_commit(unsigned barrier) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
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

// The groups' tiles, counted once a block: `locate` reads offsets from memory for every
// tile, some thousand cycles in each of a block's roles, and this one a few words of
// shared memory.
constexpr unsigned kListed = 256;           // experts that are listed; more are located in memory
struct Groups {
  unsigned last[kListed];                   // tiles up to and with this expert
  unsigned begin[kListed], end[kListed];    // its rows
};

// By one whole warp, before a barrier of the block.
__device__ __forceinline__ void list_groups(const Product& a, unsigned tile_rows, Groups& g) {
  const unsigned lane = threadIdx.x % 32;
  unsigned before = 0;
  if (!a.offsets || a.experts > kListed) return;
  for (unsigned e0 = 0; e0 < a.experts; e0 += 32) {
    const unsigned e = e0 + lane;
    unsigned begin = 0, end = 0;
    if (e < a.experts) run_of(a, e, &begin, &end);
    unsigned sum = end > begin ? (end - begin + tile_rows - 1) / tile_rows : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned up = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += up;
    }
    if (e < a.experts) {
      g.last[e] = before + sum;
      g.begin[e] = begin;
      g.end[e] = end;
    }
    before += __shfl_sync(~0u, sum, 31);
  }
}

// As `locate`, with the groups listed.
__device__ __forceinline__ Tile look_up(const Product& a, const Groups& g, unsigned tile_rows, unsigned index) {
  if (!a.offsets || a.experts > kListed) return locate(a, tile_rows, index);
  const unsigned lane = threadIdx.x % 32;
  for (unsigned e0 = 0; e0 < a.experts; e0 += 32) {
    const unsigned e = e0 + lane;
    const unsigned here = __ballot_sync(~0u, e < a.experts && index < g.last[e]);
    if (!here) continue;
    const unsigned owner = e0 + __ffs(here) - 1;
    const unsigned row = g.begin[owner] + (index - (owner ? g.last[owner - 1] : 0)) * tile_rows;
    return {owner, row, min(tile_rows, g.end[owner] - row)};
  }
  return {0, 0, 0};
}

// The tiles that a block does, one after the other: every grid-th.  Called by a whole warp.
struct Walk {
  const Product& a;
  const Groups& groups;
  unsigned tile_rows, channel_tiles, at;
  Tile tile;
  unsigned channel_tile;

  __device__ __forceinline__ Walk(const Product& p, const Groups& g, unsigned rows, unsigned channels)
      : a(p), groups(g), tile_rows(rows), channel_tiles(channels), at(blockIdx.x) {}
  __device__ __forceinline__ bool next() {
    tile = look_up(a, groups, tile_rows, at / channel_tiles);
    channel_tile = at % channel_tiles;
    at += gridDim.x;
    return tile.rows;
  }
};

template <class T, int BN>
__global__ void __launch_bounds__(kMmaThreads, 1)
    product_tiles(const Product a, const __grid_constant__ CUtensorMap weights, const __grid_constant__ CUtensorMap rows,
                  unsigned channel_tiles) {
  using Shape = MmaShape<BN>;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[Shape::stages], empty[Shape::stages], summed[2], drained[2], issued;
  __shared__ unsigned tensor_base;
  __shared__ Groups groups;
  const unsigned at_stages = (shared_at(raw) + 1023) / 1024 * 1024, at_full = shared_at(full), at_empty = shared_at(empty);
  const unsigned low_operand = operand_low(at_stages);
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (unsigned s = 0; s < Shape::stages; ++s) {
      barrier_init(full + s, 1);
      barrier_init(empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(summed + s, 1);
      barrier_init(drained + s, 8);
    }
    barrier_init(&issued, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&weights) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&rows) : "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_at(&tensor_base)),
                 "r"(Shape::columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 3) list_groups(a, BN, groups);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned base = tensor_base;
  const unsigned steps = (a.padded + Shape::spans * kSpan - 1) / (Shape::spans * kSpan);
  Walk walk(a, groups, BN, channel_tiles);

  if (warp == 0) {
    unsigned stage = 0, phase = 0, filled = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const int y = (int)(walk.tile.expert * a.channels + walk.channel_tile * kTileM);
      for (unsigned k = 0; k < steps; ++k) {
        if (!(ok = warp_wait(at_empty + stage * 8, phase ^ 1))) break;
        const unsigned to = at_stages + stage * Shape::stage_bytes, barrier = at_full + stage * 8;
        if (elected()) {
          expect(barrier, Shape::stage_bytes);
#pragma unroll
          for (unsigned s = 0; s < Shape::spans; ++s) {
            const int x = (int)((k * Shape::spans + s) * kSpan);      // behind the inner size zeros arrive
            tma_load(to + s * Shape::span_bytes, &weights, barrier, x, y);
            tma_load(to + s * Shape::span_bytes + kTileM * kSpan, &rows, barrier, x, (int)walk.tile.row);
          }
        }
        if (++filled > Shape::stages) filled = Shape::stages;
        if (++stage == Shape::stages) { stage = 0; phase ^= 1; }
      }
    }
    // no block ends with copies into its shared memory in flight
    if (!ok)
      for (unsigned n = 0; n < filled; ++n) {
        stage = stage ? stage - 1 : Shape::stages - 1;
        if (stage == Shape::stages - 1) phase ^= 1;
        warp_wait(at_full + stage * 8, phase);
      }
  } else if (warp == 1) {
    unsigned stage = 0, phase = 0, half = 0, turn = 0;
    bool ok = true;
    while (ok && walk.next()) {
      ok = warp_wait(shared_at(drained) + half * 8, turn ^ 1);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (unsigned k = 0; ok && k < steps; ++k) {
        if (!(ok = warp_wait(at_full + stage * 8, phase))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned w = low_operand + stage * (Shape::stage_bytes / 16), q = w + kTileM * kSpan / 16, d = base + half * BN;
        if (elected()) {
#pragma unroll
          for (unsigned s = 0; s < Shape::spans; ++s) {
#pragma unroll
            for (unsigned i = 0; i < kSpan / 32; ++i) {
              const unsigned at = s * (Shape::span_bytes / 16) + 2 * i;
              mma_i8<BN>(d, w + at, q + at, k || s || i);
            }
          }
          mma_commit(at_empty + stage * 8);
        }
        if (++stage == Shape::stages) { stage = 0; phase ^= 1; }
      }
      if (ok && elected()) mma_commit(shared_at(summed) + half * 8);
      __syncwarp();
      half ^= 1;
      turn ^= half == 0;
    }
    // nor with matrix instructions that still write to the tensor memory it gives back
    if (!ok) {
      if (elected()) mma_commit(shared_at(&issued));
      warp_wait(shared_at(&issued), 0);
    }
  } else if (warp >= 4) {
    unsigned half = 0, turn = 0;
    bool ok = true;
    while (walk.next()) {        // after a wait that ran out: no more waits, and NaN for all tiles that are left
      const Tile tile = walk.tile;
      // a quarter of the channels, and every second 32 of the rows
      const unsigned quarter = warp % 4, odd = (warp - 4) / 4 * 32;
      const unsigned n = walk.channel_tile * kTileM + quarter * 32 + lane;
      const uint64_t c = (uint64_t)tile.expert * a.channels + n;
      const bool in = n < a.channels;
      const float ws = in ? a.weight_scale[c] : 0.f, b = in && a.bias ? a.bias[c] : 0.f;
      float mine = odd + lane < tile.rows ? a.scale[tile.row + odd + lane] : 0.f;      // of the first 32 rows
      ok = ok && warp_wait(shared_at(summed) + half * 8, turn);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      T* out = static_cast<T*>(a.out) + (uint64_t)(tile.row + odd) * a.channels + n;
      const unsigned from = base + half * BN + (quarter * 32 << 16);
#pragma unroll 1
      for (unsigned r0 = odd; r0 < tile.rows; r0 += 64) {
        int v[32];
        tensor_load(from + r0, v);        // what lies there, where the sums never came
        const float next = r0 + 64 + lane < tile.rows ? a.scale[tile.row + r0 + 64 + lane] : 0.f;
        const unsigned rows_left = in ? tile.rows - r0 : 0;
#pragma unroll
        for (unsigned j = 0; j < 32; ++j) {
          const float s = __shfl_sync(~0u, mine, j);
          const float value = ok ? fmaf((float)v[j], s * ws, b) : NAN;
          if (j < rows_left) *out = from_float<T>(value);
          out += a.channels;
        }
        out += (uint64_t)32 * a.channels;
        mine = next;
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (ok && lane == 0) barrier_arrive(drained + half);
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
  by_type(type, [&](auto t) {
    using T = decltype(t);
    const unsigned blocks = (unsigned)a.count;
    const uint64_t packs = ceil_div(a.inner * sizeof(T), 16 * kQuantizeThreads);
    if (!a.wide || packs > 8) quantize_rows<T, 0><<<blocks, kQuantizeThreads, 0, stream>>>(a);
    else if (packs <= 1) quantize_rows<T, 1><<<blocks, kQuantizeThreads, 0, stream>>>(a);
    else if (packs <= 2) quantize_rows<T, 2><<<blocks, kQuantizeThreads, 0, stream>>>(a);
    else if (packs <= 4) quantize_rows<T, 4><<<blocks, kQuantizeThreads, 0, stream>>>(a);
    else quantize_rows<T, 8><<<blocks, kQuantizeThreads, 0, stream>>>(a);
  });
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
  const cuuint32_t box[2] = {kSpan, box_rows}, step[2] = {1, 1};
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

// Which kernel a product takes, and its tile's rows: 0 for product_rows.  The host does
// not know the groups, so it goes by the rows of an expert on average.
//
// A block takes its tiles in rounds, and 128 bytes of inner size take a tile 0.23, 0.35
// or 0.44 us at 64, 128 or 256 rows (from 500 and 2000 rows x 4096 x 4096; tiles of 32
// rows took 0.24), so the tile is the one whose rounds of a B200's 148 SMs cost least,
// the smaller of equals: 500 rows take 17.5 us by 64, 14.2 by 128 and 17.8 by 256; 2000 rows 48.6 by 64
// and 30.4 by 256.  A group's last tile is half empty on average.
unsigned tile_rows_of(uint64_t rows, uint64_t experts, uint64_t channels) {
  const uint64_t each = ceil_div(rows, experts);
  if (rows <= 8 || each <= 2) return 0;
  const uint64_t groups = experts < rows ? experts : rows;
  static const struct { unsigned rows; uint64_t cost; } shapes[] = {{64, 23}, {128, 35}, {256, 44}};
  unsigned best = 0;
  uint64_t least = ~0ull;
  for (const auto& s : shapes) {
    const uint64_t row_tiles = experts == 1 ? ceil_div(rows, s.rows) : ceil_div(2 * rows + groups * s.rows, 2 * s.rows);
    const uint64_t tiles = row_tiles * ceil_div(channels, kTileM);
    const uint64_t cost = ceil_div(tiles, 148) * s.cost;
    if (cost < least) {
      least = cost;
      best = s.rows;
    }
  }
  return best;
}

// Whether rows are quantized where they are used: few of them, eight of which fit shared memory.
bool on_the_way(unsigned tile_rows, uint64_t padded) { return !tile_rows && padded <= 24 * 1024; }

template <int BN>
void tiles(int type, const Product& a, int device, cudaStream_t stream) {
  const unsigned sms = sm_count(device);
  using Shape = MmaShape<BN>;
  const CUtensorMap w = tensor_map(a.weight, (uint64_t)a.experts * a.channels, a.padded, kTileM);
  const CUtensorMap q = tensor_map(a.q, a.rows, a.padded, BN);
  const unsigned channel_tiles = (unsigned)ceil_div(a.channels, kTileM);
  const uint64_t most = tile_bound(a, BN) * channel_tiles;
  need(most < (1ull << 31), "too many rows");
  const unsigned blocks = most > sms ? sms : (unsigned)most;
  by_type(type, [&](auto t) {
    constexpr auto kernel = product_tiles<decltype(t), BN>;
    room<kernel>(device);
    kernel<<<blocks, kMmaThreads, Shape::shared, stream>>>(a, w, q, channel_tiles);
  });
  check(cudaGetLastError(), "int8_product");
}

void product_by_tiles(int type, const Product& a, int device, cudaStream_t stream) {
  need((uint64_t)a.experts * a.channels < (1ull << 31), "too many channels");
  switch (tile_rows_of(a.rows, a.experts, a.channels)) {
    case 256: return tiles<256>(type, a, device, stream);
    case 128: return tiles<128>(type, a, device, stream);
    default: return tiles<64>(type, a, device, stream);
  }
}

// z: quantize on the way; nullptr: a.q and a.scale are given.
template <int RT>
void rows_at_once(int type, const Product& a, const Quantize* z, int device, cudaStream_t stream) {
  const unsigned channel_blocks = (unsigned)ceil_div(a.channels, kRowsThreads / 32);
  const uint64_t most = tile_bound(a, RT) * channel_blocks;
  need(most < (1ull << 31), "too many rows");
  by_type(type, [&](auto t) {
    if (z) {
      constexpr auto kernel = product_rows<decltype(t), RT, true>;
      const unsigned shared = RT * a.padded;
      room<kernel>(device);
      kernel<<<(unsigned)most, kRowsThreads, shared, stream>>>(a, *z, channel_blocks);
    } else {
      product_rows<decltype(t), RT, false><<<(unsigned)most, kRowsThreads, 0, stream>>>(a, Quantize{}, channel_blocks);
    }
  });
  check(cudaGetLastError(), "int8_product");
}

void product_by_rows(int type, const Product& a, const Quantize* z, int device, cudaStream_t stream) {
  const uint64_t each = ceil_div(a.rows, a.experts);
  if (a.rows == 1) rows_at_once<1>(type, a, z, device, stream);
  else if (a.rows == 2 || each <= 2) rows_at_once<2>(type, a, z, device, stream);
  else if (a.rows <= 4) rows_at_once<4>(type, a, z, device, stream);
  else rows_at_once<8>(type, a, z, device, stream);
}

Quantize quantize_args(int type, const void* x, int64_t x_stride, uint64_t x_rows, unsigned inner, const int32_t* rows,
                       unsigned divisor, uint64_t count, int8_t* q, float* scale, bool kept = true) {
  need(known_type(type), "unknown element type");
  need(inner > 0 && inner <= EPS_B200_INT8_INNER, "inner size out of range");
  need(rows ? divisor > 0 : count <= x_rows, "more rows than x has");
  need(!count || (!kept || (q && scale)) && (x || !x_rows), "null input or output");
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
  if (on_the_way(tile_rows_of(rows, experts ? experts : 1, channels), eps_b200_int8_stride(inner))) return 0;
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
    const auto st = static_cast<cudaStream_t>(stream);
    const unsigned tile_rows = tile_rows_of(p.rows, p.experts, p.channels);
    if (!tile_rows) {
      OnDevice on(a->device);
      return product_by_rows(a->type, p, nullptr, a->device, st);
    }
    OnDevice on(a->device);
    product_by_tiles(a->type, p, a->device, st);
  });
}

int eps_b200_int8_linear(const EpsB200Int8Product* a, const void* x, int64_t x_stride, uint64_t x_rows,
                         const int32_t* rows, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Product p = product_args(a);
    if (!p.rows) return;
    const uint64_t bytes = eps_b200_int8_product_workspace(a->rows, a->experts, a->channels, a->inner);
    need(!bytes || (a->workspace && a->workspace_bytes >= bytes), "int8 workspace too small");
    auto* q = static_cast<int8_t*>(a->workspace);
    auto* scale = reinterpret_cast<float*>(q + (uint64_t)p.rows * p.padded);
    const unsigned tile_rows = tile_rows_of(p.rows, p.experts, p.channels);
    const bool direct = on_the_way(tile_rows, p.padded);
    need(direct || q, "null workspace");
    const Quantize z = quantize_args(a->type, x, x_stride, x_rows, a->inner, rows, a->rows_divisor, a->rows, q, scale, !direct);
    p.q = q;
    p.scale = scale;
    const auto st = static_cast<cudaStream_t>(stream);
    OnDevice on(a->device);
    if (direct) return product_by_rows(a->type, p, &z, a->device, st);
    quantize(a->type, z, st);
    if (tile_rows) product_by_tiles(a->type, p, a->device, st);
    else product_by_rows(a->type, p, nullptr, a->device, st);
  });
}

}  // extern "C"
