// low_rank.cu -- low-rank adapters of many requests at once (eps_b200_low_rank).
//
// Mathematics, for a row t with adapter a:
//   u = down[a] x[t],   out[t] = base[t] + scale[a] * up[a] u
//
// Bound: x and base are read and out is written once, each adapter in use is read once
// for the rows that have it; 2 R operations a value of x and of out are far below what
// the matrix instructions give, so what counts is that loads stay in flight.  Rows are
// taken in units of one adapter and up to 64 rows (16 where the call has few).  A
// cluster works on a unit: its warps share out the inner size, each summing its share of
// u for its rows, the parts are added over the warps and, through distributed shared
// memory, over the blocks; then its warps share out the channels.  One launch, no u in
// memory; a launch before it sorts many rows by adapter.
//
// Fragments need no exchange between lanes: a sum over k may take its terms in any order,
// so each lane of a matrix instruction's row takes 16 consecutive bytes and gives them to
// the places that the instruction has for it, the same for both operands.  In the second
// product the columns are dealt so that a lane ends up with 16 bytes of consecutive
// channels.  So every lane copies what it needs itself, asynchronously and some turns
// ahead, into shared memory that no other lane reads; the copies of base go on while u is
// still being added up.
//
// Precision: 16-bit products are exact and summed in float.  u is not rounded to 16
// bits: it goes on as the sum of two 16-bit values (float16: under a power of two of the
// row, so that its range does not matter).  Floats are cut into three bfloat16 values,
// which is exact, and the six largest of the nine products are summed; the others are
// below 2^-25 of the first.
#include <algorithm>
#include <cmath>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

constexpr unsigned kThreads = 256, kWarps = kThreads / 32;
constexpr unsigned kFew = 64;             // rows that the units are found for without a sort
constexpr unsigned kUnitTiles = 4;        // 16-row tiles of a unit of sorted rows
constexpr unsigned kUnit = kUnitTiles * 16;
constexpr unsigned kSortThreads = 1024, kSortBatch = 8;      // ids of a thread that are asked for at once

struct Unit {
  int32_t adapter;                        // -1: none
  uint32_t begin, count, unused;          // rows order[begin ..]
};

struct Call {
  const void *down, *up, *x, *base;
  void* out;
  const float* scale;
  const int32_t* ids;
  int64_t x_stride, base_stride, out_stride;
  uint32_t rows, adapters, rank, inner, padded, channels;
  const Unit* units;                      // sorted rows
  const uint32_t* unit_count;
  const int32_t* order;
};

// ------------------------------------------------------------ matrix instructions
template <class T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, f16>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two floats as three pairs of bfloat16 whose sums they are.  Each is the nearest to what
// is left, so what the dropped products lose has no sign of its own.
__device__ __forceinline__ void cut(float a, float b, uint32_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    p[i] = reinterpret_cast<const uint32_t&>(h);
    a -= __uint_as_float(p[i] << 16);
    b -= __uint_as_float(p[i] & 0xFFFF0000u);
  }
}

// The products of cut operands that count, small ones first: (plane of a, plane of b).
__device__ constexpr int kTerms[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};

// BYTES from p to this lane's place in shared memory, or zeros.
template <int BYTES>
__device__ __forceinline__ void copy_ahead(unsigned to, const void* p, bool there) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p), "r"(there ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(p), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
template <class P>
__device__ __forceinline__ P own_shared(unsigned at) {
  P r;
  if constexpr (sizeof(P) == 16) {
    uint4& x = reinterpret_cast<uint4&>(r);
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
  } else if constexpr (sizeof(P) == 8) {
    uint2& x = reinterpret_cast<uint2&>(r);
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(at) : "memory");
  } else {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(reinterpret_cast<uint32_t&>(r)) : "r"(at) : "memory");
  }
  return r;
}

// 16 bytes of a row from p on, of which the first `left` values are there; the others are
// 0.  WIDE: rows begin and end on 16 bytes.
template <class T, bool WIDE>
__device__ __forceinline__ void copy_row(unsigned to, const T* p, int left) {
  constexpr int V = 16 / sizeof(T);
  if constexpr (WIDE) {
    copy_ahead<16>(to, p, left > 0);
  } else {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = i < left ? p[i] : from_float<T>(0.f);
    const uint4& x = reinterpret_cast<const uint4&>(r);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
  }
}

template <class T, bool WIDE>
__device__ __forceinline__ void store_row(T* p, int left, const Pack<T, 16 / sizeof(T)>& r) {
  constexpr int V = 16 / sizeof(T);
  if constexpr (WIDE) {
    if (left > 0) store_pack<T, V>(p, r);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) p[i] = r.v[i];
  }
}

// --------------------------------------------------------------------- the shapes
// What a kernel for type T, padded rank R and M tiles of 16 rows is cut into.
template <class T, int R, int M>
struct Shape {
  static constexpr bool kFloat = std::is_same_v<T, float>;
  static constexpr int kEach = 16 / sizeof(T);                   // values of a lane's load of x and down
  static constexpr int kStep = 4 * kEach;                        // inner values that a warp takes at once
  // tiles of a warp in the first product: R / 8 x 4 sums a lane each
  static constexpr int kTiles = M == 1 ? 1 : kFloat ? (R <= 16 ? 2 : 1) : R <= 32 ? 4 : R == 64 ? 2 : 1;
  static constexpr int kAcross = M / kTiles;                     // warps side by side over the rows
  static constexpr int kAlong = kWarps / kAcross;                // and along the inner size
  // second product: a lane's ranks of one load, loads, instructions, and 16-bit parts of u
  static constexpr int kRanks = R / 4 < kEach ? R / 4 : kEach;
  static constexpr int kLoads = R / (4 * kRanks);
  static constexpr int kPairsInOne = !kFloat && R == 8;          // both parts of u in one instruction
  static constexpr int kMultiplies = kPairsInOne || kRanks <= 4 ? kLoads : 2 * kLoads;
  static constexpr int kParts = kFloat ? 3 : kPairsInOne ? 1 : 2;
  static constexpr int kRun = 4 * kEach;                         // channels that a warp takes at once
  static constexpr int kMatrices = kEach / 2;                    // of 8 channels
  static constexpr bool kKeep = R * sizeof(T) <= 256;            // up's fragments stay in registers for all tiles
  // a warp's copies under way: pieces of a lane's 16 bytes of x and down, or of base and up
  static constexpr bool kWeights = R * sizeof(T) <= 64;          // down and up are copied ahead too
  static constexpr int kRows = (kTiles > M ? kTiles : M) * 2 * 512;
  static constexpr int kDown = kWeights ? R / 8 * 512 : 0;
  static constexpr int kUpPiece = kRanks * sizeof(T);
  static constexpr int kUp = kWeights ? kMatrices * kLoads * kUpPiece * 32 : 0;
  static constexpr int kSlot = kRows + (kDown > kUp ? kDown : kUp);
  static constexpr int kAhead = M == 1 ? 4 : 2;
  static constexpr size_t kCopies = (size_t)kWarps * kAhead * kSlot;
  // the warps' sums, in two rounds; the first becomes the block's part, the others u's fragments
  static constexpr size_t kPart = (size_t)M * 16 * R * 4;
  static constexpr size_t kFragments = (size_t)M * kMultiplies * kParts * 512;
  static constexpr int kRounds = kAlong > 1 ? 2 : 1;
  static constexpr size_t kSums = kAlong / kRounds * kPart;
  static constexpr size_t kBytes = kCopies + (kSums > kPart + kFragments ? kSums : kPart + kFragments);
};

// A unit's rows, as every block of the cluster finds them.
template <int M>
struct Found {
  int32_t row[M * 16];
  int32_t adapter;
  uint32_t count;
};

// The unit of this number among few rows: rows of one adapter, 16 at most, in order.
// False if there are fewer units.
__device__ __forceinline__ bool find_few(const Call& c, unsigned number, Found<1>& f) {
  __shared__ int32_t ids[kFew];
  __shared__ uint32_t starts[2];
  __shared__ unsigned first;
  const unsigned t = threadIdx.x;
  int32_t id = -1;
  if (t < c.rows) {
    id = c.ids[t];
    if ((uint32_t)id >= c.adapters) id = -1;
  }
  if (t < kFew) ids[t] = id;
  __syncthreads();
  unsigned before = 0, all = 0;            // rows of the same adapter
  if (t < c.rows)
    for (unsigned s = 0; s < c.rows; ++s) {
      const bool same = ids[s] == id;
      before += same && s < t;
      all += same;
    }
  const bool start = t < c.rows && before % 16 == 0;
  if (t < kFew) {
    const unsigned b = __ballot_sync(~0u, start);
    if (t % 32 == 0) starts[t / 32] = b;
  }
  __syncthreads();
  const unsigned low = starts[0], high = starts[1];
  if (number >= (unsigned)(__popc(low) + __popc(high))) return false;
  if (start) {
    const unsigned mine = t < 32 ? __popc(low & ((1u << t) - 1)) : __popc(low) + __popc(high & ((1u << (t - 32)) - 1));
    if (mine == number) {
      f.adapter = id;
      f.count = min(16u, all - before);
      first = before;
    }
  }
  __syncthreads();
  if (t < c.rows && id == f.adapter && before - first < 16) f.row[before - first] = (int32_t)t;
  __syncthreads();
  return true;
}

__device__ __forceinline__ bool find_sorted(const Call& c, unsigned number, Found<kUnitTiles>& f) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (number >= *c.unit_count) return false;
  const Unit u = c.units[number];
  if (threadIdx.x < u.count) f.row[threadIdx.x] = c.order[u.begin + threadIdx.x];
  if (threadIdx.x == 0) {
    f.adapter = u.adapter;
    f.count = u.count;
  }
  __syncthreads();
  return true;
}

// ----------------------------------------------------------------- a warp's turns
// The turns of a warp's lane: steps along the inner size, then runs of channels.  Turn i's
// copies lie in slot i % kAhead.
template <class T, int R, int M, bool WIDE>
struct Turns {
  using S = Shape<T, R, M>;
  const Call& c;
  const Found<M>& f;
  unsigned tiles, across, step, steps, run, runs, slots;     // first step and number of steps, first run and number of runs
  const T *down, *up;

  __device__ __forceinline__ Turns(const Call& c, const Found<M>& f, unsigned rank, unsigned blocks, unsigned shared) : c(c), f(f) {
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, quad = lane % 4;
    const unsigned along = warp / S::kAcross;
    across = warp % S::kAcross;
    tiles = (f.count + 15) / 16;
    const unsigned all = c.padded / S::kStep, share = rank * S::kAlong + along, shares = blocks * S::kAlong;
    step = (unsigned)((uint64_t)all * share / shares);
    steps = across * S::kTiles < tiles ? (unsigned)((uint64_t)all * (share + 1) / shares) - step : 0;
    const unsigned every = (c.channels + S::kRun - 1) / S::kRun;
    run = (unsigned)((uint64_t)every * rank / blocks) + warp;
    const unsigned end = (unsigned)((uint64_t)every * (rank + 1) / blocks);
    runs = run < end ? (end - run + kWarps - 1) / kWarps : 0;
    slots = shared + warp * S::kAhead * S::kSlot + lane * 16;
    down = static_cast<const T*>(c.down) + ((uint64_t)f.adapter * R + g) * c.padded + quad * S::kEach;
    up = static_cast<const T*>(c.up) + (uint64_t)f.adapter * c.channels * R + quad * S::kRanks;
  }
  __device__ __forceinline__ unsigned slot(unsigned i) const { return slots + i % S::kAhead * S::kSlot; }
  __device__ __forceinline__ unsigned upper(unsigned i) const { return slot(i) + S::kRows; }
  // where a lane's smaller pieces lie, one lane's next to the other's
  __device__ __forceinline__ unsigned up_piece(unsigned i, int k) const {
    return upper(i) - threadIdx.x % 32 * (16 - S::kUpPiece) + k * S::kUpPiece * 32;
  }
  __device__ __forceinline__ const T* down_at(unsigned i, int n) const { return down + (size_t)n * 8 * c.padded + (step + i) * S::kStep; }
  // column g of matrix j is channel kEach (g / 2) + 2 j + g % 2 of the run
  __device__ __forceinline__ const T* up_at(unsigned i, int j, int l) const {
    const unsigned g = threadIdx.x % 32 / 4;
    const unsigned channel = (run + (i - steps) * kWarps) * S::kRun + g / 2 * S::kEach + 2 * j + g % 2;
    return up + (size_t)min(channel, c.channels - 1) * R + l * 4 * S::kRanks;
  }

  __device__ __forceinline__ void copy(unsigned i) const {
    const unsigned lane = threadIdx.x % 32, g = lane / 4, quad = lane % 4;
    if (i < steps) {
      const unsigned k = (step + i) * S::kStep + quad * S::kEach;
      const int left = (int)c.inner - (int)k;
#pragma unroll
      for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned r = (across * S::kTiles + m) * 16 + h * 8 + g;
          const bool there = r < f.count;        // a row behind the unit's last counts as zeros
          copy_row<T, WIDE>(slot(i) + (m * 2 + h) * 512, static_cast<const T*>(c.x) + (int64_t)f.row[there ? r : 0] * c.x_stride + (left > 0 ? k : 0),
                            there ? left : 0);
        }
      if constexpr (S::kWeights) {
#pragma unroll
        for (int n = 0; n < R / 8; ++n) copy_ahead<16>(upper(i) + n * 512, down_at(i, n), true);
      }
    } else if (i < steps + runs) {
      const unsigned at = (run + (i - steps) * kWarps) * S::kRun + quad * S::kEach;
      const int left = (int)c.channels - (int)at;
      if (c.base) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          if (m >= tiles) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned r = m * 16 + h * 8 + g;
            const bool there = r < f.count;
            copy_row<T, WIDE>(slot(i) + (m * 2 + h) * 512,
                              static_cast<const T*>(c.base) + (int64_t)f.row[there ? r : 0] * c.base_stride + (left > 0 ? at : 0), there ? left : 0);
          }
        }
      }
      if constexpr (S::kWeights) {
#pragma unroll
        for (int j = 0; j < S::kMatrices; ++j)
#pragma unroll
          for (int l = 0; l < S::kLoads; ++l) copy_ahead<S::kUpPiece>(up_piece(i, j * S::kLoads + l), up_at(i, j, l), true);
      }
    }
    copies_end();
  }
};

// ------------------------------------------------------------------- u = down x
template <class T, int R, int M, bool WIDE>
__device__ __forceinline__ void inner_product(const Turns<T, R, M, WIDE>& t, float* sums) {
  using S = Shape<T, R, M>;
  using P = Pack<T, S::kEach>;
  constexpr int kCols = R / 8;
  float acc[S::kTiles][kCols][4] = {};
  for (unsigned i = 0; i < t.steps; ++i) {
    P d[kCols], x[S::kTiles][2];
    if constexpr (!S::kWeights) {
#pragma unroll
      for (int n = 0; n < kCols; ++n) d[n] = load_pack<T, S::kEach>(t.down_at(i, n));
    }
    copies_wait<S::kAhead - 1>();
#pragma unroll
    for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) x[m][h] = own_shared<P>(t.slot(i) + (m * 2 + h) * 512);
    if constexpr (S::kWeights) {
#pragma unroll
      for (int n = 0; n < kCols; ++n) d[n] = own_shared<P>(t.upper(i) + n * 512);
    }
    t.copy(i + S::kAhead);
    if constexpr (S::kFloat) {
#pragma unroll
      for (int m = 0; m < S::kTiles; ++m) {
        uint32_t a[3][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t p[3];
            cut(x[m][h].v[2 * e], x[m][h].v[2 * e + 1], p);
#pragma unroll
            for (int q = 0; q < 3; ++q) a[q][2 * e + h] = p[q];
          }
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
          uint32_t b0[3], b1[3];
          cut(d[n].v[0], d[n].v[1], b0);
          cut(d[n].v[2], d[n].v[3], b1);
          // summed apart and added in float: the matrix instruction's sums are cut off, not rounded
          float part[4] = {};
#pragma unroll
          for (int q = 0; q < 6; ++q) multiply<bf16>(part, a[kTerms[q][0]], b0[kTerms[q][1]], b1[kTerms[q][1]]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][n][e] += part[e];
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < kCols; ++n) {
        const uint32_t* const b = reinterpret_cast<const uint32_t*>(&d[n]);
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m) {
          const uint32_t* const lo = reinterpret_cast<const uint32_t*>(&x[m][0]);
          const uint32_t* const hi = reinterpret_cast<const uint32_t*>(&x[m][1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t a[4] = {lo[2 * k], hi[2 * k], lo[2 * k + 1], hi[2 * k + 1]};
            multiply<T>(acc[m][n], a, b[2 * k], b[2 * k + 1]);
          }
        }
      }
    }
  }
  // the warps along the inner size write their sums, half of them at a time
  const unsigned lane = threadIdx.x % 32, g = lane / 4, quad = lane % 4, along = threadIdx.x / 32 / S::kAcross;
  constexpr unsigned kHalf = S::kAlong / S::kRounds;
#pragma unroll
  for (unsigned round = 0; round < S::kRounds; ++round) {
    if (round) __syncthreads();
    if (along / kHalf == round) {
#pragma unroll
      for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* const row = sums + ((along % kHalf * M + t.across * S::kTiles + m) * 16 + h * 8 + g) * R + 2 * quad;
#pragma unroll
          for (int n = 0; n < kCols; ++n) {
            float2& to = *reinterpret_cast<float2*>(row + n * 8);
            float2 v = make_float2(acc[m][n][2 * h], acc[m][n][2 * h + 1]);
            if (round) v.x += to.x, v.y += to.y;
            to = v;
          }
        }
    }
  }
}

// --------------------------------------------------- u as the next product's fragments
__device__ __forceinline__ uint32_t pair_of(bf16, float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(p);
}
__device__ __forceinline__ uint32_t pair_of(f16, float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(p);
}
template <class T> __device__ __forceinline__ float left_over(float v) {
  const float r = v - to_float(from_float<T>(v));
  return isfinite(r) ? r : 0.f;            // an infinity is all in the first part
}

// Adds u up over the cluster and writes its fragments; factor[row] is what the second
// product's sums take.
template <class T, int R, int M>
__device__ __forceinline__ void lay_out(const Call& c, const Found<M>& f, unsigned blocks, const float* part, uint32_t* fragments, float* factor) {
  using S = Shape<T, R, M>;
  constexpr unsigned kLanes = R / 2 < 32 ? R / 2 : 32;        // lanes of a row, two ranks each at a time
  constexpr int kTimes = R / 2 / kLanes;
  const float scale = c.scale ? c.scale[f.adapter] : 1.f;
  for (unsigned item = threadIdx.x; item < M * 16 * kLanes; item += kThreads) {      // whole warps: M * 16 * kLanes is a multiple of 32
    const unsigned row = item / kLanes, q = item % kLanes;
    float2 u[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
      const unsigned r = 2 * (i * kLanes + q);
      u[i] = make_float2(0.f, 0.f);
      for (unsigned b = 0; b < blocks; ++b) {
        const float2 v = cluster_load(reinterpret_cast<const float2*>(part + row * R + r), b);
        u[i].x += v.x;
        u[i].y += v.y;
      }
      if (r >= c.rank) u[i].x = 0.f;         // an infinity times the padding's 0
      if (r + 1 >= c.rank) u[i].y = 0.f;
    }
    float times = 1.f, back = 1.f;
    if constexpr (std::is_same_v<T, f16>) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < kTimes; ++i) top = fmaxf(top, fmaxf(fabsf(u[i].x), fabsf(u[i].y)));
#pragma unroll
      for (unsigned o = kLanes / 2; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      // the largest goes to [2^13, 2^14): two parts then hold all but 2^-38 of it
      const int e = (int)(__float_as_uint(top) >> 23);
      if (e < 255) {                         // else an infinity, or NaN, stays what it is
        times = __uint_as_float((uint32_t)min(254 + 13 - e, 253) << 23);
        back = 1.f / times;
      }
    }
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
      const unsigned r = 2 * (i * kLanes + q);
      const unsigned load = r / (4 * S::kRanks), quad = r / S::kRanks % 4, at = r % S::kRanks;
      const unsigned multiply = S::kRanks <= 4 ? load : 2 * load + at / 4;
      const unsigned lane = row % 8 * 4 + quad, upper = row % 16 / 8, which = at % 4 / 2 * 2 + upper;
      uint32_t* const to = fragments + ((row / 16 * S::kMultiplies + multiply) * S::kParts * 32 + lane) * 4;
      const float a = u[i].x * times, b = u[i].y * times;
      if constexpr (S::kFloat) {
        uint32_t p[3];
        cut(a, b, p);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          to[k * 128 + which] = p[k];
          if constexpr (R == 8) to[k * 128 + 2 + upper] = 0;     // 8 ranks fill half of an instruction
        }
      } else {
        const uint32_t first = pair_of(T{}, a, b), second = pair_of(T{}, left_over<T>(a), left_over<T>(b));
        if constexpr (S::kPairsInOne) {
          to[upper] = first;
          to[2 + upper] = second;
        } else {
          to[which] = first;
          to[128 + which] = second;
        }
      }
    }
    if (q == 0) factor[row] = scale * back;
  }
}

// ------------------------------------------------------- out = base + factor * up u
template <class T, int R, int M, bool WIDE>
__device__ __forceinline__ void outer_product(const Turns<T, R, M, WIDE>& t, const uint32_t* fragments, const float* factor) {
  using S = Shape<T, R, M>;
  using P = Pack<T, S::kRanks>;
  using O = Pack<T, S::kEach>;
  const Call& c = t.c;
  const unsigned lane = threadIdx.x % 32, g = lane / 4, quad = lane % 4;
  for (unsigned i = t.steps; i < t.steps + t.runs; ++i) {
    const unsigned at = (t.run + (i - t.steps) * kWarps) * S::kRun + quad * S::kEach;          // this lane's channels
    const int left = (int)c.channels - (int)at;
    P held[S::kKeep ? S::kMatrices : 1][S::kKeep ? S::kLoads : 1];
    if constexpr (S::kKeep && !S::kWeights) {
#pragma unroll
      for (int j = 0; j < S::kMatrices; ++j)
#pragma unroll
        for (int l = 0; l < S::kLoads; ++l) held[j][l] = load_pack<T, S::kRanks>(t.up_at(i, j, l));
    }
    copies_wait<S::kAhead - 1>();
    O before[M][2];
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (m < t.tiles && c.base) {
#pragma unroll
        for (int h = 0; h < 2; ++h) before[m][h] = own_shared<O>(t.slot(i) + (m * 2 + h) * 512);
      }
    if constexpr (S::kWeights) {
#pragma unroll
      for (int j = 0; j < S::kMatrices; ++j)
#pragma unroll
        for (int l = 0; l < S::kLoads; ++l) held[j][l] = own_shared<P>(t.up_piece(i, j * S::kLoads + l));
    }
    t.copy(i + S::kAhead);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if (m >= t.tiles) break;
      float acc[S::kMatrices][4] = {};
#pragma unroll
      for (int l = 0; l < S::kLoads; ++l) {
#pragma unroll
        for (int k = 0; k < (S::kRanks <= 4 ? 1 : 2); ++k) {
          const int q = S::kRanks <= 4 ? l : 2 * l + k;
          uint32_t a[S::kParts][4];
#pragma unroll
          for (int p = 0; p < S::kParts; ++p) {
            const uint4 w = reinterpret_cast<const uint4*>(fragments)[((m * S::kMultiplies + q) * S::kParts + p) * 32 + lane];
            a[p][0] = w.x, a[p][1] = w.y, a[p][2] = w.z, a[p][3] = w.w;
          }
#pragma unroll
          for (int j = 0; j < S::kMatrices; ++j) {
            P d;
            if constexpr (S::kKeep) d = held[j][l];
            else d = load_pack<T, S::kRanks>(t.up_at(i, j, l));
            if constexpr (S::kFloat) {
              uint32_t b0[3], b1[3] = {0, 0, 0};
              cut(d.v[0], d.v[1], b0);
              if constexpr (S::kRanks == 4) cut(d.v[2], d.v[3], b1);
              float part[4] = {};
#pragma unroll
              for (int n = 0; n < 6; ++n) multiply<bf16>(part, a[kTerms[n][0]], b0[kTerms[n][1]], b1[kTerms[n][1]]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[j][e] += part[e];
            } else {
              const uint32_t* const b = reinterpret_cast<const uint32_t*>(&d);
              if constexpr (S::kPairsInOne) {
                multiply<T>(acc[j], a[0], b[0], b[0]);
              } else {
                multiply<T>(acc[j], a[1], b[2 * k], b[2 * k + 1]);
                multiply<T>(acc[j], a[0], b[2 * k], b[2 * k + 1]);
              }
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned r = m * 16 + h * 8 + g;
        if (r >= t.f.count) continue;
        float v[S::kEach];
        if (c.base) {
          widen(before[m][h], v);
        } else {
#pragma unroll
          for (int e = 0; e < S::kEach; ++e) v[e] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < S::kMatrices; ++j) {
          v[2 * j] = fmaf(acc[j][2 * h], factor[r], v[2 * j]);
          v[2 * j + 1] = fmaf(acc[j][2 * h + 1], factor[r], v[2 * j + 1]);
        }
        store_row<T, WIDE>(static_cast<T*>(c.out) + (int64_t)t.f.row[r] * c.out_stride + at, left, narrow<T, S::kEach>(v));
      }
    }
  }
}

// Rows without an adapter: base as it is.
template <class T, int M, bool WIDE>
__device__ __forceinline__ void copy_rows(const Call& c, const Found<M>& f, unsigned rank, unsigned blocks) {
  if (c.base == c.out) return;
  constexpr unsigned V = WIDE ? 16 / sizeof(T) : 1;
  const unsigned packs = (c.channels + V - 1) / V;
  const unsigned begin = (unsigned)((uint64_t)packs * rank / blocks), end = (unsigned)((uint64_t)packs * (rank + 1) / blocks);
  for (unsigned r = threadIdx.x / 32; r < f.count; r += kWarps)
    for (unsigned p = begin + threadIdx.x % 32; p < end; p += 32) {
      Pack<T, V> v;
      if (c.base) {
        v = load_once<T, V>(static_cast<const T*>(c.base) + (int64_t)f.row[r] * c.base_stride + p * V);
      } else {
#pragma unroll
        for (unsigned i = 0; i < V; ++i) v.v[i] = from_float<T>(0.f);
      }
      store_pack<T, V>(static_cast<T*>(c.out) + (int64_t)f.row[r] * c.out_stride + p * V, v);
    }
}

template <class T, int R, int M, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2) low_rank_rows(Call c) {
  using S = Shape<T, R, M>;
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ Found<M> found;
  __shared__ float factor[M * 16];
  const unsigned rank = cluster_rank(), blocks = cluster_size(), number = blockIdx.x / blocks;
  // every block of a cluster finds the same, so all or none of them go on
  if constexpr (M == 1) {
    if (!find_few(c, number, found)) return;
  } else {
    if (!find_sorted(c, number, found)) return;
  }
  if (found.adapter < 0) {
    copy_rows<T, M, WIDE>(c, found, rank, blocks);
    return;
  }
  const Turns<T, R, M, WIDE> turns(c, found, rank, blocks, shared_at(shared));
  for (unsigned i = 0; i < S::kAhead; ++i) turns.copy(i);
  float* const part = reinterpret_cast<float*>(shared + S::kCopies);
  uint32_t* const fragments = reinterpret_cast<uint32_t*>(shared + S::kCopies + S::kPart);
  inner_product<T, R, M, WIDE>(turns, part);
  __syncthreads();
  constexpr int kWritten = S::kAlong / S::kRounds;
  if constexpr (kWritten > 1) {
    for (unsigned i = threadIdx.x; i < M * 16 * R / 4; i += kThreads) {
      float4 s = reinterpret_cast<const float4*>(part)[i];
#pragma unroll
      for (int w = 1; w < kWritten; ++w) {
        const float4 v = reinterpret_cast<const float4*>(part)[w * (M * 16 * R / 4) + i];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      reinterpret_cast<float4*>(part)[i] = s;
    }
  }
  cluster_sync();
  lay_out<T, R, M>(c, found, blocks, part, fragments, factor);
  __syncthreads();
  cluster_arrive();                        // this block has read from the others
  outer_product<T, R, M, WIDE>(turns, fragments, factor);
  cluster_wait();                          // no block leaves while another reads from it
}

// ---------------------------------------------------------------- rows by adapter
// One block: counts the rows of each adapter, lists the units and their rows.  The order of
// an adapter's rows is left to the atomics: no row's result depends on it.
__global__ void __launch_bounds__(kSortThreads) low_rank_sort(const int32_t* ids, uint32_t rows, uint32_t adapters, Unit* units, uint32_t* unit_count,
                                                              int32_t* order) {
  extern __shared__ __align__(16) unsigned char shared[];
  uint32_t* const count = reinterpret_cast<uint32_t*>(shared);      // [adapters + 1], the last for rows without one
  uint32_t* const start = count + adapters + 1;
  uint32_t* const unit = start + adapters + 1;
  __shared__ uint2 sums[32];
  const unsigned t = threadIdx.x, lane = t % 32, warp = t / 32;
  asm volatile("griddepcontrol.launch_dependents;");
  for (unsigned a = t; a <= adapters; a += kSortThreads) count[a] = 0;
  __syncthreads();
  const unsigned turns = (rows + kSortThreads - 1) / kSortThreads;
  auto each = [&](auto what) {              // whole warps; lanes of one adapter go together
    for (unsigned i = 0; i < turns; i += kSortBatch) {
      uint32_t a[kSortBatch];
#pragma unroll
      for (unsigned j = 0; j < kSortBatch; ++j) {
        const unsigned r = (i + j) * kSortThreads + t;
        a[j] = r < rows ? min((uint32_t)ids[r], adapters) : ~0u;
      }
#pragma unroll
      for (unsigned j = 0; j < kSortBatch; ++j) {
        if (i + j >= turns) break;
        const unsigned peers = __match_any_sync(~0u, a[j]);
        if (a[j] != ~0u) what((i + j) * kSortThreads + t, a[j], peers);
      }
    }
  };
  each([&](unsigned, uint32_t a, unsigned peers) {
    if (lane == __ffs(peers) - 1) atomicAdd(&count[a], __popc(peers));
  });
  __syncthreads();
  // exclusive sums of rows and units, a run of adapters a thread
  const unsigned run = (adapters + kSortThreads) / kSortThreads, first = min(t * run, adapters + 1), last = min(first + run, adapters + 1);
  uint2 s = make_uint2(0, 0);
  for (unsigned a = first; a < last; ++a) {
    s.x += count[a];
    s.y += (count[a] + kUnit - 1) / kUnit;
  }
  uint2 before = s;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t x = __shfl_up_sync(~0u, before.x, o), y = __shfl_up_sync(~0u, before.y, o);
    if (lane >= o) before.x += x, before.y += y;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  before.x -= s.x, before.y -= s.y;
  for (unsigned w = 0; w < warp; ++w) before.x += sums[w].x, before.y += sums[w].y;
  for (unsigned a = first; a < last; ++a) {
    start[a] = before.x;
    unit[a] = before.y;
    before.x += count[a];
    before.y += (count[a] + kUnit - 1) / kUnit;
  }
  if (t == kSortThreads - 1) *unit_count = before.y;
  __syncthreads();
  for (unsigned a = warp; a <= adapters; a += kSortThreads / 32)
    for (unsigned u = lane; u * kUnit < count[a]; u += 32)
      units[unit[a] + u] = Unit{a < adapters ? (int32_t)a : -1, start[a] + u * kUnit, min(kUnit, count[a] - u * kUnit), 0};
  __syncthreads();
  each([&](unsigned r, uint32_t a, unsigned peers) {
    const int leader = __ffs(peers) - 1;
    uint32_t at = 0;
    if (lane == leader) at = atomicAdd(&start[a], __popc(peers));
    at = __shfl_sync(peers, at, leader) + __popc(peers & ((1u << lane) - 1));
    order[at] = (int32_t)r;
  });
}

// ------------------------------------------------------------------------ host side
uint32_t padded_rank(uint32_t rank) {
  uint32_t r = 8;
  while (r < rank) r *= 2;
  return r;
}

uint64_t most_units(uint64_t rows, uint32_t adapters) { return rows / kUnit + std::min<uint64_t>(rows, (uint64_t)adapters + 1); }

struct Space {
  uint64_t units, order, bytes;
  Space(uint64_t rows, uint32_t adapters) {
    units = 16;                             // the count of units lies first
    order = units + most_units(rows, adapters) * sizeof(Unit);
    bytes = rows <= kFew ? 0 : order + rows * 4;
  }
};

template <class T, int R, int M, bool WIDE>
void launch_rows(const Call& c, uint64_t units, unsigned cluster, bool early, int device, cudaStream_t stream) {
  constexpr auto kernel = low_rank_rows<T, R, M, WIDE>;
  room<kernel, false>(device);               // L1 keeps what down and up bring
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = cluster;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = (unsigned)(units * cluster);
  config.blockDim = kThreads;
  config.dynamicSmemBytes = Shape<T, R, M>::kBytes;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = early ? 2 : 1;
  check(cudaLaunchKernelEx(&config, kernel, c), "low_rank_rows");
}

template <class T, int M, bool WIDE>
void by_rank(const Call& c, uint64_t units, unsigned cluster, bool early, int device, cudaStream_t stream) {
  switch (padded_rank(c.rank)) {
    case 8: return launch_rows<T, 8, M, WIDE>(c, units, cluster, early, device, stream);
    case 16: return launch_rows<T, 16, M, WIDE>(c, units, cluster, early, device, stream);
    case 32: return launch_rows<T, 32, M, WIDE>(c, units, cluster, early, device, stream);
    case 64: return launch_rows<T, 64, M, WIDE>(c, units, cluster, early, device, stream);
    default: return launch_rows<T, 128, M, WIDE>(c, units, cluster, early, device, stream);
  }
}

template <class T>
void launch(Call c, bool wide, void* workspace, int device, cudaStream_t stream) {
  const unsigned slots = sm_count(device) * 2;
  auto cluster_for = [&](uint64_t units) {
    unsigned n = 8;
    while (n > 1 && units * n > slots) n /= 2;
    return n;
  };
  if (c.rows <= kFew) {
    const unsigned cluster = 8;
    wide ? by_rank<T, 1, true>(c, c.rows, cluster, false, device, stream) : by_rank<T, 1, false>(c, c.rows, cluster, false, device, stream);
    return;
  }
  const Space space(c.rows, c.adapters);
  char* const w = static_cast<char*>(workspace);
  auto* const count = reinterpret_cast<uint32_t*>(w);
  auto* const units = reinterpret_cast<Unit*>(w + space.units);
  auto* const order = reinterpret_cast<int32_t*>(w + space.order);
  c.unit_count = count;
  c.units = units;
  c.order = order;
  room<low_rank_sort>(device);
  low_rank_sort<<<1, kSortThreads, 3 * ((size_t)c.adapters + 1) * 4, stream>>>(c.ids, c.rows, c.adapters, units, count, order);
  check(cudaGetLastError(), "low_rank_sort");
  const uint64_t most = most_units(c.rows, c.adapters);
  const unsigned cluster = cluster_for(c.rows / kUnit + std::min<uint64_t>(c.rows, c.adapters) / 2);
  wide ? by_rank<T, kUnitTiles, true>(c, most, cluster, true, device, stream)
       : by_rank<T, kUnitTiles, false>(c, most, cluster, true, device, stream);
}

// Whether two tensors of rows share memory; columns of one wider tensor do not.
bool overlap(const void* a, int64_t a_stride, uint64_t a_columns, const void* b, int64_t b_stride, uint64_t b_columns, uint64_t rows, uint64_t size) {
  const auto at = reinterpret_cast<uintptr_t>(a), bt = reinterpret_cast<uintptr_t>(b);
  const uint64_t a_end = at + ((rows - 1) * (uint64_t)a_stride + a_columns) * size, b_end = bt + ((rows - 1) * (uint64_t)b_stride + b_columns) * size;
  if (a_end <= bt || b_end <= at) return false;
  if (a_stride != b_stride || a_stride <= 0) return true;
  const uint64_t pitch = (uint64_t)a_stride * size;
  const uint64_t ahead = bt >= at ? (bt - at) % pitch : (pitch - (at - bt) % pitch) % pitch;     // of b's columns before a's next
  return ahead < a_columns * size || ahead + b_columns * size > pitch;
}

bool wide_rows(const void* p, int64_t stride, size_t size) { return aligned(p, 16) && stride * (int64_t)size % 16 == 0; }

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_low_rank_rank(uint32_t rank) { return rank > EPS_B200_LOW_RANK ? 0 : padded_rank(rank); }
uint64_t eps_b200_low_rank_inner(uint32_t inner) { return round_up(inner, 32); }

uint64_t eps_b200_low_rank_workspace(uint64_t rows, uint32_t adapters) {
  return rows < (1ull << 31) && adapters <= EPS_B200_LOW_RANK_ADAPTERS ? Space(rows, adapters).bytes : 0;
}

int eps_b200_low_rank(const EpsB200LowRank* a, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    need(a, "null adapter argument");
    need(known_type(a->type), "unknown element type");
    need(a->adapters > 0 && a->adapters <= EPS_B200_LOW_RANK_ADAPTERS, "1 to 16384 adapters");
    need(a->rank > 0 && a->rank <= EPS_B200_LOW_RANK, "a rank is 1 to 128");
    need(a->inner > 0 && a->inner < (1u << 30) && a->channels > 0 && a->channels < (1u << 30), "inner and channels are 1 to 2^30");
    need(a->rows < (1ull << 31), "too many rows");
    need(a->down && a->up && aligned(a->down, 16) && aligned(a->up, 16), "down and up must be 16-byte aligned");
    if (!a->rows) return;
    need(a->ids && a->x && a->out, "null adapter rows");
    need(a->x_stride >= 0 && a->base_stride >= 0, "row strides are 0 or more");
    need(a->rows == 1 || a->out_stride >= (int64_t)a->channels, "rows of out overlap");
    const size_t size = size_of(a->type);
    need(!overlap(a->out, a->out_stride, a->channels, a->x, a->x_stride, a->inner, a->rows, size), "out overlaps x");
    if (a->base && !(a->base == a->out && (a->rows == 1 || a->base_stride == a->out_stride)))
      need(!overlap(a->out, a->out_stride, a->channels, a->base, a->base_stride, a->channels, a->rows, size), "out overlaps base without being it");
    const Space space(a->rows, a->adapters);
    need(!space.bytes || (a->workspace && aligned(a->workspace, 16) && a->workspace_bytes >= space.bytes), "the adapters' workspace is too small");
    Call c{};
    c.down = a->down;
    c.up = a->up;
    c.x = a->x;
    c.base = a->base;
    c.out = a->out;
    c.scale = a->scale;
    c.ids = a->ids;
    c.x_stride = a->x_stride;
    c.base_stride = a->base_stride;
    c.out_stride = a->out_stride;
    c.rows = (uint32_t)a->rows;
    c.adapters = a->adapters;
    c.rank = a->rank;
    c.inner = a->inner;
    c.padded = (uint32_t)eps_b200_low_rank_inner(a->inner);
    c.channels = a->channels;
    OnDevice on(a->device);
    const bool wide = wide_rows(a->x, a->x_stride, size) && a->inner * size % 16 == 0 && wide_rows(a->out, a->out_stride, size) &&
                      (!a->base || wide_rows(a->base, a->base_stride, size)) && a->channels * size % 16 == 0;
    const auto s = static_cast<cudaStream_t>(stream);
    if (a->type == EPS_B200_F32) launch<float>(c, wide, a->workspace, a->device, s);
    else if (a->type == EPS_B200_BF16) launch<bf16>(c, wide, a->workspace, a->device, s);
    else launch<f16>(c, wide, a->workspace, a->device, s);
  });
}

}  // extern "C"
