// low_rank.cu -- low-rank adapters of many requests at once (eps_b200_low_rank).
//
// Mathematics, for a row t with adapter a:
//   u = down[a] x[t],   out[t] = base[t] + scale[a] * up[a] u
//
// Bound: x and base are read and out is written once, each adapter in use is read once
// for the rows that have it; 2 R operations a value of x and of out are far below what
// the matrix instructions give, so what counts is that loads stay in flight.  Rows are
// taken in units of one adapter and up to 32 rows (64 for larger ranks, whose adapters are
// then read less often; 16 where the call has few).  A cluster works on a unit: its warps
// share out the inner size, each summing its share of u for its rows, the parts are added
// over the warps and, through distributed shared memory, over the blocks; then its warps
// share out the channels.  One launch, no u in memory; a launch before it sorts more than
// 128 rows by adapter.
//
// Fragments need no exchange between lanes: a sum over k may take its terms in any order,
// so each lane of a matrix instruction's row takes 16 consecutive bytes and gives them to
// the places that the instruction has for it, the same for both operands.  In the second
// product the columns are dealt so that a lane ends up with 16 bytes of consecutive
// channels.  Every warp copies what it needs itself, asynchronously and a turn ahead, into
// shared memory of its own, whole lines of 128 bytes of a row at a time; the copies of base
// go on while u is still being added up.
//
//   8189 rows x 4096 x 4096 bf16, rank 16, 32 adapters: 51.4 us, 210 MB at 4.1 TB/s.  7 us of
// it are the sort, finding the units and joining u; x takes 15 and base and out 25, one
// after the other in every block, since all blocks begin at once.  (A plain sum of base and
// x takes 30.)  Rank 64, 4096 rows: 53 us, rank 128: 81, where the matrix instructions and
// the adapters' lines from L2 count.  61 rows with an adapter each: 10.3 us; one row: 6.2.
//
// Precision: 16-bit products are exact and summed in float.  u is not rounded to 16
// bits: it goes on as the sum of two 16-bit values (float16: under a power of two of the
// row, so that its range does not matter).  Floats are cut into three bfloat16 values,
// which is exact but next to the smallest floats, and the six largest of the nine products are summed; the others are
// below 2^-25 of the first.
#include <algorithm>
#include <cmath>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

constexpr unsigned kThreads = 256, kWarps = kThreads / 32;
// Rows that the units are found for without a sort.  4096 x 4096, rank 16: 128 rows of 64
// adapters take 12.8 us and sorted 18.2, of one adapter 14.5 and 11.0; 256 rows 22.0 and
// 18.8, 23.3 and 11.0; 64 rows 8.8 and 17.2, 8.5 and 10.6.
constexpr unsigned kFew = 128;
// 16-row tiles of a unit of sorted rows, by the padded rank: 8192 rows x 4096 x 4096 take
// 50.8 us with 2 and 53.6 with 4 at rank 16, 75 and 65 at rank 32.
__host__ __device__ constexpr int unit_tiles(int rank) { return rank <= 16 ? 2 : 4; }
constexpr unsigned kSortBlocks = 8, kSortThreads = 1024, kSortBatch = 4;      // ids of a thread that are asked for at once

struct Unit {
  int32_t adapter;                        // -1: none
  uint32_t begin, count, unused;          // rows order[begin ..]
};

struct Call {
  const void *down, *up, *x, *base;
  void* out;
  const float* scale;
  const int32_t* ids;
  uint32_t x_stride, base_stride, out_stride;        // bytes
  uint32_t rows, adapters, rank, inner, padded, channels;
  bool x_wide, out_wide;                  // rows of x, and of base and out, begin and end on 16 bytes
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

// How rows begin and end: on 16 bytes (ALIGN 16), on 4, or anywhere (2).  Below 16 `wide`
// says that this tensor's do nevertheless.
// 16 bytes of a row from p on, of which the first `left` values are there; the others are
// 0.
template <class T, int ALIGN>
__device__ __forceinline__ void copy_row(unsigned to, const T* p, int left, bool wide) {
  constexpr int V = 16 / sizeof(T);
  if (ALIGN == 16 || wide) {
    copy_ahead<16>(to, left > 0 ? p : p + min(left, 0), left > 0);
  } else if constexpr (ALIGN == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = i * (int)(4 / sizeof(T));
      copy_ahead<4>(to + 4 * i, left > n ? p + n : p + min(left, 0), left > n);
    }
  } else {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = i < left ? p[i] : from_float<T>(0.f);
    const uint4& x = reinterpret_cast<const uint4&>(r);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
  }
}

template <class T, int ALIGN>
__device__ __forceinline__ void store_row(T* p, int left, const Pack<T, 16 / sizeof(T)>& r, bool wide) {
  constexpr int V = 16 / sizeof(T), E = 4 / sizeof(T);
  if (ALIGN == 16 || wide) {
    if (left > 0) store_pack<T, V>(p, r);
  } else if constexpr (ALIGN == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i * E < left) store_pack<T, E>(p + i * E, reinterpret_cast<const Pack<T, E>*>(&r)[i]);
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
  // 64-byte pieces of a row that a warp takes at once
  static constexpr int kPieces = 2;
  static constexpr int kStep = 4 * kEach * kPieces;              // inner values
  // tiles of a warp in the first product: R / 8 x 4 sums a lane each
  static constexpr int kMost = kFloat ? (R <= 16 ? 2 : 1) : R <= 32 ? 4 : R == 64 ? 2 : 1;
  static constexpr int kTiles = M < kMost ? M : kMost;
  static constexpr int kAcross = M / kTiles;                     // warps side by side over the rows
  static constexpr int kAlong = kWarps / kAcross;                // and along the inner size
  // second product: a lane's ranks of one load, loads, instructions, and 16-bit parts of u
  static constexpr int kRanks = R / 4 < kEach ? R / 4 : kEach;
  static constexpr int kLoads = R / (4 * kRanks);
  static constexpr int kPairsInOne = !kFloat && R == 8;          // both parts of u in one instruction
  static constexpr int kMultiplies = kPairsInOne || kRanks <= 4 ? kLoads : 2 * kLoads;
  static constexpr int kParts = kFloat ? 3 : kPairsInOne ? 1 : 2;
  static constexpr int kRun = 4 * kEach * kPieces;               // channels that a warp takes at once
  static constexpr int kMatrices = kEach / 2;                    // of 8 channels
  static constexpr bool kHold = M * kMultiplies * kParts <= 8;    // u's stay in registers for all runs
  // a warp's copies under way: lines of 128 bytes of x and down, or of base and up
  // down and up are copied ahead too, where shared memory has room: rank 16 of 8192 rows x 4096
  // x 4096 takes 52 us so and 108 without; rank 64 of 4096 rows 52 both ways
  static constexpr bool kWeights = R * sizeof(T) <= 64;
  static constexpr int kRows = M * 16 * 128;
  static constexpr int kDown = kWeights ? R * 128 : 0;
  static constexpr int kUp = kWeights ? kRun * R * (int)sizeof(T) : 0;
  static constexpr int kSlot = kRows + (kDown > kUp ? kDown : kUp);
  static constexpr int kAhead = 2;
  static constexpr size_t kCopies = (size_t)kWarps * kAhead * kSlot;
  // the warps' sums, in two rounds; the first becomes the block's part, the others u's fragments
  static constexpr size_t kPart = (size_t)M * 16 * R * 4;
  static constexpr size_t kFragments = (size_t)M * kMultiplies * kParts * 512;
  static constexpr int kRounds = kAlong > 1 ? 2 : 1;
  static constexpr size_t kSums = kAlong / kRounds * kPart;
  static constexpr size_t kBytes = kCopies + (kSums > kPart + kFragments ? kSums : kPart + kFragments);
};

// Blocks an SM that registers are kept for; shared memory has room for as many.
__host__ __device__ constexpr int blocks_an_sm(int rank, int tiles) {
  return tiles == 1 ? (rank <= 16 ? 3 : rank <= 64 ? 2 : 1) : rank <= 16 ? 2 : 1;
}

// A unit's rows, as every block of the cluster finds them.
template <int M>
struct Found {
  int32_t row[M * 16];
  int32_t adapter;
  uint32_t count;
};

// The unit of this number among few rows, a thread each: rows of one adapter, 16 at most,
// in order.  False if there are fewer units.
__device__ __forceinline__ bool find_few(const Call& c, unsigned number, Found<1>& f) {
  __shared__ __align__(16) int32_t ids[kFew];
  __shared__ uint32_t starts[kWarps];
  __shared__ unsigned first;
  const unsigned t = threadIdx.x, warp = t / 32, lane = t % 32;
  int32_t id = -2;                         // no row
  if (t < c.rows) {
    id = c.ids[t];
    if ((uint32_t)id >= c.adapters) id = -1;
  }
  if (t < kFew) ids[t] = id;
  __syncthreads();
  unsigned before = 0, all = 0;            // rows of the same adapter
  for (unsigned s = 0; s < c.rows; s += 4) {
    const int4 four = *reinterpret_cast<const int4*>(ids + s);
    const int32_t each[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const bool same = each[j] == id;
      before += same && s + j < t;
      all += same;
    }
  }
  const bool start = t < c.rows && before % 16 == 0;
  const unsigned mine = __ballot_sync(~0u, start);
  if (lane == 0) starts[warp] = mine;
  __syncthreads();
  unsigned rank = 0, units = 0;            // of this thread's row among those that begin a unit
#pragma unroll
  for (unsigned w = 0; w < kWarps; ++w) {
    const unsigned n = (unsigned)__popc(starts[w]);
    rank += w < warp ? n : w == warp ? (unsigned)__popc(starts[w] & ((1u << lane) - 1)) : 0;
    units += n;
  }
  if (number >= units) return false;
  if (start && rank == number) {
    f.adapter = id;
    f.count = min(16u, all - before);
    first = before;
  }
  __syncthreads();
  if (t < c.rows && id == f.adapter && before - first < 16) f.row[before - first] = (int32_t)t;
  __syncthreads();
  return true;
}

template <int M>
__device__ __forceinline__ bool find_sorted(const Call& c, unsigned number, Found<M>& f) {
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
// The turns of a warp: steps along the inner size, then runs of channels.  Turn i's copies
// lie in slot i % kAhead; they are asked for in order, so that pointers are moved on and
// not made anew.  A line of 128 bytes is copied by eight lanes, and read as two pieces by
// the four lanes of a matrix row; the halves of every second line change places, so that
// two rows lie in different banks.
template <class T, int R, int M, int ALIGN>
struct Turns {
  using S = Shape<T, R, M>;
  static constexpr unsigned kStepOn = S::kAlong * S::kStep, kRunOn = kWarps * S::kRun;      // from one turn to the next
  const Call& c;
  unsigned tiles, across, steps, runs, slots;
  const T *x, *down, *base;                 // this lane's 16 bytes of a line, of the next turn to be copied
  const char* up;                           // of a run of channels, whose ranks lie one after the other
  int64_t up_left;                          // bytes from there on
  T* out;                                   // this lane's channels of the first run
  int x_left, base_left, out_left;          // columns from there on, some below 0 behind the last
  int32_t line[M * 4], row[M * 2];          // rows i * 4 + lane / 8 and i * 8 + lane / 4 of the unit; -1 behind the last

  __device__ __forceinline__ Turns(const Call& c, const Found<M>& f, unsigned rank, unsigned blocks, unsigned shared) : c(c) {
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, quad = lane % 4, eighth = lane % 8;
    const unsigned along = warp / S::kAcross;
    across = warp % S::kAcross;
    tiles = (f.count + 15) / 16;
    // warps take steps and runs in turn, so that a block reads its rows in long pieces
    const unsigned all = c.padded / S::kStep, stop = (unsigned)((uint64_t)all * (rank + 1) / blocks);
    const unsigned step = (unsigned)((uint64_t)all * rank / blocks) + along;
    steps = across * S::kTiles < tiles && step < stop ? (stop - step + S::kAlong - 1) / S::kAlong : 0;
    const unsigned every = (c.channels + S::kRun - 1) / S::kRun;
    const unsigned run = (unsigned)((uint64_t)every * rank / blocks) + warp, end = (unsigned)((uint64_t)every * (rank + 1) / blocks);
    runs = run < end ? (end - run + kWarps - 1) / kWarps : 0;
    slots = shared + warp * S::kAhead * S::kSlot;
    const unsigned k = step * S::kStep + eighth * S::kEach, channel = run * S::kRun + eighth * S::kEach;
    x = static_cast<const T*>(c.x) + k;
    x_left = (int)c.inner - (int)k;
    base = static_cast<const T*>(c.base) + channel;
    base_left = (int)c.channels - (int)channel;
    const T* const mine = static_cast<const T*>(c.down) + (uint64_t)f.adapter * R * c.padded + step * S::kStep;
    down = S::kWeights ? mine + (uint64_t)(lane / 8) * c.padded + eighth * S::kEach : mine + (uint64_t)g * c.padded + quad * S::kEach;
    const uint64_t at = (uint64_t)run * S::kRun * R * sizeof(T), whole = (uint64_t)c.channels * R * sizeof(T);
    up = static_cast<const char*>(c.up) + f.adapter * whole + at;
    up_left = (int64_t)(whole - at);
    out = static_cast<T*>(c.out) + run * S::kRun + quad * S::kEach;
    out_left = (int)c.channels - (int)(run * S::kRun + quad * S::kEach);
#pragma unroll
    for (int i = 0; i < M * 4; ++i) line[i] = i * 4 + lane / 8 < f.count ? f.row[i * 4 + lane / 8] : -1;
#pragma unroll
    for (int i = 0; i < M * 2; ++i) row[i] = i * 8 + g < f.count ? f.row[i * 8 + g] : -1;
  }
  __device__ __forceinline__ unsigned slot(unsigned i) const { return slots + i % S::kAhead * S::kSlot; }
  static __device__ __forceinline__ const T* row_at(const T* p, int32_t r, uint32_t stride) {
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + (uint64_t)(uint32_t)r * stride);
  }
  // where lines i * 4 + lane / 8 are copied to, and rows i * 8 + lane / 4 are read from
  static __device__ __forceinline__ unsigned line_place(unsigned slot, int i) {
    const unsigned lane = threadIdx.x % 32;
    return slot + i * 512 + lane / 8 * 128 + ((lane % 8) ^ (lane / 8 % 2 * 4)) * 16;
  }
  static __device__ __forceinline__ unsigned piece_place(unsigned slot, int i, int piece) {
    const unsigned lane = threadIdx.x % 32, g = lane / 4;
    return slot + i * 1024 + g * 128 + ((piece * 4 + lane % 4) ^ (g % 2 * 4)) * 16;
  }
  // the 16 bytes number n of a run's ranks; lines of more than two channels are turned by
  // what a matrix's next two columns are ahead
  static __device__ __forceinline__ unsigned up_place(unsigned n) {
    constexpr unsigned kChannels = 128 / (R * sizeof(T));        // of a line
    if constexpr (kChannels > 2) n ^= n / 8 / (S::kEach / kChannels > 0 ? S::kEach / kChannels : 1) % (kChannels / 2) * (2 * R * sizeof(T) / 16);
    return n * 16;
  }

  __device__ __forceinline__ void copy(unsigned i) {
    const unsigned to = slot(i);
    if (i < steps) {
      // rows behind the unit's last are left as they lie: what they give is not used
#pragma unroll
      for (int m = 0; m < M * 4; ++m)
        if (m / (S::kTiles * 4) == (int)across && line[m] >= 0) copy_row<T, ALIGN>(line_place(to, m), row_at(x, line[m], c.x_stride), x_left, c.x_wide);
      x += kStepOn;
      x_left -= kStepOn;
      if constexpr (S::kWeights) {
#pragma unroll
        for (int n = 0; n < R / 4; ++n) copy_ahead<16>(line_place(to + S::kRows, n), down + (size_t)n * 4 * c.padded, true);
        down += kStepOn;
      }
    } else if (i < steps + runs) {
      if (c.base) {
#pragma unroll
        for (int m = 0; m < M * 4; ++m)
          if (line[m] >= 0) copy_row<T, ALIGN>(line_place(to, m), row_at(base, line[m], c.base_stride), base_left, c.out_wide);
        base += kRunOn;
        base_left -= kRunOn;
      }
      if constexpr (S::kWeights) {
#pragma unroll
        for (int n = 0; n < S::kUp / 512; ++n) {
          const unsigned at = (n * 32 + threadIdx.x % 32) * 16;
          copy_ahead<16>(to + S::kRows + up_place(n * 32 + threadIdx.x % 32), (int64_t)at < up_left ? up + at : static_cast<const char*>(c.up), (int64_t)at < up_left);
        }
        up += (size_t)kRunOn * R * sizeof(T);
        up_left -= (int64_t)kRunOn * R * sizeof(T);
      }
    }
    copies_end();
  }
  // Waits for turn i's copies, all lanes'.
  __device__ __forceinline__ void wait() const {
    copies_wait<S::kAhead - 1>();
    __syncwarp();
  }
  // Asks for turn i + kAhead's, when all lanes have read turn i's.
  __device__ __forceinline__ void copy_behind(unsigned i) {
    __syncwarp();
    copy(i + S::kAhead);
  }
};

// ------------------------------------------------------------------- u = down x
template <class T, int R, int M, int ALIGN>
__device__ __forceinline__ void inner_product(Turns<T, R, M, ALIGN>& t, float* sums) {
  using S = Shape<T, R, M>;
  using P = Pack<T, S::kEach>;
  constexpr int kCols = R / 8;
  float acc[S::kTiles][kCols][4] = {};
  for (unsigned i = 0; i < t.steps; ++i) {
    P weight[S::kWeights ? S::kPieces : 1][kCols], rows[S::kPieces][S::kTiles][2];
    auto load_weight = [&](int q) {
#pragma unroll
      for (int n = 0; n < kCols; ++n) weight[0][n] = load_pack<T, S::kEach>(t.down + (size_t)n * 8 * t.c.padded + q * 4 * S::kEach);
    };
    if constexpr (!S::kWeights) load_weight(0);
    t.wait();
    const unsigned from = t.slot(i) + t.across * S::kTiles * 2048;
#pragma unroll
    for (int q = 0; q < S::kPieces; ++q) {
#pragma unroll
      for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) rows[q][m][h] = own_shared<P>(t.piece_place(from, m * 2 + h, q));
      if constexpr (S::kWeights) {
#pragma unroll
        for (int n = 0; n < kCols; ++n) weight[q][n] = own_shared<P>(t.piece_place(t.slot(i) + S::kRows, n, q));
      }
    }
    t.copy_behind(i);
#pragma unroll
    for (int q = 0; q < S::kPieces; ++q) {
      const auto& x = rows[q];
      if constexpr (!S::kWeights)
        if (q > 0) load_weight(q);
      const auto& d = weight[S::kWeights ? q : 0];
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
              for (int k = 0; k < 3; ++k) a[k][2 * e + h] = p[k];
            }
#pragma unroll
          for (int n = 0; n < kCols; ++n) {
            uint32_t b0[3], b1[3];
            cut(d[n].v[0], d[n].v[1], b0);
            cut(d[n].v[2], d[n].v[3], b1);
            // summed apart and added in float: the matrix instruction's sums are cut off, not rounded
            float part[4] = {};
#pragma unroll
            for (int k = 0; k < 6; ++k) multiply<bf16>(part, a[kTerms[k][0]], b0[kTerms[k][1]], b1[kTerms[k][1]]);
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
    if constexpr (!S::kWeights) t.down += t.kStepOn;
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
template <class T, int R, int M, int ALIGN>
__device__ __forceinline__ void outer_product(Turns<T, R, M, ALIGN>& t, const uint32_t* fragments, const float* factor) {
  using S = Shape<T, R, M>;
  using P = Pack<T, S::kRanks>;
  using O = Pack<T, S::kEach>;
  const Call& c = t.c;
  const unsigned lane = threadIdx.x % 32, g = lane / 4;
  auto fragment = [&](int m, int q, int p) { return reinterpret_cast<const uint4*>(fragments)[((m * S::kMultiplies + q) * S::kParts + p) * 32 + lane]; };
  uint4 u[S::kHold ? M : 1][S::kHold ? S::kMultiplies : 1][S::kHold ? S::kParts : 1];
  if constexpr (S::kHold) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int q = 0; q < S::kMultiplies; ++q)
#pragma unroll
        for (int p = 0; p < S::kParts; ++p) u[m][q][p] = fragment(m, q, p);
  }
  float by[M * 2];
#pragma unroll
  for (int m = 0; m < M * 2; ++m) by[m] = factor[m * 8 + g];
  for (unsigned i = t.steps; i < t.steps + t.runs; ++i) {
    // column g of matrix j of a piece is its channel kEach (g / 2) + 2 j + g % 2
    auto up_offset = [&](int piece, int j, int l) {
      const unsigned channel = piece * 4 * S::kEach + g / 2 * S::kEach + j * 2 + g % 2;
      return (channel * R + l * 4 * S::kRanks + lane % 4 * S::kRanks) * (unsigned)sizeof(T);
    };
    t.wait();
    O before[M * 2][S::kPieces];
#pragma unroll
    for (int m = 0; m < M * 2; ++m)
#pragma unroll
      for (int q = 0; q < S::kPieces; ++q)
        if (m / 2 < t.tiles && c.base) before[m][q] = own_shared<O>(t.piece_place(t.slot(i), m, q));
    P held[S::kWeights ? S::kPieces : 1][S::kMatrices][S::kLoads];
    auto hold = [&](int piece) {
#pragma unroll
      for (int j = 0; j < S::kMatrices; ++j)
#pragma unroll
        for (int l = 0; l < S::kLoads; ++l) {
          const unsigned at = up_offset(piece, j, l);
          if constexpr (S::kWeights) held[piece][j][l] = own_shared<P>(t.slot(i) + S::kRows + t.up_place(at / 16) + at % 16);
          else held[0][j][l] = load_pack<T, S::kRanks>(reinterpret_cast<const T*>((int64_t)at < t.up_left ? t.up + at : static_cast<const char*>(c.up)));
        }
    };
    hold(0);
    if constexpr (S::kWeights) hold(1);
    t.copy_behind(i);
#pragma unroll
    for (int e = 0; e < M * S::kPieces; ++e) {
      const int m = e % M, piece = e / M;
      if constexpr (!S::kWeights)
        if (e == M) hold(1);
      if (m >= t.tiles) continue;
      float acc[S::kMatrices][4] = {};
#pragma unroll
      for (int l = 0; l < S::kLoads; ++l) {
#pragma unroll
        for (int k = 0; k < (S::kRanks <= 4 ? 1 : 2); ++k) {
          const int n = S::kRanks <= 4 ? l : 2 * l + k;
          uint32_t a[S::kParts][4];
#pragma unroll
          for (int p = 0; p < S::kParts; ++p) {
            uint4 w;
            if constexpr (S::kHold) w = u[m][n][p];
            else w = fragment(m, n, p);
            a[p][0] = w.x, a[p][1] = w.y, a[p][2] = w.z, a[p][3] = w.w;
          }
#pragma unroll
          for (int j = 0; j < S::kMatrices; ++j) {
            const P d = held[S::kWeights ? piece : 0][j][l];
            if constexpr (S::kFloat) {
              uint32_t b0[3], b1[3] = {0, 0, 0};
              cut(d.v[0], d.v[1], b0);
              if constexpr (S::kRanks == 4) cut(d.v[2], d.v[3], b1);
              float part[4] = {};
#pragma unroll
              for (int k6 = 0; k6 < 6; ++k6) multiply<bf16>(part, a[kTerms[k6][0]], b0[kTerms[k6][1]], b1[kTerms[k6][1]]);
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
        const int32_t r = t.row[m * 2 + h];
        if (r < 0) continue;
        float v[S::kEach], plus[S::kEach];
#pragma unroll
        for (int j = 0; j < S::kMatrices; ++j) v[2 * j] = acc[j][2 * h], v[2 * j + 1] = acc[j][2 * h + 1];
        if (c.base) {
          widen(before[m * 2 + h][piece], plus);
          vfma<S::kEach>(v, v, by[m * 2 + h], plus);
        } else {
          vmul<S::kEach>(v, v, by[m * 2 + h]);
        }
        store_row<T, ALIGN>(const_cast<T*>(t.row_at(t.out, r, c.out_stride)) + piece * 4 * S::kEach, t.out_left - piece * 4 * S::kEach, narrow<T, S::kEach>(v), c.out_wide);
      }
    }
    if constexpr (!S::kWeights) {
      t.up += (size_t)t.kRunOn * R * sizeof(T);
      t.up_left -= (int64_t)t.kRunOn * R * sizeof(T);
    }
    t.out += t.kRunOn;
    t.out_left -= t.kRunOn;
  }
}

// Rows without an adapter: base as it is.  A block has few of them, so each thread asks for
// kMany packs before it stores the first (one at a time the rows without an adapter took
// longer than all others).
template <class T, int M, int ALIGN>
__device__ __forceinline__ void copy_rows(const Call& c, const Found<M>& f, unsigned rank, unsigned blocks) {
  if (c.base == c.out) return;
  constexpr unsigned V = ALIGN / sizeof(T) > 0 ? ALIGN / sizeof(T) : 1, kMany = 8;
  const unsigned packs = (c.channels + V - 1) / V;
  const unsigned begin = (unsigned)((uint64_t)packs * rank / blocks), end = (unsigned)((uint64_t)packs * (rank + 1) / blocks);
  each_pack<kMany>(begin, end, f.count, threadIdx.x, kThreads, [&](const unsigned (&row)[kMany], const unsigned (&pack)[kMany], const bool (&there)[kMany]) {
    Pack<T, V> v[kMany];
    uint32_t to[kMany];
#pragma unroll
    for (unsigned j = 0; j < kMany; ++j) {
      to[j] = (uint32_t)f.row[row[j]];
      if (c.base) {
        v[j] = load_pack<T, V>(reinterpret_cast<const T*>(static_cast<const char*>(c.base) + (uint64_t)to[j] * c.base_stride) + pack[j] * V);
      } else {
#pragma unroll
        for (unsigned e = 0; e < V; ++e) v[j].v[e] = from_float<T>(0.f);
      }
    }
#pragma unroll
    for (unsigned j = 0; j < kMany; ++j)
      if (there[j]) store_pack<T, V>(reinterpret_cast<T*>(static_cast<char*>(c.out) + (uint64_t)to[j] * c.out_stride) + pack[j] * V, v[j]);
  });
}

template <class T, int R, int M, int ALIGN>
__global__ void __launch_bounds__(kThreads, blocks_an_sm(R, M)) low_rank_rows(Call c) {
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
    copy_rows<T, M, ALIGN>(c, found, rank, blocks);
    return;
  }
  Turns<T, R, M, ALIGN> turns(c, found, rank, blocks, shared_at(shared));
  for (unsigned i = 0; i < S::kAhead; ++i) turns.copy(i);
  float* const part = reinterpret_cast<float*>(shared + S::kCopies);
  uint32_t* const fragments = reinterpret_cast<uint32_t*>(shared + S::kCopies + S::kPart);
  inner_product<T, R, M, ALIGN>(turns, part);
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
  outer_product<T, R, M, ALIGN>(turns, fragments, factor);
  cluster_wait();                          // no block leaves while another reads from it
}

// ---------------------------------------------------------------- rows by adapter
// One cluster, a run of rows a block: counts the rows of each adapter, lists the units and
// their rows.  The order of an adapter's rows is left to the atomics: no row's result
// depends on it.
__global__ void __cluster_dims__(kSortBlocks) __launch_bounds__(kSortThreads) low_rank_sort(const int32_t* ids, uint32_t rows, uint32_t adapters,
                                                                                            uint32_t unit_rows, Unit* units, uint32_t* unit_count,
                                                                                            int32_t* order) {
  extern __shared__ __align__(16) unsigned char shared[];
  uint32_t* const count = reinterpret_cast<uint32_t*>(shared);      // [adapters + 1], the last for rows without one
  uint32_t* const start = count + adapters + 1;                     // [adapters + 2]
  uint32_t* const unit = start + adapters + 2;                      // [adapters + 1]
  __shared__ uint2 sums[32];
  const unsigned t = threadIdx.x, lane = t % 32, warp = t / 32, rank = cluster_rank();
  asm volatile("griddepcontrol.launch_dependents;");
  for (unsigned a = t; a <= adapters; a += kSortThreads) count[a] = 0;
  __syncthreads();
  const unsigned begin = (uint64_t)rows * rank / kSortBlocks, end = (uint64_t)rows * (rank + 1) / kSortBlocks;
  auto each = [&](auto what) {              // whole warps; lanes of one adapter go together
    for (unsigned i = begin; i < end; i += kSortBatch * kSortThreads) {
      uint32_t a[kSortBatch];
#pragma unroll
      for (unsigned j = 0; j < kSortBatch; ++j) {
        const unsigned r = i + j * kSortThreads + t;
        a[j] = r < end ? min((uint32_t)ids[r], adapters) : ~0u;
      }
#pragma unroll
      for (unsigned j = 0; j < kSortBatch; ++j) {
        if (i + j * kSortThreads >= end) break;
        const unsigned peers = __match_any_sync(~0u, a[j]);
        if (a[j] != ~0u) what(i + j * kSortThreads + t, a[j], peers);
      }
    }
  };
  each([&](unsigned, uint32_t a, unsigned peers) {
    if (lane == __ffs(peers) - 1) atomicAdd(&count[a], __popc(peers));
  });
  cluster_sync();
  // rows of each adapter, and of those in the blocks before this one; a run of adapters a thread
  const unsigned run = (adapters + kSortThreads) / kSortThreads, first = min(t * run, adapters + 1), last = min(first + run, adapters + 1);
  uint2 s = make_uint2(0, 0);
  for (unsigned a = first; a < last; ++a) {
    uint32_t all = 0, before = 0;
#pragma unroll
    for (unsigned b = 0; b < kSortBlocks; ++b) {
      const uint32_t n = cluster_load(count + a, b);
      before += b < rank ? n : 0;
      all += n;
    }
    start[a] = all;
    unit[a] = before;
    s.x += all;
    s.y += (all + unit_rows - 1) / unit_rows;
  }
  cluster_sync();                          // the counts have been read: each becomes the place of this block's next row
  uint2 ahead = s;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t x = __shfl_up_sync(~0u, ahead.x, o), y = __shfl_up_sync(~0u, ahead.y, o);
    if (lane >= o) ahead.x += x, ahead.y += y;
  }
  if (lane == 31) sums[warp] = ahead;
  __syncthreads();
  ahead.x -= s.x, ahead.y -= s.y;
  for (unsigned w = 0; w < warp; ++w) ahead.x += sums[w].x, ahead.y += sums[w].y;
  for (unsigned a = first; a < last; ++a) {
    const uint32_t all = start[a];
    count[a] = unit[a] + ahead.x;
    start[a] = ahead.x;
    unit[a] = ahead.y;
    ahead.x += all;
    ahead.y += (all + unit_rows - 1) / unit_rows;
  }
  if (t == kSortThreads - 1) {
    start[adapters + 1] = rows;
    if (rank == 0) *unit_count = ahead.y;
  }
  __syncthreads();
  for (unsigned a = warp * kSortBlocks + rank; a <= adapters; a += kSortThreads / 32 * kSortBlocks) {
    const uint32_t from = start[a], n = start[a + 1] - from;
    for (unsigned u = lane; u * unit_rows < n; u += 32)
      units[unit[a] + u] = Unit{a < adapters ? (int32_t)a : -1, from + u * unit_rows, min(unit_rows, n - u * unit_rows), 0};
  }
  each([&](unsigned r, uint32_t a, unsigned peers) {
    const int leader = __ffs(peers) - 1;
    uint32_t at = 0;
    if (lane == leader) at = atomicAdd(&count[a], __popc(peers));
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

uint64_t most_units(uint64_t rows, uint32_t adapters, unsigned unit_rows) {
  return rows / unit_rows + std::min<uint64_t>(rows, (uint64_t)adapters + 1);
}

struct Space {
  uint64_t units, order, bytes;
  Space(uint64_t rows, uint32_t adapters) {
    units = 16;                             // the count of units lies first
    order = units + most_units(rows, adapters, 32) * sizeof(Unit);      // the smallest units are the most
    bytes = rows <= kFew ? 0 : order + rows * 4;
  }
};

template <class T, int R, int M, int ALIGN>
void launch_rows(const Call& c, uint64_t units, unsigned cluster, bool early, int device, cudaStream_t stream) {
  constexpr auto kernel = low_rank_rows<T, R, M, ALIGN>;
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

// FEW: units of few rows, found without a sort.
template <class T, bool FEW, int ALIGN>
void by_rank(const Call& c, uint64_t units, unsigned cluster, int device, cudaStream_t stream) {
  auto go = [&](auto r) {
    constexpr int R = decltype(r)::value;
    launch_rows<T, R, FEW ? 1 : unit_tiles(R), ALIGN>(c, units, cluster, !FEW, device, stream);
  };
  switch (padded_rank(c.rank)) {
    case 8: return go(std::integral_constant<int, 8>{});
    case 16: return go(std::integral_constant<int, 16>{});
    case 32: return go(std::integral_constant<int, 32>{});
    case 64: return go(std::integral_constant<int, 64>{});
    default: return go(std::integral_constant<int, 128>{});
  }
}

template <class T>
void launch(Call c, int align, void* workspace, int device, cudaStream_t stream) {
  const unsigned sms = sm_count(device);
  const int rank = (int)padded_rank(c.rank);
  // The blocks of a unit: as many as keep all blocks at once on the SMs, and a quarter
  // more.  A block has some 3 us of its own (finding its unit, joining u): 79 units of 1531
  // floats rows take 28 us with 4 blocks each, 34 with 2 and 40 with 1; 190 units of 2000
  // rows 15 us with one, 18 with 2 and 27 with 4.
  auto cluster_for = [&](uint64_t units, unsigned each) {
    unsigned n = 8;
    while (n > 1 && units * n > sms * each * 5 / 4) n /= 2;
    return n;
  };
  auto run = [&](auto few, uint64_t units, unsigned cluster) {
    constexpr bool FEW = decltype(few)::value;
    if (align == 16) by_rank<T, FEW, 16>(c, units, cluster, device, stream);
    else if constexpr (sizeof(T) == 4) by_rank<T, FEW, 4>(c, units, cluster, device, stream);
    else align == 4 ? by_rank<T, FEW, 4>(c, units, cluster, device, stream) : by_rank<T, FEW, 2>(c, units, cluster, device, stream);
  };
  if (c.rows <= kFew) return run(std::true_type{}, c.rows, cluster_for(c.rows, 2));
  const Space space(c.rows, c.adapters);
  char* const w = static_cast<char*>(workspace);
  auto* const count = reinterpret_cast<uint32_t*>(w);
  auto* const units = reinterpret_cast<Unit*>(w + space.units);
  auto* const order = reinterpret_cast<int32_t*>(w + space.order);
  c.unit_count = count;
  c.units = units;
  c.order = order;
  const unsigned unit_rows = unit_tiles(rank) * 16;
  room<low_rank_sort>(device);
  low_rank_sort<<<kSortBlocks, kSortThreads, (3 * (size_t)c.adapters + 4) * 4, stream>>>(c.ids, c.rows, c.adapters, unit_rows, units, count, order);
  check(cudaGetLastError(), "low_rank_sort");
  const uint64_t most = most_units(c.rows, c.adapters, unit_rows);
  const unsigned cluster = cluster_for(c.rows / unit_rows + std::min<uint64_t>(c.rows, c.adapters) / 2, blocks_an_sm(rank, unit_tiles(rank)));
  run(std::false_type{}, most, cluster);
}

// Whether every row begins and ends on n bytes.
bool rows_on(size_t n, const void* p, int64_t stride, uint64_t columns, size_t size) {
  return aligned(p, n) && stride * (int64_t)size % (int64_t)n == 0 && columns * size % n == 0;
}

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

uint64_t eps_b200_low_rank_rank(uint32_t rank) { return rank > EPS_B200_LOW_RANK ? 0 : padded_rank(rank); }
uint64_t eps_b200_low_rank_inner(uint32_t inner) { return round_up(inner, 64); }

uint64_t eps_b200_low_rank_workspace(uint64_t rows, uint32_t adapters) {
  return rows < (1ull << 31) && adapters <= EPS_B200_LOW_RANK_ADAPTERS ? Space(rows, adapters).bytes : 0;
}

int eps_b200_low_rank(const EpsB200LowRank* a, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    need(a, "null adapter argument");
    need(known_type(a->type), "unknown element type");
    need(a->adapters > 0 && a->adapters <= EPS_B200_LOW_RANK_ADAPTERS, "1 to 16384 adapters");
    need(a->rank > 0 && a->rank <= EPS_B200_LOW_RANK, "a rank is 1 to 128");
    need(a->inner > 0 && a->inner < (1u << 30) && a->channels > 0 && a->channels < (1u << 30), "inner and channels are below 2^30");
    need(a->rows < (1ull << 31), "too many rows");
    need(a->down && a->up && aligned(a->down, 16) && aligned(a->up, 16), "down and up must be 16-byte aligned");
    if (!a->rows) return;
    need(a->ids && a->x && a->out, "null adapter rows");
    need(a->x_stride >= 0 && a->base_stride >= 0, "row strides are 0 or more");
    need(a->rows == 1 || (a->x_stride < (1 << 30) && a->base_stride < (1 << 30) && a->out_stride < (1 << 30)), "row strides are below 2^30");
    need(a->rows == 1 || a->out_stride >= (int64_t)a->channels, "rows of out overlap");
    const size_t size = size_of(a->type);
    need(aligned(a->x, size) && aligned(a->base, size) && aligned(a->out, size), "rows are not aligned to their type");
    need(words(a->scale, a->ids), "scale and ids are 4-byte aligned");
    need(!overlap({a->out, a->out_stride, a->channels}, {a->x, a->x_stride, a->inner}, a->rows, size), "out overlaps x");
    if (a->base && !(a->base == a->out && (a->rows == 1 || a->base_stride == a->out_stride)))
      need(!overlap({a->out, a->out_stride, a->channels}, {a->base, a->base_stride, a->channels}, a->rows, size), "out overlaps base without being it");
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
    // a stride of one row alone is never used
    c.x_stride = a->rows == 1 ? 0 : (uint32_t)(a->x_stride * (int64_t)size);
    c.base_stride = a->rows == 1 ? 0 : (uint32_t)(a->base_stride * (int64_t)size);
    c.out_stride = a->rows == 1 ? 0 : (uint32_t)(a->out_stride * (int64_t)size);
    c.rows = (uint32_t)a->rows;
    c.adapters = a->adapters;
    c.rank = a->rank;
    c.inner = a->inner;
    c.padded = (uint32_t)eps_b200_low_rank_inner(a->inner);
    c.channels = a->channels;
    OnDevice on(a->device);
    auto x_on = [&](size_t n) { return rows_on(n, a->x, a->x_stride, a->inner, size); };
    auto out_on = [&](size_t n) {
      return rows_on(n, a->out, a->out_stride, a->channels, size) && (!a->base || rows_on(n, a->base, a->base_stride, a->channels, size));
    };
    c.x_wide = x_on(16);
    c.out_wide = out_on(16);
    const int align = c.x_wide && c.out_wide ? 16 : x_on(4) && out_on(4) ? 4 : 2;
    const auto s = static_cast<cudaStream_t>(stream);
    if (a->type == EPS_B200_F32) launch<float>(c, align, a->workspace, a->device, s);
    else if (a->type == EPS_B200_BF16) launch<bf16>(c, align, a->workspace, a->device, s);
    else launch<f16>(c, align, a->workspace, a->device, s);
  });
}

}  // extern "C"
