// block_norm.cu -- the norms before and after a block, fused with its gate and
// residual scale (eps_b200_block_norm, eps_b200_block_norm_backward).
//
// Mathematics (per row of D values; N = rms or layer norm, weight w, bias b):
//   n = N_post(y),  h = x + c a n  with a = activation(gate), c = scale * channel_scale,
//   z = N_pre(h)
// backward, with r the reciprocal deviation, hat the normed value before its weight:
//   q = dz w_pre,   dh' = dh + r2 (q - [layer] mean(q) - hhat mean(q hhat))
//   dgate = c dh' n a',   dn = c dh' a,   p = dn w_post
//   dy = r1 (p - [layer] mean(p) - yhat mean(p yhat)),   dx = dh'
//   dw_pre = sum_rows dz hhat, db_pre = sum_rows dz, dw_post = sum_rows dn yhat,
//   db_post = sum_rows dn, dchannel = sum_rows scale dh' a n
//
// Bound: bytes.  Forward reads x, y, gate and writes h, z; backward reads dh, dz,
// h, y, gate and writes dx, dy, dgate: each value once.  What stands in the way is
// the chain of each row (reduce, use, reduce again) and the instructions around it,
// so: a row's values are copied into shared memory while its predecessors are worked
// on; the statistics of the next row are reduced together with this row's sums, which
// halves the barriers; and a kernel has no branch on what is given: missing weights
// are staged as ones, missing tensors as zeros.
//
// A row belongs to a group of lanes (a power of two up to a warp, or a whole block),
// V consecutive elements a lane NIT times.
//
// Measured at 16381 x 2048 bf16: forward (rms, element gate) 69 us, 4.9 TB/s; backward
// (layer norm, every gradient) 145 us, 3.7 TB/s, and 8 us to add up the blocks' column
// sums; in float 109 us, 6.2 TB/s, and (rms) 213 us, 5.0 TB/s, both with the sums.  Forward before its rows were copied ahead: 127 us; with the copies but two
// barriers more a row, 97.  Backward is bound by instructions at 16 warps an SM, whose
// registers the 40 column sums of a lane fill.
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "dense.cuh"

namespace eps_b200 {
namespace dense {
namespace {

struct Norm {
  unsigned columns;
  uint64_t rows;
  unsigned width;                  // lanes of a row
  int layer, gate, activation, post_norm, pre_norm, narrow;   // narrow: parameters have the type of y
  float epsilon, scale, inverse_columns;
  const void *x, *y, *g, *h, *dh, *dz;
  int64_t xs, ys, gs, hs, dhs, dzs;
  const void *post_w, *post_b, *channel, *pre_w, *pre_b;
  void *out_h, *out_z, *dx, *dy, *dg;
  int64_t out_hs, out_zs, dxs, dys, dgs;
  float* partial;                  // [blocks][5][columns]
  int want;                        // bit i: column sum i is wanted
  const void* somewhere;           // 16-byte aligned device memory, for copies of nothing
};

// The column sums of the backward pass, in this order in `partial`.
enum { kPostWeight, kPostBias, kChannel, kPreWeight, kPreBias, kSums };

// 1 / (1 + 2^-t) with t = g log2 e: two instructions of the special-function unit, each
// good to two units of the last place; subnormal powers count as 0, which 1 + hides.
// Rounding t costs another |g| / 2 units.  Gates of 16 bits have a unit 2^13 or 2^16 as
// large and go without (a gate of -20 is off by some ten units of float); a float block
// takes what t lost, e = t - g log2 e, into account as 2^e = 1 + e ln 2.  Where t is
// not finite, or so large that the result is 0 or 1, there is nothing to add.
template <int V, bool FINE>
__device__ __forceinline__ void sigmoid(const float (&g)[V], float (&s)[V]) {
  constexpr float kLog = 1.4426950408889634f, kLogRest = 1.925963e-8f;      // log2 e and what its float lacks
  vmul<V>(s, g, kLog);
  [[maybe_unused]] float e[V];
  if constexpr (FINE) {
    vfma<V>(e, g, -kLog, s);
    vfma<V>(e, g, -kLogRest, e);
    vfma<V>(e, e, 0.6931471805599453f, 1.f);
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = fabsf(s[j]) < 256.f ? e[j] : 1.f;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s[j]) : "f"(-s[j]));
  if constexpr (FINE) vfma<V>(s, s, e, 1.f);
  else vadd<V>(s, s, 1.f);
#pragma unroll
  for (int j = 0; j < V; ++j) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(s[j]));
}

// act(g) and, where SLOPE, its derivative for V values; the choice is made once for
// all of them.
template <int V, bool SLOPE, bool FINE>
__device__ __forceinline__ void activate(const float (&g)[V], int activation, float (&a)[V], float (&slope)[V]) {
  if (activation == EPS_B200_ACT_SIGMOID) {
    sigmoid<V, FINE>(g, a);
    if (SLOPE) {
#pragma unroll
      for (int j = 0; j < V; ++j) slope[j] = fmaf(-a[j], a[j], a[j]);
    }
  } else if (activation == EPS_B200_ACT_SILU) {
    float s[V];
    sigmoid<V, FINE>(g, s);
    vmul<V>(a, g, s);
    if (SLOPE) {
#pragma unroll
      for (int j = 0; j < V; ++j) slope[j] = fmaf(a[j], 1.f - s[j], s[j]);
    }
  } else if (activation == EPS_B200_ACT_TANH) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a[j] = tanhf(g[j]);
      slope[j] = fmaf(-a[j], a[j], 1.f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a[j] = g[j];
      slope[j] = 1.f;
    }
  }
}

template <bool FINE>
__device__ __forceinline__ float activate_one(float g, int activation, float* slope) {
  float v[1] = {g}, a[1], s[1];
  activate<1, true, FINE>(v, activation, a, s);
  *slope = s[0];
  return a[0];
}

// A lane's own record in shared memory: bytes rounded up to an odd number of 16-byte
// words, so that eight neighbouring lanes reading word k of theirs meet all banks once.
__host__ __device__ constexpr unsigned record(unsigned bytes) { return ((bytes + 15) / 16 | 1) * 16; }

// A parameter vector's V elements from column c on: 1 or 0 (`missing`) where there is
// none, 0 behind the last column.
template <class T, int V>
__device__ __forceinline__ void parameter(const Norm& n, const void* p, unsigned c, float missing, float (&r)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = c < n.columns ? missing : 0.f;
  if (!p || c >= n.columns) return;
  if (n.narrow) widen(load_pack<T, V>(static_cast<const T*>(p) + c), r);
  else widen(load_pack<float, V>(static_cast<const float*>(p) + c), r);
}

// The four vectors that a row is worked on with, as a lane uses them.  Where a lane
// has few columns it writes them down in its record once, in float: rows then read
// them at fixed places.
//   forward   0: c w_post   1: c b_post   2: w_pre    3: b_pre
//   backward  0: w_post     1: b_post     2: w_pre    3: c
constexpr int kVectors = 4;

template <class T, int V, int NIT, bool STAGED, bool FORWARD>
struct Parameters {
  static constexpr unsigned kRecord = STAGED ? record(kVectors * NIT * V * 4) : 0;
  const Norm& n;
  unsigned lane;
  float* mine;             // STAGED: the lane's record, [kVectors][NIT][V]

  __device__ __forceinline__ Parameters(const Norm& norm, unsigned l, void* room)
      : n(norm), lane(l), mine(reinterpret_cast<float*>(static_cast<char*>(room) + threadIdx.x * kRecord)) {
    if constexpr (STAGED) {
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          float r[V];
          read(k, i, r);
          Pack<float, V> x;
#pragma unroll
          for (int j = 0; j < V; ++j) x.v[j] = r[j];
          *reinterpret_cast<Pack<float, V>*>(mine + (k * NIT + i) * V) = x;
        }
    }
  }
  __device__ __forceinline__ void read(int k, int i, float (&r)[V]) const {
    const unsigned c = (i * n.width + lane) * V;
    if (k == 0) parameter<T, V>(n, n.post_w, c, 1.f, r);
    if (k == 1) parameter<T, V>(n, n.post_b, c, 0.f, r);
    if (k == 2) parameter<T, V>(n, n.pre_w, c, 1.f, r);
    if (k == 3) FORWARD ? parameter<T, V>(n, n.pre_b, c, 0.f, r) : parameter<T, V>(n, n.channel, c, 1.f, r);
    if (FORWARD && k < 2) {
      float s[V];
      parameter<T, V>(n, n.channel, c, 1.f, s);
      vmul<V>(r, r, s);
    }
    if (FORWARD ? k < 2 : k == 3) vmul<V>(r, r, n.scale);
  }
  __device__ __forceinline__ void get(int k, int i, float (&r)[V]) const {
    if constexpr (STAGED) {
      const Pack<float, V> x = *reinterpret_cast<const Pack<float, V>*>(mine + (k * NIT + i) * V);
#pragma unroll
      for (int j = 0; j < V; ++j) r[j] = x.v[j];
    } else {
      read(k, i, r);
    }
  }
};

template <int V>
__device__ __forceinline__ float total(const float (&v)[V]) {
  if constexpr (V == 8) {
    float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    vadd<4>(a, a, b);
    float c[2] = {a[0], a[1]}, d[2] = {a[2], a[3]};
    vadd<2>(c, c, d);
    return c[0] + c[1];
  } else {
    float s = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) s += v[j];
    return s;
  }
}

// (v - mean) * r: the difference first, since v r and mean r may both be large.
template <int V>
__device__ __forceinline__ void centre(float (&v)[V], float mean, float r) {
  vadd<V>(v, v, -mean);
  vmul<V>(v, v, r);
}

// A lane's part of a row's mean, or of its mean square about `mean`.  It divides by
// the columns itself, so that sums cannot overflow across lanes where the mean does
// not; what it holds behind the last column does not count.
template <int V, int NIT, bool SQUARE>
__device__ __forceinline__ float share(const Norm& n, unsigned lane, const float (&v)[NIT][V], float mean) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const float inside = (i * n.width + lane) * V < n.columns ? n.inverse_columns : 0.f;
    if constexpr (SQUARE) {
      float d[V];
      vadd<V>(d, v[i], -mean);
      vmul<V>(d, d, d);
      s = fmaf(total<V>(d), inside, s);
    } else {
      s = fmaf(total<V>(v[i]), inside, s);
    }
  }
  return s;
}

// How rows reach the lanes.  Blocks walk the rows, and in the two ways with a ring a
// row's values are under way two rows ahead, past registers and L1:
//   kBulk    a block's row: one thread copies each tensor's row whole;
//   kLanes   rows of a few lanes: a lane copies its own 16 bytes of each tensor and
//            reads back only those, so that no barrier is involved;
//   kDirect  without 16-byte alignment, or with several packs a lane: loaded as needed.
// Lanes behind the row's end, rows behind the last one and missing tensors read zeros.
enum Way { kDirect, kLanes, kBulk };
constexpr unsigned kAhead = 2, kSlots = kAhead + 1;
constexpr unsigned kLanesThreads = 128;      // of a block where rows have up to 32 lanes

template <int V, int NIT, int P>
constexpr Way kWay = V < 4 || NIT > 1 ? kDirect : P == 1 ? kLanes : kBulk;

__device__ __forceinline__ void copy16(unsigned to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// What both directions share: the block's rows, and the lane's.  Where a block has one
// row at a time, all but `lane` is the same for all threads, and written so that the
// compiler can tell: it then costs no registers of the lanes.
template <Way WAY, int P>
struct Walk {
  unsigned lane, passes, mine;             // passes of the block, and how many of them have a row for this lane
  uint64_t stride, row;
  __device__ __forceinline__ explicit Walk(const Norm& n) {
    if constexpr (P > 1) {
      lane = threadIdx.x;
      stride = gridDim.x;
      row = blockIdx.x;
      passes = mine = (unsigned)((n.rows - row + stride - 1) / stride);
    } else {
      lane = threadIdx.x % n.width;
      const unsigned groups = blockDim.x / n.width;
      stride = (uint64_t)gridDim.x * groups;
      const uint64_t first = (uint64_t)blockIdx.x * groups;     // blocks do not outnumber groups of rows
      row = first + threadIdx.x / n.width;
      passes = (unsigned)((n.rows - first + stride - 1) / stride);
      mine = row < n.rows ? (unsigned)((n.rows - row + stride - 1) / stride) : 0;
    }
  }
};

// One tensor of those rows.  In a slot of the ring a tensor takes V * sizeof(T) bytes
// a thread: as its row lies (kBulk), or in planes of 16 bytes a lane (kLanes).
template <class T, int V, int NIT, Way WAY>
struct Source {
  static constexpr unsigned kBytes = V * sizeof(T);
  const char* p;           // the next row
  int64_t step;            // bytes from one row of the walk to the next
  bool there;              // the tensor is given

  template <class W>
  __device__ __forceinline__ Source(const Norm& n, const W& w, const void* tensor, int64_t stride) {
    there = tensor != nullptr;
    p = there ? static_cast<const char*>(tensor) + (int64_t)w.row * stride * (int64_t)sizeof(T) : static_cast<const char*>(n.somewhere);
    step = there ? (int64_t)w.stride * stride * (int64_t)sizeof(T) : 0;
  }
  // to: the tensor's bytes in a slot, a shared address
  __device__ __forceinline__ void ask(unsigned to, bool live, unsigned lane) {
#pragma unroll
    for (unsigned k = 0; k < kBytes / 16; ++k)
      copy16(to + (k * kLanesThreads + threadIdx.x) * 16, p + (live && there ? lane * kBytes + k * 16 : 0), live && there);
    p += step;
  }
  __device__ __forceinline__ void ask_row(unsigned to, unsigned row_bytes, uint64_t* barrier) {
    if (there) bulk_copy(to, p, row_bytes, barrier);
  }
  __device__ __forceinline__ void asked_row() { p += step; }
  __device__ __forceinline__ void get(const Norm& n, unsigned from, bool live, unsigned lane, float (&r)[NIT][V]) {
    if constexpr (WAY != kDirect) {
      Pack<T, V> x;
#pragma unroll
      for (unsigned k = 0; k < kBytes / 16; ++k) {
        uint4& q = reinterpret_cast<uint4*>(&x)[k];
        const unsigned at = from + (WAY == kBulk ? threadIdx.x * kBytes + k * 16 : (k * kLanesThreads + threadIdx.x) * 16);
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(at) : "memory");
      }
      widen(x, r[0]);
    } else {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const unsigned c = (i * n.width + lane) * V;
        Pack<T, V> x{};
        if (live && there && c < n.columns) x = load_pack<T, V>(reinterpret_cast<const T*>(p) + c);      // read again: kept in L1
        widen(x, r[i]);
      }
    }
  }
  __device__ __forceinline__ void next() {
    if constexpr (WAY == kDirect) p += step;
  }
};

// One tensor that is written.
template <class T, int V, int NIT>
struct Sink {
  char* p;
  int64_t step;
  template <class W>
  __device__ __forceinline__ Sink(const W& w, void* tensor, int64_t stride) {
    p = static_cast<char*>(tensor) + (tensor ? (int64_t)w.row * stride * (int64_t)sizeof(T) : 0);
    step = tensor ? (int64_t)w.stride * stride * (int64_t)sizeof(T) : 0;
  }
  __device__ __forceinline__ void put(const Norm& n, int i, unsigned lane, bool live, const float (&v)[V]) const {
    const unsigned c = (i * n.width + lane) * V;
    if (live && p && c < n.columns) store_pack<T, V>(reinterpret_cast<T*>(p) + c, narrow<T, V>(v));
  }
  __device__ __forceinline__ void next() { p += step; }
};

// The ring's shared memory before its first copy: zeros, which stay where nothing is
// copied, and the slots' barriers.
template <Way WAY>
__device__ __forceinline__ void open_ring(char* ring, unsigned bytes, uint64_t (&arrived)[kSlots]) {
  if constexpr (WAY == kBulk) {
    for (unsigned i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(ring + i) = uint4{};
    if (threadIdx.x < kSlots) barrier_init(arrived + threadIdx.x, 1);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
}

// A place in the ring: a slot, its bytes, and the parity of its barrier's phase.
struct Place {
  unsigned index = 0, bytes = 0, phase = 0;
  __device__ __forceinline__ void next(unsigned slot_bytes) {
    bytes += slot_bytes;
    if (++index == kSlots) { index = bytes = 0; phase ^= 1; }
  }
};

// Whether the row at `at` has arrived; what a lane reads then is its own row's.
template <Way WAY>
__device__ __forceinline__ bool arrive(uint64_t (&arrived)[kSlots], const Place& at, bool expected, bool gave_up) {
  if constexpr (WAY == kLanes) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
  if constexpr (WAY == kBulk) return !expected || barrier_wait(arrived + at.index, at.phase, gave_up);
  return true;
}

// No block ends, or writes to the ring, with copies into it in flight.  Where no wait ran
// out, all rows that were asked for have arrived.
template <Way WAY>
__device__ __forceinline__ void close_ring(uint64_t (&arrived)[kSlots], bool good, unsigned asked) {
  if constexpr (WAY == kLanes) asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (WAY == kBulk) {
    if (good || threadIdx.x != 0) return;
    for (unsigned i = asked > kSlots ? asked - kSlots : 0; i < asked; ++i) barrier_wait(arrived + i % kSlots, i / kSlots & 1);
  }
}

template <class TX, class TY, int V>
__host__ __device__ constexpr unsigned forward_bytes() { return V * (sizeof(TX) + 2 * sizeof(TY)); }     // of a thread in a slot
template <class TX, class TY, int V>
__host__ __device__ constexpr unsigned backward_bytes() { return V * (2 * sizeof(TX) + 3 * sizeof(TY)); }

template <class TX, class TY, int V, int NIT, int P, int GATE>
__global__ void __launch_bounds__(512) block_norm_forward(const Norm n) {
  constexpr Way kHow = kWay<V, NIT, P>;
  constexpr bool kStaged = V * NIT <= 8, kFine = std::is_same_v<TY, float>;
  using Given = Parameters<TY, V, NIT, kStaged, true>;
  extern __shared__ __align__(16) char room[];       // the staged parameters, then the ring
  __shared__ float shared[kRowSumShared];
  __shared__ uint64_t arrived[kSlots];
  const unsigned slot_bytes = forward_bytes<TX, TY, V>() * blockDim.x;
  clear_row_sums<P>(shared);
  open_ring<kHow>(room + Given::kRecord * blockDim.x, kSlots * slot_bytes, arrived);
  unsigned turn = 0;
  const Walk<kHow, P> w(n);
  const unsigned lane = w.lane;
  // the tensors' places in a slot
  const unsigned at_x = shared_at(room) + Given::kRecord * blockDim.x, at_y = at_x + V * (unsigned)sizeof(TX) * blockDim.x,
                 at_g = at_y + V * (unsigned)sizeof(TY) * blockDim.x;
  Source<TX, V, NIT, kHow> x(n, w, n.x, n.xs);
  Source<TY, V, NIT, kHow> y(n, w, n.y, n.ys), gate(n, w, GATE == EPS_B200_GATE_ELEMENT ? n.g : nullptr, n.gs);
  Sink<TX, V, NIT> h(w, n.out_h, n.out_hs);
  Sink<TY, V, NIT> z(w, n.out_z, n.out_zs);
  bool good = true;          // no wait has run out; after one that has, nothing is copied or waited for long, and results are NaN
  unsigned asked = 0;
  Place fill, here;
  auto ask = [&] {
    const bool live = good && asked < w.mine;
    asked += live;
    if constexpr (kHow == kBulk) {
      if (threadIdx.x == 0 && live) {
        const unsigned bx = n.columns * (unsigned)sizeof(TX), by = n.columns * (unsigned)sizeof(TY);
        barrier_expect(arrived + fill.index, bx + (y.there ? by : 0) + (GATE == EPS_B200_GATE_ELEMENT ? by : 0));
        x.ask_row(at_x + fill.bytes, bx, arrived + fill.index);
        y.ask_row(at_y + fill.bytes, by, arrived + fill.index);
        if (GATE == EPS_B200_GATE_ELEMENT) gate.ask_row(at_g + fill.bytes, by, arrived + fill.index);
      }
      x.asked_row();
      y.asked_row();
      gate.asked_row();
    } else if constexpr (kHow == kLanes) {
      x.ask(at_x + fill.bytes, live && lane * V < n.columns, lane);
      y.ask(at_y + fill.bytes, live && lane * V < n.columns, lane);
      if (GATE == EPS_B200_GATE_ELEMENT) gate.ask(at_g + fill.bytes, live && lane * V < n.columns, lane);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    fill.next(slot_bytes);
  };
  ask();
  ask();
  const Given p(n, lane, room);
  const bool layer = n.layer, post = n.post_norm;
  const TY* row_gates = static_cast<const TY*>(n.g) + w.row;

  // the first row's y and its statistics
  float v[NIT][V], mean = 0.f, r = 1.f;
  good = arrive<kHow>(arrived, here, true, false);
  y.get(n, at_y, 0 < w.mine, lane, v);
  y.next();
  {
    float s[1];
    if (layer) {
      s[0] = share<V, NIT, false>(n, lane, v, 0.f);
      row_sum<1, P>(s, n.width, shared, turn);
      mean = s[0];
    }
    s[0] = share<V, NIT, true>(n, lane, v, mean);
    row_sum<1, P>(s, n.width, shared, turn);
    r = __frsqrt_rn(s[0] + n.epsilon);
  }
  for (unsigned pass = 0; pass < w.passes; ++pass) {
    const bool live = pass < w.mine;
    if (!post) { mean = 0.f; r = 1.f; }
    if (!good) r = NAN;
    // the slot of the row before: every lane has passed a barrier since it read it
    if constexpr (kHow != kDirect) ask();
    float t[NIT][V];
    x.get(n, at_x + here.bytes, live, lane, t);
    x.next();
    float open = 1.f, unused;
    if (GATE == EPS_B200_GATE_ROW) {
      if (live) open = activate_one<kFine>(to_float(*row_gates), n.activation, &unused);
      row_gates += w.stride;
    }
    float g[NIT][V];
    if (GATE == EPS_B200_GATE_ELEMENT) {
      gate.get(n, at_g + here.bytes, live, lane, g);
      gate.next();
    }
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float a[V], b[V];
      p.get(0, i, a);
      p.get(1, i, b);
      centre<V>(v[i], mean, r);
      vfma<V>(v[i], v[i], a, b);
      if (GATE == EPS_B200_GATE_ELEMENT) {
        activate<V, false, kFine>(g[i], n.activation, a, b);
        vfma<V>(v[i], v[i], a, t[i]);
      } else {
        vfma<V>(v[i], v[i], open, t[i]);
      }
      h.put(n, i, lane, live, v[i]);
    }
    h.next();
    // the next row's y; its statistics together with this row's h's
    here.next(slot_bytes);
    good &= arrive<kHow>(arrived, here, pass + 1 < w.passes, !good);
    y.get(n, at_y + here.bytes, pass + 1 < w.mine, lane, t);
    y.next();
    float s[2], m = 0.f;
    mean = 0.f;
    if (layer) {
      s[0] = share<V, NIT, false>(n, lane, v, 0.f);
      s[1] = share<V, NIT, false>(n, lane, t, 0.f);
      row_sum<2, P>(s, n.width, shared, turn);
      m = s[0];
      mean = s[1];
    }
    s[0] = share<V, NIT, true>(n, lane, v, m);
    s[1] = share<V, NIT, true>(n, lane, t, mean);
    row_sum<2, P>(s, n.width, shared, turn);
    const float rh = __frsqrt_rn(s[0] + n.epsilon);
    r = __frsqrt_rn(s[1] + n.epsilon);
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float a[V], b[V];
      p.get(2, i, a);
      p.get(3, i, b);
      centre<V>(v[i], m, rh);
      vfma<V>(v[i], v[i], a, b);
      z.put(n, i, lane, live, v[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = t[i][j];
    }
    z.next();
  }
  close_ring<kHow>(arrived, good, asked);
}

// The column sums of a lane stay in registers where a lane has few columns, else in
// shared memory (each lane its own columns: no conflict, no atomic).  They leave a
// block once; block_norm_columns adds the blocks up in order.  Single elements are read
// as needed, so a second block an SM hides their latency (572 -> 284 us at 27148 x 1207).
template <class TX, class TY, int V, int NIT, int P, int GATE>
__global__ void __launch_bounds__(512, V == 1 && NIT <= 4 ? 2 : 1) block_norm_gradient(const Norm n) {
  constexpr int N = V * NIT;
  constexpr Way kHow = kWay<V, NIT, P>;
  constexpr bool kHeld = N <= 8, kFine = std::is_same_v<TY, float>;
  using Given = Parameters<TY, V, NIT, kHeld, false>;
  extern __shared__ __align__(16) char room[];      // the staged parameters, then the ring; in the end the sums
  float* const sums = reinterpret_cast<float*>(room);      // [wanted][N][blockDim.x]
  __shared__ float shared[kRowSumShared];
  __shared__ uint64_t arrived[kSlots];
  const unsigned slot_bytes = backward_bytes<TX, TY, V>() * blockDim.x;
  clear_row_sums<P>(shared);
  open_ring<kHow>(room + Given::kRecord * blockDim.x, kSlots * slot_bytes, arrived);
  unsigned turn = 0;
  const Walk<kHow, P> w(n);
  const unsigned lane = w.lane, groups = blockDim.x / n.width;
  const unsigned cell = N * blockDim.x;
  const unsigned wanted = __popc(n.want);
  auto slot_of = [&](int k) { return __popc(n.want & ((1 << k) - 1)); };      // of a wanted sum
  float held[kHeld ? kSums : 1][kHeld ? NIT : 1][V];
  if constexpr (kHeld) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) held[k][j / V][j % V] = 0.f;
  } else {
    for (unsigned i = threadIdx.x; i < wanted * cell; i += blockDim.x) sums[i] = 0.f;
    __syncthreads();
  }
  // column sums k of the lane's pack i grow by a * b, or by a
  auto add = [&](int k, int i, const auto& a, const auto& b) {
    if constexpr (kHeld) {
      if constexpr (std::is_same_v<std::decay_t<decltype(b)>, float>) vadd<V>(held[k][i], held[k][i], a);
      else vfma<V>(held[k][i], a, b, held[k][i]);
    } else if (n.want >> k & 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float* const s = sums + slot_of(k) * cell + (i * V + j) * blockDim.x + threadIdx.x;
        *s = fmaf(part<V>(a, j), part<V>(b, j), *s);
      }
    }
  };

  const unsigned bx = V * (unsigned)sizeof(TX) * blockDim.x, by = V * (unsigned)sizeof(TY) * blockDim.x;
  const unsigned at_dh = shared_at(room) + Given::kRecord * blockDim.x, at_h = at_dh + bx, at_dz = at_h + bx, at_y = at_dz + by, at_g = at_y + by;
  Source<TX, V, NIT, kHow> sdh(n, w, n.dh, n.dhs), sh(n, w, n.dz ? n.h : nullptr, n.hs);
  Source<TY, V, NIT, kHow> sdz(n, w, n.dz, n.dzs), sy(n, w, n.y, n.ys), sg(n, w, GATE == EPS_B200_GATE_ELEMENT ? n.g : nullptr, n.gs);
  Sink<TX, V, NIT> dx(w, n.dx, n.dxs);
  Sink<TY, V, NIT> dy(w, n.dy, n.dys), dg(w, GATE == EPS_B200_GATE_ELEMENT ? n.dg : nullptr, n.dgs);
  bool good = true;          // no wait has run out; after one that has, nothing is copied or waited for long, and results are NaN
  unsigned asked = 0;
  Place fill, here;
  auto ask = [&] {
    const bool live = good && asked < w.mine;
    asked += live;
    if constexpr (kHow == kBulk) {
      if (threadIdx.x == 0 && live) {
        const unsigned rx = n.columns * (unsigned)sizeof(TX), ry = n.columns * (unsigned)sizeof(TY);
        uint64_t* const b = arrived + fill.index;
        barrier_expect(b, (sdh.there ? rx : 0) + (sdz.there ? rx + ry : 0) + (sy.there ? ry : 0) + (GATE == EPS_B200_GATE_ELEMENT ? ry : 0));
        sdh.ask_row(at_dh + fill.bytes, rx, b);
        sh.ask_row(at_h + fill.bytes, rx, b);
        sdz.ask_row(at_dz + fill.bytes, ry, b);
        sy.ask_row(at_y + fill.bytes, ry, b);
        if (GATE == EPS_B200_GATE_ELEMENT) sg.ask_row(at_g + fill.bytes, ry, b);
      }
      sdh.asked_row();
      sh.asked_row();
      sdz.asked_row();
      sy.asked_row();
      sg.asked_row();
    } else if constexpr (kHow == kLanes) {
      sdh.ask(at_dh + fill.bytes, live && lane * V < n.columns, lane);
      sh.ask(at_h + fill.bytes, live && lane * V < n.columns, lane);
      sdz.ask(at_dz + fill.bytes, live && lane * V < n.columns, lane);
      sy.ask(at_y + fill.bytes, live && lane * V < n.columns, lane);
      if (GATE == EPS_B200_GATE_ELEMENT) sg.ask(at_g + fill.bytes, live && lane * V < n.columns, lane);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    fill.next(slot_bytes);
  };
  ask();
  ask();
  const Given p(n, lane, room);
  const bool layer = n.layer, post = n.post_norm;
  const TY* row_gates = static_cast<const TY*>(n.g) + w.row;

  // the first row's statistics, of h and of y
  float mean[2] = {0.f, 0.f}, r[2];
  float h[NIT][V], y[NIT][V];
  good = arrive<kHow>(arrived, here, true, false);
  sh.get(n, at_h, 0 < w.mine, lane, h);
  sy.get(n, at_y, 0 < w.mine, lane, y);
  {
    float s[2];
    if (layer) {
      s[0] = share<V, NIT, false>(n, lane, h, 0.f);
      s[1] = share<V, NIT, false>(n, lane, y, 0.f);
      row_sum<2, P>(s, n.width, shared, turn);
      mean[0] = s[0];
      mean[1] = s[1];
    }
    s[0] = share<V, NIT, true>(n, lane, h, mean[0]);
    s[1] = share<V, NIT, true>(n, lane, y, mean[1]);
    row_sum<2, P>(s, n.width, shared, turn);
    r[0] = __frsqrt_rn(s[0] + n.epsilon);
    r[1] = __frsqrt_rn(s[1] + n.epsilon);
  }
  for (unsigned pass = 0; pass < w.passes; ++pass) {
    const bool live = pass < w.mine, more = pass + 1 < w.mine;
    if (!post) { mean[1] = 0.f; r[1] = 1.f; }
    if (!good) r[0] = r[1] = NAN;
    // the slot of the row before: every lane has passed a barrier since it read it
    if constexpr (kHow != kDirect) ask();
    const unsigned now = here.bytes;
    here.next(slot_bytes);
    good &= arrive<kHow>(arrived, here, pass + 1 < w.passes, !good);
    float d[NIT][V], q[NIT][V], s[4];
    // through the norm after
    sdz.get(n, at_dz + now, live, lane, q);
    sdz.next();
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float u[V];
      p.get(2, i, u);
      centre<V>(h[i], mean[0], r[0]);
      add(kPreWeight, i, q[i], h[i]);
      add(kPreBias, i, q[i], 1.f);
      vmul<V>(q[i], q[i], u);               // 0 behind the row's end
      s[0] += total<V>(q[i]);
      vmul<V>(u, q[i], h[i]);
      s[1] += total<V>(u);
    }
    // the next row's means, or mean squares, of h and y
    sh.next();
    sy.next();
    {
      float t[NIT][V];
      sh.get(n, at_h + here.bytes, more, lane, t);
      s[2] = layer ? share<V, NIT, false>(n, lane, t, 0.f) : share<V, NIT, true>(n, lane, t, 0.f);
      sy.get(n, at_y + here.bytes, more, lane, t);
      s[3] = layer ? share<V, NIT, false>(n, lane, t, 0.f) : share<V, NIT, true>(n, lane, t, 0.f);
    }
    row_sum<4, P>(s, n.width, shared, turn);
    const float mq = layer ? s[0] * n.inverse_columns : 0.f, mh = s[1] * n.inverse_columns, next_h = s[2], next_y = s[3];
    sdh.get(n, at_dh + now, live, lane, d);
    sdh.next();
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      vfma<V>(h[i], h[i], -mh, q[i]);
      vadd<V>(h[i], h[i], -mq);
      vfma<V>(d[i], h[i], r[0], d[i]);
      dx.put(n, i, lane, live, d[i]);
    }
    dx.next();
    // through the scale, the gate and the norm before
    float open = 1.f, slope1 = 0.f, sum_gate[1] = {0.f};
    if (GATE == EPS_B200_GATE_ROW && live) open = activate_one<kFine>(to_float(*row_gates), n.activation, &slope1);
    float g[NIT][V];
    if (GATE == EPS_B200_GATE_ELEMENT) {
      sg.get(n, at_g + now, live, lane, g);
      sg.next();
    }
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float nv[V], a[V], slope[V], u[V];
      p.get(0, i, u);
      p.get(1, i, nv);
      centre<V>(y[i], mean[1], r[1]);
      vfma<V>(nv, y[i], u, nv);             // what the gate sees
      if (GATE == EPS_B200_GATE_ELEMENT) {
        activate<V, true, kFine>(g[i], n.activation, a, slope);
        vmul<V>(a, a, d[i]);
      } else {
        vmul<V>(a, d[i], open);
      }
      add(kChannel, i, a, nv);              // without n.scale, which the block's sums take at the end
      p.get(3, i, q[i]);
      if (GATE != EPS_B200_GATE_NONE) {
        vmul<V>(nv, nv, d[i]);
        vmul<V>(nv, nv, q[i]);
        if (GATE == EPS_B200_GATE_ELEMENT) {
          vmul<V>(nv, nv, slope);
          dg.put(n, i, lane, live, nv);
        } else {
          sum_gate[0] += total<V>(nv);
        }
      }
      vmul<V>(q[i], q[i], a);
      add(kPostWeight, i, q[i], y[i]);
      add(kPostBias, i, q[i], 1.f);
      vmul<V>(q[i], q[i], u);               // 0 behind the row's end
      s[0] += total<V>(q[i]);
      vmul<V>(u, q[i], y[i]);
      s[1] += total<V>(u);
    }
    dg.next();
    if (GATE == EPS_B200_GATE_ROW) {
      row_sum<1, P>(sum_gate, n.width, shared, turn);
      if (live && lane == 0 && n.dg) static_cast<TY*>(n.dg)[row_gates - static_cast<const TY*>(n.g)] = from_float<TY>(sum_gate[0] * slope1);
      row_gates += w.stride;
    }
    const float r_now = r[1];
    sh.get(n, at_h + here.bytes, more, lane, h);
    if (layer) {
      float t[NIT][V];
      mean[0] = next_h;
      mean[1] = next_y;
      s[2] = share<V, NIT, true>(n, lane, h, mean[0]);
      sy.get(n, at_y + here.bytes, more, lane, t);
      s[3] = share<V, NIT, true>(n, lane, t, mean[1]);
      row_sum<4, P>(s, n.width, shared, turn);
    } else {
      row_sum<2, P>(reinterpret_cast<float(&)[2]>(s), n.width, shared, turn);
      s[2] = next_h;
      s[3] = next_y;
    }
    const float mp = layer && post ? s[0] * n.inverse_columns : 0.f, my = post ? s[1] * n.inverse_columns : 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      vfma<V>(q[i], y[i], -my, q[i]);
      vadd<V>(q[i], q[i], -mp);
      vmul<V>(q[i], q[i], r_now);
      dy.put(n, i, lane, live, q[i]);
    }
    dy.next();
    r[0] = __frsqrt_rn(s[2] + n.epsilon);
    r[1] = __frsqrt_rn(s[3] + n.epsilon);
    sy.get(n, at_y + here.bytes, more, lane, y);
  }
  close_ring<kHow>(arrived, good, asked);
  if (!wanted) return;
  if constexpr (kHeld) {
    __syncthreads();        // the staged parameters and the ring lie there
#pragma unroll
    for (int k = 0; k < kSums; ++k)
      if (n.want >> k & 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) sums[slot_of(k) * cell + j * blockDim.x + threadIdx.x] = held[k][j / V][j % V];
      }
  }
  __syncthreads();
  // the block's groups of lanes in order, then out
  for (unsigned c = threadIdx.x; c < n.columns; c += blockDim.x) {
    const unsigned at = c / V, i = at / n.width, l = at % n.width, j = c % V;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (!(n.want >> k & 1)) continue;
      float t = 0.f;
      for (unsigned g = 0; g < groups; ++g) t += sums[slot_of(k) * cell + (i * V + j) * blockDim.x + g * n.width + l];
      n.partial[((uint64_t)blockIdx.x * kSums + k) * n.columns + c] = k == kChannel ? t * n.scale : t;
    }
  }
}

struct Columns {
  const float* partial;
  float* out[kSums];
  unsigned columns, blocks;
};

// out[k][c] = the sum over blocks of partial[block][k][c]: 32 columns a block of
// threads, 32 runs of blocks, joined in order.
constexpr unsigned kRuns = 32;
__global__ void __launch_bounds__(32 * kRuns) block_norm_columns(const Columns p) {
  __shared__ float part[kRuns][33];
  const unsigned l = threadIdx.x % 32, c = blockIdx.x * 32 + l, run = threadIdx.x / 32, k = blockIdx.y;
  if (!p.out[k]) return;
  float s = 0.f;
  if (c < p.columns) {
#pragma unroll 8
    for (unsigned b = run; b < p.blocks; b += kRuns) s += p.partial[((uint64_t)b * kSums + k) * p.columns + c];
  }
  part[run][l] = s;
  __syncthreads();
  s = part[l][run];                      // lane: run, warp: column
#pragma unroll
  for (int o = 16; o; o /= 2) s += __shfl_xor_sync(~0u, s, o);
  if (l == 0 && blockIdx.x * 32 + run < p.columns) p.out[k][blockIdx.x * 32 + run] = s;
}

// How a row is spread: V elements a lane, `nit` times, over `width` lanes.
struct Spread { int v, nit; unsigned width, threads; };

// The elements of a wide access of these types.
template <class TX, class TY>
constexpr int kWide = std::is_same_v<TY, float> ? 4 : 8;

// A lane holds one wide pack where that fits 512 lanes (and, for a float residual
// of a 16-bit block, the shared memory of 256), else up to sixteen elements; without
// 16-byte alignment four single ones up to 2048 columns, where the column sums still
// fit registers and two blocks an SM (27148 x 1207 bfloat16, backward: 284 us, against
// 663 with sixteen a lane and the sums in shared memory), and sixteen beyond.
Spread spread_of(unsigned columns, int residual, int type, bool wide) {
  Spread s{};
  s.v = !wide ? 1 : type == EPS_B200_F32 ? 4 : 8;
  const unsigned packs = (unsigned)ceil_div(columns, s.v);
  if (!wide) s.nit = packs <= 32 ? 1 : packs <= 2048 ? 4 : 16;
  else s.nit = packs <= (residual != type ? 256 : 512) ? 1 : packs <= 1024 ? 2 : 4;
  const unsigned lanes = (unsigned)ceil_div(packs, s.nit);
  if (lanes <= 32) {
    s.width = 1;
    while (s.width < lanes) s.width *= 2;
    s.threads = kLanesThreads;
  } else {
    s.width = s.threads = (unsigned)round_up(lanes, 32);
  }
  return s;
}

constexpr unsigned kMostBlocks = 8 * 160;   // of the gradient: 8 an SM, 160 SMs

// Blocks that fit the GPU at once, or fewer where the rows need fewer.
template <auto Kernel>
unsigned resident(int device, const Spread& s, size_t shared, uint64_t rows, unsigned most) {
  room<Kernel>(device);
  uint64_t n = (uint64_t)sm_count(device) * blocks_each<Kernel>(device, s.threads, shared);
  if (n > most) n = most;
  const uint64_t all = ceil_div(rows, s.threads / s.width);
  return (unsigned)(all < n ? all : n);
}

template <class TX, class TY, int V, int NIT, int P, int GATE>
void forward(const Norm& n, const Spread& s, int device, cudaStream_t stream) {
  constexpr auto kKernel = block_norm_forward<TX, TY, V, NIT, P, GATE>;
  const unsigned lane = Parameters<TY, V, NIT, V * NIT <= 8, true>::kRecord + (kWay<V, NIT, P> != kDirect ? kSlots * forward_bytes<TX, TY, V>() : 0);
  kKernel<<<resident<kKernel>(device, s, lane * s.threads, n.rows, ~0u), s.threads, lane * s.threads, stream>>>(n);
  check(cudaGetLastError(), "block_norm");
}

// The number of blocks, which is the number of partial sums.
template <class TX, class TY, int V, int NIT, int P, int GATE>
unsigned backward(const Norm& n, const Spread& s, int device, uint64_t space, cudaStream_t stream) {
  constexpr auto kKernel = block_norm_gradient<TX, TY, V, NIT, P, GATE>;
  constexpr bool kRing = kWay<V, NIT, P> != kDirect;
  const unsigned held = (unsigned)__builtin_popcount((unsigned)n.want) * NIT * V * 4;
  const unsigned walked = Parameters<TY, V, NIT, V * NIT <= 8, false>::kRecord + (kRing ? kSlots * backward_bytes<TX, TY, V>() : 0);
  const unsigned shared = (walked > held ? walked : held) * s.threads;       // the sums take the others' place in the end
  const unsigned blocks = resident<kKernel>(device, s, shared, n.rows, kMostBlocks);
  need(!n.want || space >= (uint64_t)blocks * kSums * n.columns * 4, "block norm workspace too small");
  kKernel<<<blocks, s.threads, shared, stream>>>(n);
  check(cudaGetLastError(), "block_norm_backward");
  return blocks;
}

template <int N> using Int = std::integral_constant<int, N>;

template <class F>
void by_gate(int gate, F f) {
  gate == EPS_B200_GATE_NONE ? f(Int<EPS_B200_GATE_NONE>{}) : gate == EPS_B200_GATE_ROW ? f(Int<EPS_B200_GATE_ROW>{})
                                                                                        : f(Int<EPS_B200_GATE_ELEMENT>{});
}

// f(V, NIT, P): P as row_sum has it.
template <int W, class F>
void by_spread(const Spread& s, F f) {
  const unsigned warps = s.width / 32;
  if (s.v == W) {
    if (s.nit == 4) { if constexpr (W == 4) f(Int<W>{}, Int<4>{}, Int<16>{}); }
    else if (s.nit == 2) f(Int<W>{}, Int<2>{}, Int<16>{});
    else if (warps <= 1) f(Int<W>{}, Int<1>{}, Int<1>{});
    else if (warps <= 4) f(Int<W>{}, Int<1>{}, Int<4>{});
    else if (warps <= 8) f(Int<W>{}, Int<1>{}, Int<8>{});
    else f(Int<W>{}, Int<1>{}, Int<16>{});
  } else {
    if (s.nit == 1) f(Int<1>{}, Int<1>{}, Int<1>{});
    else if (s.nit == 16) f(Int<1>{}, Int<16>{}, Int<16>{});
    else if (warps <= 1) f(Int<1>{}, Int<4>{}, Int<1>{});
    else warps <= 8 ? f(Int<1>{}, Int<4>{}, Int<8>{}) : f(Int<1>{}, Int<4>{}, Int<16>{});
  }
}

template <class F>
void by_type(int residual, int type, F f) {
  if (type == EPS_B200_F32) f(float{}, float{});
  else if (type == EPS_B200_BF16) residual == EPS_B200_F32 ? f(float{}, bf16{}) : f(bf16{}, bf16{});
  else residual == EPS_B200_F32 ? f(float{}, f16{}) : f(f16{}, f16{});
}

// Whether rows at `p` with this stride (elements) and type take 16-byte accesses.
bool rows_wide(const void* p, int64_t stride, int type) {
  return !p || (aligned(p, 16) && stride * (int64_t)size_of(type) % 16 == 0);
}

Norm checked(const EpsB200BlockNorm* a) {
  need(a, "null block norm arguments");
  need(a->kind == EPS_B200_NORM_RMS || a->kind == EPS_B200_NORM_LAYER, "unknown kind of norm");
  need(a->gate_kind >= EPS_B200_GATE_NONE && a->gate_kind <= EPS_B200_GATE_ELEMENT, "unknown kind of gate");
  need(a->activation >= EPS_B200_ACT_NONE && a->activation <= EPS_B200_ACT_TANH, "unknown activation");
  need(known_type(a->type) && known_type(a->residual_type) && known_type(a->parameter_type), "unknown element type");
  need(a->residual_type == a->type || a->residual_type == EPS_B200_F32, "the residual has the block's type or float32");
  need(a->parameter_type == a->type || a->parameter_type == EPS_B200_F32, "parameters have the block's type or float32");
  need(a->columns > 0 && a->columns <= EPS_B200_BLOCK_NORM_COLUMNS, "columns out of range");
  need(a->rows < (1ull << 31), "too many rows");
  need(a->epsilon > 0.f && a->epsilon < 1e30f, "epsilon must be positive");
  need(a->scale == a->scale, "the scale is not a number");
  // tensors without rows may have no address
  need(!a->rows || (a->gate_kind != EPS_B200_GATE_NONE) == (a->gate != nullptr), "gate and gate_kind disagree");
  need(!a->rows || !a->gate || a->y, "a gate needs a block output");
  Norm n{};
  n.columns = a->columns;
  n.rows = a->rows;
  n.layer = a->kind == EPS_B200_NORM_LAYER;
  n.gate = a->gate_kind;
  n.activation = a->activation;
  n.post_norm = a->post_norm != 0;
  n.pre_norm = a->pre_norm != 0;
  n.narrow = a->parameter_type == a->type;
  n.epsilon = a->epsilon;
  n.scale = a->scale;
  n.inverse_columns = 1.f / (float)a->columns;
  n.y = a->y;
  n.ys = a->y_stride;
  n.g = a->gate;
  n.gs = a->gate_stride;
  n.post_w = a->post_weight;
  n.post_b = a->post_bias;
  n.channel = a->channel_scale;
  n.pre_w = a->pre_weight;
  n.pre_b = a->pre_bias;
  if (!n.post_norm) n.post_w = n.post_b = nullptr;
  if (!n.y) {      // then the block adds nothing: zeros, times what is finite
    n.post_w = n.post_b = n.channel = nullptr;
    n.scale = 1.f;
  }
  return n;
}

bool parameters_wide(const Norm& n, int type) {
  for (const void* p : {n.post_w, n.post_b, n.channel, n.pre_w, n.pre_b})
    if (!aligned(p, 16)) return false;
  return n.columns % (type == EPS_B200_F32 ? 4 : 8) == 0;
}

}  // namespace
}  // namespace dense
}  // namespace eps_b200

using namespace eps_b200::dense;

extern "C" {

int eps_b200_block_norm(const EpsB200BlockNorm* a, const void* x, int64_t x_stride, void* h, int64_t h_stride,
                        void* z, int64_t z_stride, void* stream, EpsB200Status* status) {
  return guard(status, [&] {
    Norm n = checked(a);
    need(!n.rows || x, "null residual");
    need(!n.rows || h || !n.y, "null output of the residual");
    need(!n.rows || z || !n.pre_norm, "null output of the norm");
    if (!n.rows) return;
    n.x = n.somewhere = x; n.xs = x_stride;
    n.out_h = h; n.out_hs = h_stride;
    n.out_z = z; n.out_zs = z_stride;
    if (!n.out_h && !n.pre_norm) return;
    OnDevice on(a->device);
    bool wide = parameters_wide(n, a->type) && rows_wide(n.y, n.ys, a->type) && rows_wide(x, x_stride, a->residual_type) &&
                rows_wide(h, h_stride, a->residual_type) && rows_wide(z, z_stride, a->type);
    if (n.gate == EPS_B200_GATE_ELEMENT) wide = wide && rows_wide(n.g, n.gs, a->type);
    const Spread s = spread_of(n.columns, a->residual_type, a->type, wide);
    n.width = s.width;
    by_type(a->residual_type, a->type, [&](auto tx, auto ty) {
      by_spread<kWide<decltype(tx), decltype(ty)>>(s, [&](auto v, auto nit, auto warps) {
        by_gate(n.gate, [&](auto gate) {
          forward<decltype(tx), decltype(ty), decltype(v)::value, decltype(nit)::value, decltype(warps)::value,
                  decltype(gate)::value>(
              n, s, a->device, static_cast<cudaStream_t>(stream));
        });
      });
    });
  });
}

uint64_t eps_b200_block_norm_workspace(uint64_t rows, uint32_t columns) {
  uint64_t blocks = kMostBlocks;
  if (rows < blocks) blocks = rows;
  return blocks * kSums * columns * 4;
}

int eps_b200_block_norm_backward(const EpsB200BlockNorm* a, const EpsB200BlockNormGradients* d, void* stream,
                                 EpsB200Status* status) {
  return guard(status, [&] {
    Norm n = checked(a);
    need(d, "null gradients");
    need(!d->dz || n.pre_norm, "a gradient of the norm that is not there");
    const bool y = n.y || !n.rows;
    need(!n.rows || !d->dz || d->h, "the norm's gradient needs h");
    need((!d->dy && !d->dgate) || y, "gradients of a block output that is not there");
    need(!d->dgate || n.gate != EPS_B200_GATE_NONE, "gradient of a gate that is not there");
    need((!d->dpost_weight && !d->dpost_bias) || (y && n.post_norm), "gradients of a norm that is not there");
    need(!d->dchannel_scale || y, "gradient of a channel scale without a block output");
    need((!d->dpre_weight && !d->dpre_bias) || n.pre_norm, "gradients of a norm that is not there");
    n.dh = d->dh; n.dhs = d->dh_stride;
    n.dz = d->dz; n.dzs = d->dz_stride;
    if (!n.dz) n.pre_w = nullptr;        // zeros come in that way, whatever the weight is
    n.h = d->h; n.hs = d->h_stride;
    n.dx = d->dx; n.dxs = d->dx_stride;
    n.dy = d->dy; n.dys = d->dy_stride;
    n.dg = d->dgate; n.dgs = d->dgate_stride;
    float* const out[kSums] = {d->dpost_weight, d->dpost_bias, d->dchannel_scale, d->dpre_weight, d->dpre_bias};
    for (int k = 0; k < kSums; ++k)
      if (out[k]) n.want |= 1 << k;
    OnDevice on(a->device);
    const auto st = static_cast<cudaStream_t>(stream);
    if (!n.rows) {
      for (float* o : out)
        if (o) check(cudaMemsetAsync(o, 0, n.columns * 4, st), "cudaMemsetAsync");
      return;
    }
    need(!n.want || (d->workspace && aligned(d->workspace, 16)), "the workspace must be there and 16-byte aligned");
    n.somewhere = n.dz ? n.dz : n.dh ? n.dh : n.y ? n.y : d->dx ? d->dx : n.want ? d->workspace : nullptr;
    if (!n.somewhere) return;       // nothing comes in and nothing is asked for
    bool wide = parameters_wide(n, a->type) && rows_wide(n.y, n.ys, a->type) && rows_wide(n.dh, n.dhs, a->residual_type) &&
                rows_wide(n.dz, n.dzs, a->type) && rows_wide(n.h, n.hs, a->residual_type) &&
                rows_wide(n.dx, n.dxs, a->residual_type) && rows_wide(n.dy, n.dys, a->type);
    if (n.gate == EPS_B200_GATE_ELEMENT) wide = wide && rows_wide(n.g, n.gs, a->type) && rows_wide(n.dg, n.dgs, a->type);
    const Spread s = spread_of(n.columns, a->residual_type, a->type, wide);
    n.width = s.width;
    unsigned blocks = 0;
    n.partial = static_cast<float*>(d->workspace);
    by_type(a->residual_type, a->type, [&](auto tx, auto ty) {
      by_spread<kWide<decltype(tx), decltype(ty)>>(s, [&](auto v, auto nit, auto warps) {
        by_gate(n.gate, [&](auto gate) {
          blocks = backward<decltype(tx), decltype(ty), decltype(v)::value, decltype(nit)::value, decltype(warps)::value,
                  decltype(gate)::value>(
              n, s, a->device, d->workspace_bytes, st);
        });
      });
    });
    if (!n.want) return;
    Columns c{};
    c.partial = n.partial;
    for (int k = 0; k < kSums; ++k) c.out[k] = out[k];
    c.columns = n.columns;
    c.blocks = blocks;
    block_norm_columns<<<dim3((unsigned)ceil_div(n.columns, 32), kSums), 32 * kRuns, 0, st>>>(c);
    check(cudaGetLastError(), "block_norm_columns");
  });
}

}  // extern "C"
