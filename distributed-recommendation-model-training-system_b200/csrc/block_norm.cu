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
// h, y, gate and writes dx, dy, dgate: each value once, held in registers between
// the passes over the row.  A row belongs to a group of lanes (a power of two up
// to a warp, or a whole block), V consecutive elements a lane NIT times: V = 8
// where all rows are 16-byte aligned, 1 otherwise.
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

// 1 / (1 + 2^(-g log2 e)): two instructions of the special-function unit, each good
// to two units of the last place; subnormal powers count as 0, which 1 + hides.
template <int V>
__device__ __forceinline__ void sigmoid(const float (&g)[V], float (&s)[V]) {
  vmul<V>(s, g, -1.4426950408889634f);
#pragma unroll
  for (int j = 0; j < V; ++j) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(s[j]));
  vadd<V>(s, s, 1.f);
#pragma unroll
  for (int j = 0; j < V; ++j) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(s[j]));
}

// act(g) and, where SLOPE, its derivative for V values; the choice is made once for
// all of them.
template <int V, bool SLOPE>
__device__ __forceinline__ void activate(const float (&g)[V], int activation, float (&a)[V], float (&slope)[V]) {
  if (activation == EPS_B200_ACT_SIGMOID) {
    sigmoid<V>(g, a);
    if (SLOPE) {
#pragma unroll
      for (int j = 0; j < V; ++j) slope[j] = fmaf(-a[j], a[j], a[j]);
    }
  } else if (activation == EPS_B200_ACT_SILU) {
    float s[V];
    sigmoid<V>(g, s);
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

__device__ __forceinline__ float activate_one(float g, int activation, float* slope) {
  float v[1] = {g}, a[1], s[1];
  activate<1, true>(v, activation, a, s);
  *slope = s[0];
  return a[0];
}

// A parameter vector's V elements from column c on, `missing` where there is none.
template <class T, int V>
__device__ __forceinline__ void parameter(const void* p, int narrow, unsigned c, float missing, float (&r)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = missing;
  } else if (narrow) {
    widen(load_pack<T, V>(static_cast<const T*>(p) + c), r);
  } else {
    widen(load_pack<float, V>(static_cast<const float*>(p) + c), r);
  }
}

// The parameter vectors as a lane uses them.  Where a lane has few columns, a block
// lays its lanes' values out in shared memory once, in float and with what is missing
// filled in: rows then read them without a branch and without a bank conflict.
enum { kPostW, kPostB, kScaleC, kPreW, kPreB, kVectors };

template <class T, int V, int NIT, bool STAGED>
struct Parameters {
  const Norm& n;
  float* staged;           // [kVectors][NIT][V / 4][blockDim.x][4], or [kVectors][NIT][blockDim.x] for V == 1
  unsigned lane;

  __device__ __forceinline__ float* at(int k, int i) const { return staged + (unsigned)((k * NIT + i) * V) * blockDim.x + threadIdx.x * (V < 4 ? V : 4); }
  __device__ __forceinline__ void read(int k, int i, float (&r)[V]) const {
    const unsigned c = (i * n.width + lane) * V;
    switch (k) {
      case kPostW: parameter<T, V>(n.post_w, n.narrow, c, 1.f, r); break;
      case kPostB: parameter<T, V>(n.post_b, n.narrow, c, 0.f, r); break;
      case kScaleC: parameter<T, V>(n.channel, n.narrow, c, 1.f, r); vmul<V>(r, r, n.scale); break;
      case kPreW: parameter<T, V>(n.pre_w, n.narrow, c, 1.f, r); break;
      default: parameter<T, V>(n.pre_b, n.narrow, c, 0.f, r);
    }
  }
  __device__ __forceinline__ void stage() const {
    if constexpr (STAGED) {
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          float r[V] = {};          // 0 behind the last column: what a lane holds there adds nothing
          if ((i * n.width + lane) * V < n.columns) read(k, i, r);
#pragma unroll
          for (int j = 0; j < V; j += 4) {
            if constexpr (V >= 4) *reinterpret_cast<float4*>(at(k, i) + j * blockDim.x) = make_float4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            else *at(k, i) = r[0];
          }
        }
      // each thread reads back its own values only: no barrier
    }
  }
  __device__ __forceinline__ void get(int k, int i, float (&r)[V]) const {
    if constexpr (STAGED) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        if constexpr (V >= 4) {
          const float4 x = *reinterpret_cast<const float4*>(at(k, i) + j * blockDim.x);
          r[j] = x.x; r[j + 1] = x.y; r[j + 2] = x.z; r[j + 3] = x.w;
        } else {
          r[0] = *at(k, i);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) r[j] = 0.f;
      if ((i * n.width + lane) * V < n.columns) read(k, i, r);
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

// Means and reciprocal deviations of K rows held by the same lanes.  Two passes over
// the registers for a layer norm: the squares of what is left after the mean cannot
// cancel.  A lane divides its own sums by the columns, so that they cannot overflow
// across lanes where the mean square itself does not.
template <int V, int NIT, int K>
__device__ __forceinline__ void statistics(const Norm& n, const float (*const (&v)[K])[V], unsigned lane, float* shared,
                                           unsigned& turn, float (&mean)[K], float (&r)[K]) {
  float s[K];
#pragma unroll
  for (int k = 0; k < K; ++k) mean[k] = 0.f;
  if (n.layer) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < NIT; ++i) s[k] += total<V>(v[k][i]);     // lanes past the row hold 0
      s[k] *= n.inverse_columns;
    }
    row_sum<K>(s, n.width, shared, turn);
#pragma unroll
    for (int k = 0; k < K; ++k) mean[k] = s[k];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    s[k] = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float d[V];
      vadd<V>(d, v[k][i], -mean[k]);
      vmul<V>(d, d, d);
      s[k] = fmaf(total<V>(d), (i * n.width + lane) * V < n.columns ? n.inverse_columns : 0.f, s[k]);
    }
  }
  row_sum<K>(s, n.width, shared, turn);
#pragma unroll
  for (int k = 0; k < K; ++k) r[k] = __frsqrt_rn(s[k] + n.epsilon);
}

template <int V, int NIT>
__device__ __forceinline__ void one_row(const Norm& n, const float (&v)[NIT][V], unsigned lane, float* shared, unsigned& turn,
                                        float* mean, float* r) {
  const float(*const rows[1])[V] = {v};
  float m[1], d[1];
  statistics<V, NIT, 1>(n, rows, lane, shared, turn, m, d);
  *mean = m[0];
  *r = d[0];
}

// (v - mean) * r: the difference first, since v r and mean r may both be large.
template <int V>
__device__ __forceinline__ void centre(float (&v)[V], float mean, float r) {
  vadd<V>(v, v, -mean);
  vmul<V>(v, v, r);
}

// The rows of R tensors on their way into shared memory.  Blocks walk the rows, and
// a lane asks for its own values two rows ahead, past registers and L1: the
// reductions and barriers of a row then pass while its successors are under way.  A
// lane reads back only what it asked for itself, so no barrier is involved; lanes
// behind the row's end, rows behind the last one and missing tensors read zeros.
// Without 16-byte alignment, or with more than eight elements a lane, values are
// loaded as they are needed.
constexpr unsigned kAhead = 2, kSlots = kAhead + 1;

__device__ __forceinline__ void copy16(unsigned to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

template <class T, int V, int NIT, bool RING>
struct Source {
  const T* p;              // the tensor at the lane's first column, or NULL
  int64_t stride;
  unsigned to;             // RING: the lane's place in slot 0, a shared address; 16-byte planes blockDim.x apart
  static constexpr unsigned kPlanes = V * sizeof(T) / 16;

  __device__ __forceinline__ void ask(const Norm& n, unsigned slot, unsigned slot_bytes, uint64_t row, bool in) const {
    static_assert(!RING || NIT == 1, "one pack a lane");
    const bool there = in && p;
    const char* const from = reinterpret_cast<const char*>(there ? p + row * stride : static_cast<const T*>(n.somewhere));
#pragma unroll
    for (unsigned k = 0; k < kPlanes; ++k) copy16(to + slot * slot_bytes + k * blockDim.x * 16, from + (there ? k * 16 : 0), there);
  }
  __device__ __forceinline__ void get(const Norm& n, unsigned slot, unsigned slot_bytes, uint64_t row, bool live, unsigned lane,
                                      float (&r)[NIT][V]) const {
    if constexpr (RING) {
      Pack<T, V> x;
#pragma unroll
      for (unsigned k = 0; k < kPlanes; ++k) {
        uint4& q = reinterpret_cast<uint4*>(&x)[k];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(to + slot * slot_bytes + k * blockDim.x * 16) : "memory");
      }
      widen(x, r[0]);
    } else {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        Pack<T, V> x{};
        if (live && p && (i * n.width + lane) * V < n.columns) x = load_once<T, V>(p + row * stride + i * n.width * V);
        widen(x, r[i]);
      }
    }
  }
};

template <class T, int V, int NIT>
__device__ __forceinline__ void put(const Norm& n, void* p, int64_t stride, uint64_t row, int i, unsigned lane, bool live, const float (&v)[V]) {
  const unsigned c = (i * n.width + lane) * V;
  if (live && c < n.columns) store_pack<T, V>(static_cast<T*>(p) + row * stride + c, narrow<T, V>(v));
}

template <class TX, class TY, int V, int NIT>
struct ForwardSources {
  static constexpr bool kRing = V == 8 && NIT == 1;
  Source<TX, V, NIT, kRing> x;
  Source<TY, V, NIT, kRing> y, gate;
  static constexpr unsigned kSlot = V * (sizeof(TX) + 2 * sizeof(TY));     // bytes of a lane
};
template <class TX, class TY, int V, int NIT>
struct BackwardSources {
  static constexpr bool kRing = V == 8 && NIT == 1;
  Source<TX, V, NIT, kRing> dh, h;
  Source<TY, V, NIT, kRing> dz, y, gate;
  static constexpr unsigned kSlot = V * (2 * sizeof(TX) + 3 * sizeof(TY));
};

template <class T>
__device__ __forceinline__ const T* column(const void* p, unsigned c) {
  return p ? static_cast<const T*>(p) + c : nullptr;
}

template <class TX, class TY, int V, int NIT, int GATE>
__global__ void __launch_bounds__(V == 8 ? 512 : 1024) block_norm_forward(const Norm n) {
  using Sources = ForwardSources<TX, TY, V, NIT>;
  constexpr bool kRing = Sources::kRing, kStaged = V * NIT <= 8;
  extern __shared__ __align__(16) float room[];      // the staged parameters, then the ring
  __shared__ float shared[kRowSumShared];
  unsigned turn = 0;
  const unsigned lane = threadIdx.x % n.width, groups = blockDim.x / n.width;
  const uint64_t stride = (uint64_t)gridDim.x * groups;
  uint64_t row = (uint64_t)blockIdx.x * groups + threadIdx.x / n.width;
  const uint64_t passes = (n.rows - (uint64_t)blockIdx.x * groups + stride - 1) / stride;   // blocks do not outnumber groups of rows
  const bool in = lane * V < n.columns;
  const unsigned ring = shared_at(room + (kStaged ? kVectors * NIT * V * blockDim.x : 0)) + threadIdx.x * 16;
  const unsigned slot_bytes = Sources::kSlot * blockDim.x;
  const Sources s{{column<TX>(n.x, lane * V), n.xs, ring},
                  {column<TY>(n.y, lane * V), n.ys, ring + V * (unsigned)sizeof(TX) * blockDim.x},
                  {column<TY>(GATE == EPS_B200_GATE_ELEMENT ? n.g : nullptr, lane * V), n.gs,
                   ring + V * (unsigned)(sizeof(TX) + sizeof(TY)) * blockDim.x}};
  auto ask = [&](unsigned slot, uint64_t r) {
    if constexpr (kRing) {
      const bool there = in && r < n.rows;
      s.x.ask(n, slot, slot_bytes, r, there);
      s.y.ask(n, slot, slot_bytes, r, there);
      if (GATE == EPS_B200_GATE_ELEMENT) s.gate.ask(n, slot, slot_bytes, r, there);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
#pragma unroll
  for (unsigned k = 0; k < kAhead; ++k) ask(k, row + k * stride);
  const Parameters<TY, V, NIT, kStaged> p{n, room, lane};
  p.stage();
  unsigned slot = 0;
  for (uint64_t pass = 0; pass < passes; ++pass, row += stride) {
    const bool live = row < n.rows;
    float v[NIT][V], x[NIT][V], g[NIT][V];
    if constexpr (kRing) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
      ask(slot == 0 ? kSlots - 1 : slot - 1, row + kAhead * stride);
    }
    s.y.get(n, slot, slot_bytes, row, live, lane, v);
    float mean = 0.f, r = 1.f, row_gate = 1.f, unused;
    if (n.y && n.post_norm) one_row<V, NIT>(n, v, lane, shared, turn, &mean, &r);
    s.x.get(n, slot, slot_bytes, row, live, lane, x);
    if (GATE == EPS_B200_GATE_ELEMENT) s.gate.get(n, slot, slot_bytes, row, live, lane, g);
    slot = slot == kSlots - 1 ? 0 : slot + 1;
    if (GATE == EPS_B200_GATE_ROW && live) row_gate = activate_one(to_float(static_cast<const TY*>(n.g)[row]), n.activation, &unused);
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      if (!n.y) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = x[i][j];
      } else {
        float w[V], b[V];
        if (n.post_norm) {
          p.get(kPostW, i, w);
          p.get(kPostB, i, b);
          centre<V>(v[i], mean, r);
          vfma<V>(v[i], v[i], w, b);
        }
        if (GATE == EPS_B200_GATE_ELEMENT) {
          float a[V], slope[V];
          activate<V, false>(g[i], n.activation, a, slope);
          vmul<V>(v[i], v[i], a);
        }
        p.get(kScaleC, i, w);
        if (GATE == EPS_B200_GATE_ROW) vmul<V>(w, w, row_gate);
        vfma<V>(v[i], w, v[i], x[i]);
      }
      if (n.out_h) put<TX, V, NIT>(n, n.out_h, n.out_hs, row, i, lane, live, v[i]);
    }
    if (!n.pre_norm) continue;
    one_row<V, NIT>(n, v, lane, shared, turn, &mean, &r);
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float w[V], b[V];
      p.get(kPreW, i, w);
      p.get(kPreB, i, b);
      centre<V>(v[i], mean, r);
      vfma<V>(v[i], v[i], w, b);
      put<TY, V, NIT>(n, n.out_z, n.out_zs, row, i, lane, live, v[i]);
    }
  }
}

// The column sums of a lane stay in registers where a lane has few columns, else in
// shared memory (each lane its own columns: no conflict, no atomic).  They leave a
// block once; block_norm_columns adds the blocks up in order.
template <class TX, class TY, int V, int NIT, int GATE>
__global__ void __launch_bounds__(V == 8 ? 512 : 1024) block_norm_gradient(const Norm n) {
  using Sources = BackwardSources<TX, TY, V, NIT>;
  constexpr int N = V * NIT;
  constexpr bool kRing = Sources::kRing, kHeld = kRing;
  extern __shared__ __align__(16) float room[];     // [wanted][N][blockDim.x] sums; before them staged parameters and the ring
  __shared__ float shared[kRowSumShared];
  unsigned turn = 0;
  const unsigned lane = threadIdx.x % n.width, groups = blockDim.x / n.width;
  const unsigned cell = N * blockDim.x;
  int slot_of[kSums];
  int wanted = 0;
#pragma unroll
  for (int k = 0; k < kSums; ++k) slot_of[k] = n.want >> k & 1 ? wanted++ : -1;
  float held[kHeld ? kSums : 1][V];
  if constexpr (kHeld) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) held[k][j] = 0.f;
  } else {
    for (unsigned i = threadIdx.x; i < wanted * cell; i += blockDim.x) room[i] = 0.f;
    __syncthreads();
  }
  // column sums k of the lane's pack i grow by a * b, or by a
  auto add = [&](int k, int i, const auto& a, const auto& b) {
    if constexpr (kHeld) {
      if constexpr (std::is_same_v<std::decay_t<decltype(b)>, float>) vadd<V>(held[k], held[k], a);
      else vfma<V>(held[k], a, b, held[k]);
    } else if (slot_of[k] >= 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float* const s = room + slot_of[k] * cell + (i * V + j) * blockDim.x + threadIdx.x;
        *s = fmaf(part<V>(a, j), part<V>(b, j), *s);
      }
    }
  };

  const uint64_t stride = (uint64_t)gridDim.x * groups;
  uint64_t row = (uint64_t)blockIdx.x * groups + threadIdx.x / n.width;
  const uint64_t passes = (n.rows - (uint64_t)blockIdx.x * groups + stride - 1) / stride;
  const bool in = lane * V < n.columns;
  const unsigned ring = shared_at(room + (kRing ? kVectors * N * blockDim.x : 0)) + threadIdx.x * 16;
  const unsigned slot_bytes = Sources::kSlot * blockDim.x, bx = V * (unsigned)sizeof(TX) * blockDim.x, by = V * (unsigned)sizeof(TY) * blockDim.x;
  const Sources s{{column<TX>(n.dh, lane * V), n.dhs, ring},
                  {column<TX>(n.dz ? n.h : nullptr, lane * V), n.hs, ring + bx},
                  {column<TY>(n.dz, lane * V), n.dzs, ring + 2 * bx},
                  {column<TY>(n.y, lane * V), n.ys, ring + 2 * bx + by},
                  {column<TY>(GATE == EPS_B200_GATE_ELEMENT ? n.g : nullptr, lane * V), n.gs, ring + 2 * bx + 2 * by}};
  auto ask = [&](unsigned slot, uint64_t r) {
    if constexpr (kRing) {
      const bool there = in && r < n.rows;
      s.dh.ask(n, slot, slot_bytes, r, there);
      s.h.ask(n, slot, slot_bytes, r, there);
      s.dz.ask(n, slot, slot_bytes, r, there);
      s.y.ask(n, slot, slot_bytes, r, there);
      if (GATE == EPS_B200_GATE_ELEMENT) s.gate.ask(n, slot, slot_bytes, r, there);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
#pragma unroll
  for (unsigned k = 0; k < kAhead; ++k) ask(k, row + k * stride);
  const Parameters<TY, V, NIT, kRing> p{n, room, lane};
  p.stage();
  unsigned slot = 0;
  for (uint64_t pass = 0; pass < passes; ++pass, row += stride) {
    const bool live = row < n.rows;
    float d[NIT][V], q[NIT][V], h[NIT][V], y[NIT][V];
    if constexpr (kRing) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
      ask(slot == 0 ? kSlots - 1 : slot - 1, row + kAhead * stride);
    }
    s.h.get(n, slot, slot_bytes, row, live, lane, h);
    s.y.get(n, slot, slot_bytes, row, live, lane, y);
    float means[2], rs[2];
    const float(*const both[2])[V] = {h, y};
    statistics<V, NIT, 2>(n, both, lane, shared, turn, means, rs);
    s.dh.get(n, slot, slot_bytes, row, live, lane, d);
    // through the norm after
    if (n.dz) {
      const float r = rs[0];
      float sum[2] = {0.f, 0.f};
      s.dz.get(n, slot, slot_bytes, row, live, lane, q);
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        float w[V];
        p.get(kPreW, i, w);
        centre<V>(h[i], means[0], r);
        add(kPreWeight, i, q[i], h[i]);
        add(kPreBias, i, q[i], 1.f);
        vmul<V>(q[i], q[i], w);
        sum[0] += total<V>(q[i]);
        vmul<V>(w, q[i], h[i]);
        sum[1] += total<V>(w);
      }
      row_sum<2>(sum, n.width, shared, turn);
      const float mq = n.layer ? sum[0] * n.inverse_columns : 0.f, mh = sum[1] * n.inverse_columns;
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        vfma<V>(h[i], h[i], -mh, q[i]);
        vadd<V>(h[i], h[i], -mq);
        vfma<V>(d[i], h[i], r, d[i]);
      }
    }
    if (n.dx) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) put<TX, V, NIT>(n, n.dx, n.dxs, row, i, lane, live, d[i]);
    }
    const unsigned here = slot;
    slot = slot == kSlots - 1 ? 0 : slot + 1;
    if (!n.y) continue;
    // through the scale, the gate and the norm before
    const float r = rs[1];
    float ra = 1.f, rslope = 0.f;
    if (GATE == EPS_B200_GATE_ROW && live) ra = activate_one(to_float(static_cast<const TY*>(n.g)[row]), n.activation, &rslope);
    float g[NIT][V];
    if (GATE == EPS_B200_GATE_ELEMENT) s.gate.get(n, here, slot_bytes, row, live, lane, g);
    float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      float w[V], nv[V], a[V], slope[V], t[V];
      // y becomes its normed value, nv what the gate sees
      if (n.post_norm) {
        p.get(kPostW, i, w);
        p.get(kPostB, i, t);
        centre<V>(y[i], means[1], r);
        vfma<V>(nv, y[i], w, t);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) { nv[j] = y[i][j]; w[j] = 1.f; }
      }
      if (GATE == EPS_B200_GATE_ELEMENT) {
        activate<V, true>(g[i], n.activation, a, slope);
        vmul<V>(a, a, d[i]);
      } else {
        vmul<V>(a, d[i], ra);
      }
      add(kChannel, i, a, nv);          // without n.scale, which the block's sums take at the end
      p.get(kScaleC, i, t);
      if (GATE != EPS_B200_GATE_NONE) {
        vmul<V>(nv, nv, d[i]);
        vmul<V>(nv, nv, t);
        if (GATE == EPS_B200_GATE_ELEMENT) {
          vmul<V>(nv, nv, slope);
          if (n.dg) put<TY, V, NIT>(n, n.dg, n.dgs, row, i, lane, live, nv);
        } else {
          sum[2] += total<V>(nv);
        }
      }
      vmul<V>(q[i], a, t);
      if (n.post_norm) {
        add(kPostWeight, i, q[i], y[i]);
        add(kPostBias, i, q[i], 1.f);
        vmul<V>(q[i], q[i], w);
        sum[0] += total<V>(q[i]);
        vmul<V>(t, q[i], y[i]);
        sum[1] += total<V>(t);
      }
    }
    if (GATE == EPS_B200_GATE_ROW) {
      row_sum<3>(sum, n.width, shared, turn);
      if (live && lane == 0 && n.dg) static_cast<TY*>(n.dg)[row] = from_float<TY>(sum[2] * rslope);
    } else if (n.post_norm) {
      row_sum<2>(reinterpret_cast<float(&)[2]>(sum), n.width, shared, turn);
    }
    const float mp = n.layer ? sum[0] * n.inverse_columns : 0.f, my = sum[1] * n.inverse_columns;
    if (n.dy) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        if (n.post_norm) {
          vfma<V>(q[i], y[i], -my, q[i]);
          vadd<V>(q[i], q[i], -mp);
          vmul<V>(q[i], q[i], r);
        }
        put<TY, V, NIT>(n, n.dy, n.dys, row, i, lane, live, q[i]);
      }
    }
  }
  if constexpr (kRing) asm volatile("cp.async.wait_all;" ::: "memory");
  if (!wanted) return;
  if constexpr (kHeld) {
    __syncthreads();        // the staged parameters and the ring lie there
#pragma unroll
    for (int k = 0; k < kSums; ++k)
      if (slot_of[k] >= 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) room[slot_of[k] * cell + j * blockDim.x + threadIdx.x] = held[k][j];
      }
  }
  __syncthreads();
  // the block's groups of lanes in order, then out
  for (unsigned c = threadIdx.x; c < n.columns; c += blockDim.x) {
    const unsigned at = c / V, i = at / n.width, l = at % n.width, j = c % V;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (slot_of[k] < 0) continue;
      float t = 0.f;
      for (unsigned g = 0; g < groups; ++g) t += room[slot_of[k] * cell + (i * V + j) * blockDim.x + g * n.width + l];
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

Spread spread_of(unsigned columns, bool wide) {
  Spread s{};
  s.v = wide ? 8 : 1;
  const unsigned packs = (unsigned)ceil_div(columns, s.v);
  s.nit = wide ? (packs <= 512 ? 1 : 2) : (packs <= 32 ? 1 : packs <= 1024 ? 4 : 8);
  const unsigned lanes = (unsigned)ceil_div(packs, s.nit);
  if (lanes <= 32) {
    s.width = 1;
    while (s.width < lanes) s.width *= 2;
    s.threads = 128;
  } else {
    s.width = s.threads = (unsigned)round_up(lanes, 32);
  }
  return s;
}

constexpr unsigned kMostBlocks = 8 * 160;   // of the gradient: 8 an SM, 160 SMs

// Blocks that fit the GPU at once, or fewer where the rows need fewer.
template <class K>
unsigned resident(K kernel, const Spread& s, size_t shared, uint64_t rows, unsigned sms, unsigned most) {
  int each = 0;
  check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, (int)s.threads, shared), "occupancy");
  need(each > 0, "no room for a block");
  uint64_t n = (uint64_t)sms * (unsigned)each;
  if (n > most) n = most;
  const uint64_t all = ceil_div(rows, s.threads / s.width);
  return (unsigned)(all < n ? all : n);
}

template <class TX, class TY, int V, int NIT, int GATE>
void forward(const Norm& n, const Spread& s, unsigned sms, cudaStream_t stream) {
  auto* kernel = block_norm_forward<TX, TY, V, NIT, GATE>;
  using Sources = ForwardSources<TX, TY, V, NIT>;
  const unsigned shared = ((V * NIT <= 8 ? kVectors * NIT * V * 4 : 0) + (Sources::kRing ? kSlots * Sources::kSlot : 0)) * s.threads;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024), "cudaFuncSetAttribute");
  kernel<<<resident(kernel, s, shared, n.rows, sms, ~0u), s.threads, shared, stream>>>(n);
  check(cudaGetLastError(), "block_norm");
}

// The number of blocks, which is the number of partial sums.
template <class TX, class TY, int V, int NIT, int GATE>
unsigned backward(const Norm& n, const Spread& s, unsigned sms, uint64_t room, cudaStream_t stream) {
  auto* kernel = block_norm_gradient<TX, TY, V, NIT, GATE>;
  using Sources = BackwardSources<TX, TY, V, NIT>;
  const unsigned vectors = Sources::kRing ? kVectors : (unsigned)__builtin_popcount((unsigned)n.want);
  const unsigned shared = (vectors * NIT * V * 4 + (Sources::kRing ? kSlots * Sources::kSlot : 0)) * s.threads;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024), "cudaFuncSetAttribute");
  const unsigned blocks = resident(kernel, s, shared, n.rows, sms, kMostBlocks);
  need(!n.want || room >= (uint64_t)blocks * kSums * n.columns * 4, "block norm workspace too small");
  kernel<<<blocks, s.threads, shared, stream>>>(n);
  check(cudaGetLastError(), "block_norm_backward");
  return blocks;
}

template <int N> using Int = std::integral_constant<int, N>;

template <class F>
void by_gate(int gate, F f) {
  gate == EPS_B200_GATE_NONE ? f(Int<EPS_B200_GATE_NONE>{}) : gate == EPS_B200_GATE_ROW ? f(Int<EPS_B200_GATE_ROW>{})
                                                                                        : f(Int<EPS_B200_GATE_ELEMENT>{});
}

template <class F>
void by_spread(const Spread& s, F f) {
  if (s.v == 8) s.nit == 1 ? f(Int<8>{}, Int<1>{}) : f(Int<8>{}, Int<2>{});
  else s.nit == 1 ? f(Int<1>{}, Int<1>{}) : s.nit == 4 ? f(Int<1>{}, Int<4>{}) : f(Int<1>{}, Int<8>{});
}

template <class F>
void by_type(int residual, int type, F f) {
  if (type == EPS_B200_F32) f(float{}, float{});
  else if (type == EPS_B200_BF16) residual == EPS_B200_F32 ? f(float{}, bf16{}) : f(bf16{}, bf16{});
  else residual == EPS_B200_F32 ? f(float{}, f16{}) : f(f16{}, f16{});
}

// Whether rows at `p` with this stride (elements) and type take 16-byte accesses
// of eight (or four) elements.
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
  need(a->rows < (1ull << 40), "too many rows");
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
  return n;
}

bool parameters_wide(const Norm& n) {
  for (const void* p : {n.post_w, n.post_b, n.channel, n.pre_w, n.pre_b})
    if (!aligned(p, 16)) return false;
  return n.columns % 8 == 0;
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
    bool wide = parameters_wide(n) && rows_wide(n.y, n.ys, a->type) && rows_wide(x, x_stride, a->residual_type) &&
                rows_wide(h, h_stride, a->residual_type) && rows_wide(z, z_stride, a->type);
    if (n.gate == EPS_B200_GATE_ELEMENT) wide = wide && rows_wide(n.g, n.gs, a->type);
    const Spread s = spread_of(n.columns, wide);
    n.width = s.width;
    by_type(a->residual_type, a->type, [&](auto tx, auto ty) {
      by_spread(s, [&](auto v, auto nit) {
        by_gate(n.gate, [&](auto gate) {
          forward<decltype(tx), decltype(ty), decltype(v)::value, decltype(nit)::value, decltype(gate)::value>(
              n, s, sm_count(a->device), static_cast<cudaStream_t>(stream));
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
    n.h = d->h; n.hs = d->h_stride;
    n.somewhere = n.dz ? n.dz : n.dh ? n.dh : n.y ? n.y : d->dx;
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
    bool wide = parameters_wide(n) && rows_wide(n.y, n.ys, a->type) && rows_wide(n.dh, n.dhs, a->residual_type) &&
                rows_wide(n.dz, n.dzs, a->type) && rows_wide(n.h, n.hs, a->residual_type) &&
                rows_wide(n.dx, n.dxs, a->residual_type) && rows_wide(n.dy, n.dys, a->type);
    if (n.gate == EPS_B200_GATE_ELEMENT) wide = wide && rows_wide(n.g, n.gs, a->type) && rows_wide(n.dg, n.dgs, a->type);
    const Spread s = spread_of(n.columns, wide);
    n.width = s.width;
    need(!n.want || (d->workspace && aligned(d->workspace, 16)), "the workspace must be there and 16-byte aligned");
    unsigned blocks = 0;
    n.partial = static_cast<float*>(d->workspace);
    by_type(a->residual_type, a->type, [&](auto tx, auto ty) {
      by_spread(s, [&](auto v, auto nit) {
        by_gate(n.gate, [&](auto gate) {
          blocks = backward<decltype(tx), decltype(ty), decltype(v)::value, decltype(nit)::value, decltype(gate)::value>(
              n, s, sm_count(a->device), d->workspace_bytes, st);
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
