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
};

// The column sums of the backward pass, in this order in `partial`.
enum { kPostWeight, kPostBias, kChannel, kPreWeight, kPreBias, kSums };

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

// act(g) and its derivative.
__device__ __forceinline__ float activate(float g, int activation, float* slope) {
  if (activation == EPS_B200_ACT_NONE) { *slope = 1.f; return g; }
  if (activation == EPS_B200_ACT_TANH) {
    const float t = tanhf(g);
    *slope = fmaf(-t, t, 1.f);
    return t;
  }
  const float s = sigmoid(g);
  if (activation == EPS_B200_ACT_SIGMOID) { *slope = s * (1.f - s); return s; }
  *slope = s * fmaf(g, 1.f - s, 1.f);
  return g * s;
}

// A parameter vector's V elements from column c on, `missing` where there is none.
template <class T, int V>
__device__ __forceinline__ void parameter(const void* p, int narrow, unsigned c, float missing, float (&r)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = missing;
  } else if (narrow) {
    const Pack<T, V> k = load_pack<T, V>(static_cast<const T*>(p) + c);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = to_float(k.v[i]);
  } else {
    const Pack<float, V> k = load_pack<float, V>(static_cast<const float*>(p) + c);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = k.v[i];
  }
}

// Mean and reciprocal deviation of a row held as v[NIT][V] by its lanes.  Two
// passes over the registers for a layer norm: the squares of what is left after
// the mean cannot cancel.  A lane divides its own sums by the columns, so that they
// cannot overflow across lanes where the mean square itself does not.
template <int V, int NIT>
__device__ __forceinline__ void statistics(const Norm& n, const float (&v)[NIT][V], unsigned lane, bool live,
                                           float* shared, unsigned& turn, float* mean, float* r) {
  *mean = 0.f;
  if (n.layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[i][j];     // lanes past the row hold 0
    s[0] *= n.inverse_columns;
    row_sum<1>(s, n.width, shared, turn);
    *mean = s[0];
  }
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NIT; ++i)
    if (live && (i * n.width + lane) * V < n.columns) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[i][j] - *mean;
        s[0] = fmaf(d, d, s[0]);
      }
    }
  s[0] *= n.inverse_columns;
  row_sum<1>(s, n.width, shared, turn);
  *r = __frsqrt_rn(s[0] + n.epsilon);
}

template <class TX, class TY, int V, int NIT>
__global__ void __launch_bounds__(V == 8 ? 512 : 1024) block_norm_forward(const Norm n) {
  __shared__ float shared[kRowSumShared];
  unsigned turn = 0;
  const unsigned lane = threadIdx.x % n.width;
  const uint64_t row = (uint64_t)blockIdx.x * (blockDim.x / n.width) + threadIdx.x / n.width;
  const bool live = row < n.rows;
  const TY* const y = static_cast<const TY*>(n.y);
  Pack<TY, V> gate[NIT];
  Pack<TX, V> x[NIT];
  float v[NIT][V];
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const unsigned c = (i * n.width + lane) * V;
    const bool in = live && c < n.columns;
    Pack<TY, V> k{};
    if (in && y) k = load_once<TY, V>(y + row * n.ys + c);
    if (in && y && n.gate == EPS_B200_GATE_ELEMENT) gate[i] = load_once<TY, V>(static_cast<const TY*>(n.g) + row * n.gs + c);
    if (in) x[i] = load_once<TX, V>(static_cast<const TX*>(n.x) + row * n.xs + c);
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = to_float(k.v[j]);
  }
  float mean = 0.f, r = 1.f, row_gate = 1.f, slope;
  if (y && n.post_norm) statistics<V, NIT>(n, v, lane, live, shared, turn, &mean, &r);
  if (y && live && n.gate == EPS_B200_GATE_ROW)
    row_gate = activate(to_float(static_cast<const TY*>(n.g)[row]), n.activation, &slope);
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const unsigned c = (i * n.width + lane) * V;
    if (!live || c >= n.columns) continue;
    if (!y) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = to_float(x[i].v[j]);
    } else {
      float w[V], b[V], s[V];
      if (n.post_norm) {
        parameter<TY, V>(n.post_w, n.narrow, c, 1.f, w);
        parameter<TY, V>(n.post_b, n.narrow, c, 0.f, b);
      }
      parameter<TY, V>(n.channel, n.narrow, c, 1.f, s);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float u = n.post_norm ? fmaf((v[i][j] - mean) * r, w[j], b[j]) : v[i][j];
        if (n.gate == EPS_B200_GATE_ROW) u *= row_gate;
        else if (n.gate == EPS_B200_GATE_ELEMENT) u *= activate(to_float(gate[i].v[j]), n.activation, &slope);
        v[i][j] = fmaf(n.scale * s[j], u, to_float(x[i].v[j]));
      }
    }
    if (n.out_h) {
      Pack<TX, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = from_float<TX>(v[i][j]);
      store_pack<TX, V>(static_cast<TX*>(n.out_h) + row * n.out_hs + c, o);
    }
  }
  if (!n.pre_norm) return;
  statistics<V, NIT>(n, v, lane, live, shared, turn, &mean, &r);
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const unsigned c = (i * n.width + lane) * V;
    if (!live || c >= n.columns) continue;
    float w[V], b[V];
    parameter<TY, V>(n.pre_w, n.narrow, c, 1.f, w);
    parameter<TY, V>(n.pre_b, n.narrow, c, 0.f, b);
    Pack<TY, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = from_float<TY>(fmaf((v[i][j] - mean) * r, w[j], b[j]));
    store_pack<TY, V>(static_cast<TY*>(n.out_z) + row * n.out_zs + c, o);
  }
}

// One block walks rows blockIdx, blockIdx + grid, ... and keeps the column sums of
// its lanes in shared memory (each lane its own columns: no conflict, no atomic);
// they leave it once, and block_norm_columns adds them up in block order.
template <class TX, class TY, int V, int NIT>
__global__ void __launch_bounds__(V == 8 ? 512 : 1024) block_norm_gradient(const Norm n) {
  extern __shared__ float sums[];          // [wanted][NIT][V][blockDim.x]
  __shared__ float shared[kRowSumShared];
  unsigned turn = 0;
  const unsigned lane = threadIdx.x % n.width, groups = blockDim.x / n.width;
  const TY* const y = static_cast<const TY*>(n.y);
  const unsigned cell = NIT * V * blockDim.x;
  int slot[kSums];
  int wanted = 0;
#pragma unroll
  for (int k = 0; k < kSums; ++k) slot[k] = n.want >> k & 1 ? wanted++ : -1;
  for (unsigned i = threadIdx.x; i < wanted * cell; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  auto add = [&](int k, int i, int j, float value) {
    if (slot[k] >= 0) sums[slot[k] * cell + (i * V + j) * blockDim.x + threadIdx.x] += value;
  };

  for (uint64_t base = (uint64_t)blockIdx.x * groups; base < n.rows; base += (uint64_t)gridDim.x * groups) {
    const uint64_t row = base + threadIdx.x / n.width;
    const bool live = row < n.rows;
    Pack<TY, V> gate[NIT];
    float d[NIT][V], q[NIT][V], h[NIT][V], v[NIT][V];     // dh, dz, h, y
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const unsigned c = (i * n.width + lane) * V;
      const bool in = live && c < n.columns;
      Pack<TX, V> kd{}, kh{};
      Pack<TY, V> kq{}, ky{};
      if (in && n.dh) kd = load_once<TX, V>(static_cast<const TX*>(n.dh) + row * n.dhs + c);
      if (in && n.dz) kq = load_once<TY, V>(static_cast<const TY*>(n.dz) + row * n.dzs + c);
      if (in && n.dz) kh = load_once<TX, V>(static_cast<const TX*>(n.h) + row * n.hs + c);
      if (in && y) ky = load_once<TY, V>(y + row * n.ys + c);
      gate[i] = Pack<TY, V>{};
      if (in && y && n.gate == EPS_B200_GATE_ELEMENT) gate[i] = load_once<TY, V>(static_cast<const TY*>(n.g) + row * n.gs + c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[i][j] = to_float(kd.v[j]);
        q[i][j] = to_float(kq.v[j]);
        h[i][j] = to_float(kh.v[j]);
        v[i][j] = to_float(ky.v[j]);
      }
    }
    // through the norm after
    if (n.dz) {
      float mean, r;
      statistics<V, NIT>(n, h, lane, live, shared, turn, &mean, &r);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const unsigned c = (i * n.width + lane) * V;
        if (!live || c >= n.columns) continue;
        float w[V];
        parameter<TY, V>(n.pre_w, n.narrow, c, 1.f, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[i][j] = (h[i][j] - mean) * r;
          add(kPreWeight, i, j, q[i][j] * h[i][j]);
          add(kPreBias, i, j, q[i][j]);
          q[i][j] *= w[j];
          s[0] += q[i][j];
          s[1] = fmaf(q[i][j], h[i][j], s[1]);
        }
      }
      row_sum<2>(s, n.width, shared, turn);
      const float mq = n.layer ? s[0] * n.inverse_columns : 0.f, mh = s[1] * n.inverse_columns;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = fmaf(r, q[i][j] - mq - h[i][j] * mh, d[i][j]);
    }
    if (n.dx) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const unsigned c = (i * n.width + lane) * V;
        if (!live || c >= n.columns) continue;
        Pack<TX, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = from_float<TX>(d[i][j]);
        store_pack<TX, V>(static_cast<TX*>(n.dx) + row * n.dxs + c, o);
      }
    }
    if (!y) continue;
    // through the scale, the gate and the norm before
    float mean = 0.f, r = 1.f, ra = 1.f, rslope = 0.f;
    if (n.post_norm) statistics<V, NIT>(n, v, lane, live, shared, turn, &mean, &r);
    if (live && n.gate == EPS_B200_GATE_ROW) ra = activate(to_float(static_cast<const TY*>(n.g)[row]), n.activation, &rslope);
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const unsigned c = (i * n.width + lane) * V;
      if (!live || c >= n.columns) continue;
      float w[V], b[V], ch[V];
      parameter<TY, V>(n.post_w, n.narrow, c, 1.f, w);
      parameter<TY, V>(n.post_b, n.narrow, c, 0.f, b);
      parameter<TY, V>(n.channel, n.narrow, c, 1.f, ch);
      Pack<TY, V> og;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float a = ra, slope = rslope;
        if (n.gate == EPS_B200_GATE_ELEMENT) a = activate(to_float(gate[i].v[j]), n.activation, &slope);
        if (n.post_norm) v[i][j] = (v[i][j] - mean) * r;
        const float nv = n.post_norm ? fmaf(v[i][j], w[j], b[j]) : v[i][j];
        const float e = n.scale * d[i][j];
        add(kChannel, i, j, e * a * nv);
        const float ec = e * ch[j];
        const float dgate = ec * nv * slope;
        og.v[j] = from_float<TY>(dgate);
        s[2] += dgate;
        const float dn = ec * a;
        if (n.post_norm) {
          add(kPostWeight, i, j, dn * v[i][j]);
          add(kPostBias, i, j, dn);
        }
        q[i][j] = n.post_norm ? dn * w[j] : dn;
        s[0] += q[i][j];
        s[1] = fmaf(q[i][j], v[i][j], s[1]);
      }
      if (n.dg && n.gate == EPS_B200_GATE_ELEMENT) store_pack<TY, V>(static_cast<TY*>(n.dg) + row * n.dgs + c, og);
    }
    if (n.post_norm || n.gate == EPS_B200_GATE_ROW) row_sum<3>(s, n.width, shared, turn);
    if (live && lane == 0 && n.dg && n.gate == EPS_B200_GATE_ROW) static_cast<TY*>(n.dg)[row] = from_float<TY>(s[2]);
    const float mp = n.layer ? s[0] * n.inverse_columns : 0.f, my = s[1] * n.inverse_columns;
    if (n.dy) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const unsigned c = (i * n.width + lane) * V;
        if (!live || c >= n.columns) continue;
        Pack<TY, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j)
          o.v[j] = from_float<TY>(n.post_norm ? r * (q[i][j] - mp - v[i][j] * my) : q[i][j]);
        store_pack<TY, V>(static_cast<TY*>(n.dy) + row * n.dys + c, o);
      }
    }
  }
  if (!wanted) return;
  __syncthreads();
  // the block's groups of lanes in order, then out
  for (unsigned c = threadIdx.x; c < n.columns; c += blockDim.x) {
    const unsigned at = c / V, i = at / n.width, l = at % n.width, j = c % V;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (slot[k] < 0) continue;
      float s = 0.f;
      for (unsigned g = 0; g < groups; ++g) s += sums[slot[k] * cell + (i * V + j) * blockDim.x + g * n.width + l];
      n.partial[((uint64_t)blockIdx.x * kSums + k) * n.columns + c] = s;
    }
  }
}

struct Columns {
  const float* partial;
  float* out[kSums];
  unsigned columns, blocks;
};

// out[k][c] = the sum over blocks of partial[block][k][c]: 32 columns a block of
// threads, eight runs of blocks, joined in order.
__global__ void __launch_bounds__(256) block_norm_columns(const Columns p) {
  __shared__ float part[8][32];
  const unsigned c = blockIdx.x * 32 + threadIdx.x % 32, run = threadIdx.x / 32, k = blockIdx.y;
  if (!p.out[k]) return;
  float s = 0.f;
  if (c < p.columns)
    for (unsigned b = run; b < p.blocks; b += 8) s += p.partial[((uint64_t)b * kSums + k) * p.columns + c];
  part[run][threadIdx.x % 32] = s;
  __syncthreads();
  if (run == 0 && c < p.columns) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
    p.out[k][c] = s;
  }
}

// How a row is spread: V elements a lane, `nit` times, over `width` lanes.
struct Spread { int v, nit; unsigned width, threads; };

Spread spread_of(unsigned columns, bool wide) {
  Spread s{};
  s.v = wide ? 8 : 1;
  const unsigned packs = (unsigned)ceil_div(columns, s.v);
  if (packs <= 32) {
    s.nit = 1;
    s.width = 1;
    while (s.width < packs) s.width *= 2;
    s.threads = 128;
  } else {
    s.nit = wide ? (packs <= 512 ? 1 : 2) : (packs <= 1024 ? 1 : 8);
    s.width = s.threads = (unsigned)round_up(ceil_div(packs, s.nit), 32);
  }
  return s;
}

unsigned gradient_blocks(uint64_t rows, const Spread& s, unsigned sms) {
  const uint64_t all = ceil_div(rows, s.threads / s.width);
  const uint64_t resident = (uint64_t)sms * (s.threads <= 128 ? 8 : s.threads <= 256 ? 4 : s.threads <= 512 ? 2 : 1);
  return (unsigned)(all < resident ? all : resident);
}
constexpr unsigned kMostBlocks = 8 * 160;   // of gradient_blocks, for up to 160 SMs

template <class TX, class TY, int V, int NIT>
void forward(const Norm& n, const Spread& s, cudaStream_t stream) {
  const uint64_t blocks = ceil_div(n.rows, s.threads / s.width);
  need(blocks < (1ull << 31), "too many rows");
  block_norm_forward<TX, TY, V, NIT><<<(unsigned)blocks, s.threads, 0, stream>>>(n);
  check(cudaGetLastError(), "block_norm");
}

template <class TX, class TY, int V, int NIT>
void backward(const Norm& n, const Spread& s, unsigned blocks, cudaStream_t stream) {
  const unsigned shared = __builtin_popcount((unsigned)n.want) * NIT * V * s.threads * 4;
  check(cudaFuncSetAttribute(block_norm_gradient<TX, TY, V, NIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024),
        "cudaFuncSetAttribute");
  block_norm_gradient<TX, TY, V, NIT><<<blocks, s.threads, shared, stream>>>(n);
  check(cudaGetLastError(), "block_norm_backward");
}

template <class TX, class TY, class F>
void by_spread(const Spread& s, F f) {
  if (s.v == 8) s.nit == 1 ? f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{})
                           : f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
  else s.nit == 1 ? f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{})
                  : f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
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
    n.x = x; n.xs = x_stride;
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
      by_spread<decltype(tx), decltype(ty)>(s, [&](auto v, auto nit) {
        forward<decltype(tx), decltype(ty), decltype(v)::value, decltype(nit)::value>(n, s, static_cast<cudaStream_t>(stream));
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
    const unsigned blocks = gradient_blocks(n.rows, s, sm_count(a->device));
    need(!n.want || (d->workspace && d->workspace_bytes >= (uint64_t)blocks * kSums * n.columns * 4),
         "block norm workspace too small");
    need(!n.want || aligned(d->workspace, 16), "the workspace must be 16-byte aligned");
    n.partial = static_cast<float*>(d->workspace);
    by_type(a->residual_type, a->type, [&](auto tx, auto ty) {
      by_spread<decltype(tx), decltype(ty)>(s, [&](auto v, auto nit) {
        backward<decltype(tx), decltype(ty), decltype(v)::value, decltype(nit)::value>(n, s, blocks, st);
      });
    });
    if (!n.want) return;
    Columns c{};
    c.partial = n.partial;
    for (int k = 0; k < kSums; ++k) c.out[k] = out[k];
    c.columns = n.columns;
    c.blocks = blocks;
    block_norm_columns<<<dim3((unsigned)ceil_div(n.columns, 32), kSums), 256, 0, st>>>(c);
    check(cudaGetLastError(), "block_norm_columns");
  });
}

}  // extern "C"
