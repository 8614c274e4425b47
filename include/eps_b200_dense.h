/*
 * eps_b200_dense.h -- C ABI of the dense operators in libeps_b200.so.
 *
 * The embedding store (eps_b200.h) pulls rows and applies their gradients; these
 * entry points are the dense block that stands beside it: the norms before and
 * after a block with its gate and residual scale, routing to experts and the loss that
 * balances them, the experts' products in 8-bit integers, low-rank adapters beside a
 * shared layer, AdamW over many tensors and the norm that clips it.  None has a
 * counterpart in the reference, whose dense part is left to TensorFlow.
 *
 * Conventions:
 *  - every entry point returns 0, or a code of eps_b200.h with the message in
 *    status->message; a refused call launches nothing and writes nothing;
 *  - all pointers but the argument struct, the status and the arrays marked
 *    "host" are device pointers on `device`; nothing is allocated here: results
 *    and workspaces are the caller's, and may be reused once the stream has
 *    passed the call;
 *  - `stream` is a cudaStream_t (NULL = the legacy default stream).  Calls are
 *    asynchronous, keep nothing between calls, and can be captured in a graph (an
 *    AdamW step as eps_b200_adamw_counted);
 *  - an element type is EPS_B200_F32, _BF16 or _F16.  Sums, statistics and
 *    scores are held in 32 bits or more whatever the type;
 *  - no kernel waits longer than two seconds for a copy or a sum; where one gives up,
 *    what it still had to write becomes NaN;
 *  - the last axis of every tensor is contiguous; a row stride is given in
 *    elements.  Any alignment of the element type is accepted (16-byte aligned
 *    rows take wider loads).
 */
#ifndef EPS_B200_DENSE_H
#define EPS_B200_DENSE_H
#include "eps_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { EPS_B200_F32 = 0, EPS_B200_BF16 = 1, EPS_B200_F16 = 2 };

/* ---- Norms before and after a block, its gate and its residual scale.
 *   a = activation(gate)                        1 without a gate
 *   n = post norm of y                          y itself if post_norm == 0
 *   h = x + scale * channel_scale[d] * a * n    x if y is NULL
 *   z = pre norm of h                           not computed if pre_norm == 0
 * A norm is (v - mu) * r * weight[d] + bias[d] over a row of `columns` values:
 * EPS_B200_NORM_RMS has mu = 0, r = 1 / sqrt(mean(v^2) + epsilon), and
 * EPS_B200_NORM_LAYER mu = mean(v), r = 1 / sqrt(mean((v - mu)^2) + epsilon).
 * z is the norm of h before h is rounded to its type.  Missing weights count as
 * 1, missing biases as 0. */
enum { EPS_B200_NORM_RMS = 0, EPS_B200_NORM_LAYER = 1 };
enum { EPS_B200_GATE_NONE = 0, EPS_B200_GATE_ROW = 1, EPS_B200_GATE_ELEMENT = 2 };
enum { EPS_B200_ACT_NONE = 0, EPS_B200_ACT_SIGMOID = 1, EPS_B200_ACT_SILU = 2, EPS_B200_ACT_TANH = 3 };

#define EPS_B200_BLOCK_NORM_COLUMNS 8192u  /* most columns of a row */

typedef struct {
  int32_t device;
  int32_t kind, gate_kind, activation;
  int32_t post_norm, pre_norm;
  int32_t type;                  /* of y, gate and z, and of their gradients */
  int32_t residual_type;         /* of x and h, and of their gradients: `type` or EPS_B200_F32 */
  int32_t parameter_type;        /* of weights, biases and channel_scale: `type` or EPS_B200_F32 */
  uint32_t columns;
  uint64_t rows;
  float epsilon, scale;
  const void *y, *gate;          /* [rows, columns]; gate [rows] for EPS_B200_GATE_ROW, contiguous */
  int64_t y_stride, gate_stride;
  const void *post_weight, *post_bias, *channel_scale, *pre_weight, *pre_bias;  /* [columns] or NULL */
} EpsB200BlockNorm;

/* h may be NULL if y is (h is x then). */
EPS_B200_EXPORT int eps_b200_block_norm(const EpsB200BlockNorm* args, const void* x, int64_t x_stride,
                                        void* h, int64_t h_stride, void* z, int64_t z_stride,
                                        void* stream, EpsB200Status* status);

/* Gradients of the above from dh and dz (NULL: no gradient comes that way), the
 * statistics recomputed from h and y.  dx is the gradient of x and, where a user
 * differentiates h alone, of h.  Outputs may be NULL if unwanted; dy and dgate are
 * NULL without y.  The parameters' gradients are float32, written, not added.
 * Row sums over the batch are taken in an order that only the sizes, alignment, strides
 * and the GPU decide, so results repeat exactly.  `workspace` holds
 * eps_b200_block_norm_workspace() bytes. */
typedef struct {
  const void *dh, *dz, *h;
  int64_t dh_stride, dz_stride, h_stride;
  void *dx, *dy, *dgate;         /* dgate [rows] for EPS_B200_GATE_ROW */
  int64_t dx_stride, dy_stride, dgate_stride;
  float *dpost_weight, *dpost_bias, *dchannel_scale, *dpre_weight, *dpre_bias;  /* [columns] */
  void* workspace;
  uint64_t workspace_bytes;
} EpsB200BlockNormGradients;
EPS_B200_EXPORT uint64_t eps_b200_block_norm_workspace(uint64_t rows, uint32_t columns);
EPS_B200_EXPORT int eps_b200_block_norm_backward(const EpsB200BlockNorm* args,
                                                 const EpsB200BlockNormGradients* gradients,
                                                 void* stream, EpsB200Status* status);

/* ---- Routing of tokens to experts.
 *   s = softmax(logits) or sigmoid(logits)      a row of -inf alone has s = 0
 *   key = s + bias[e]                           the bias ranks, it does not weigh;
 *                                               the lowest where the logit is -inf
 *   the `top_groups` best of `groups` equal runs of experts, by the sum of their
 *   two best keys (their only key in groups of one expert);
 *   the `top_k` best keys of those groups, best first;
 *   weight = s (divided by their sum if `renormalise`; 0 if that is 0) * scale.
 * Equal keys and equal groups go to the lower index.  A key that is NaN or -inf, and
 * that of a masked expert (logit -inf) whatever its bias, ranks as the lowest finite
 * value; a NaN score stays NaN in its weight.
 *
 * With `order` given, the entries (token * top_k + slot) sorted by expert, equal
 * experts in entry order, their inverse `position`, and offsets[e] .. offsets[e + 1],
 * the run of expert e in `order`.  Needs eps_b200_route_experts_workspace() bytes (0 for
 * one tile of tokens). */
enum { EPS_B200_SCORE_SOFTMAX = 0, EPS_B200_SCORE_SIGMOID = 1 };
#define EPS_B200_ROUTE_EXPERTS 1024u       /* most experts */
#define EPS_B200_ROUTE_TOP_K 32u           /* most experts of a token */

typedef struct {
  int32_t device;
  int32_t type;                  /* of logits and dlogits */
  int32_t score, renormalise;
  uint32_t experts, top_k, groups, top_groups;
  uint64_t tokens;               /* tokens * top_k < 2^31 */
  float scale;
  int32_t reserved;
  const void* logits;            /* [tokens, experts] */
  int64_t logits_stride;
} EpsB200RouteExperts;

EPS_B200_EXPORT uint64_t eps_b200_route_experts_workspace(uint64_t tokens, uint32_t experts,
                                                          uint32_t top_k);
EPS_B200_EXPORT int eps_b200_route_experts(const EpsB200RouteExperts* args, const float* bias,
                                           int32_t* chosen, float* weights,
                                           int32_t* order, int32_t* position, int32_t* offsets,
                                           void* workspace, uint64_t workspace_bytes,
                                           void* stream, EpsB200Status* status);
/* dlogits from the weights' gradients (contiguous [tokens, top_k], like `chosen`);
 * bias, groups and the choice itself take no gradient.  Entries of `chosen`
 * outside [0, experts) are skipped. */
EPS_B200_EXPORT int eps_b200_route_experts_backward(const EpsB200RouteExperts* args,
                                                    const int32_t* chosen, const float* dweights,
                                                    void* dlogits, int64_t dlogits_stride,
                                                    void* stream, EpsB200Status* status);

/* ---- Matrix products in 8-bit integers, a scale for each token and channel.
 * quantize: q[r, k] = round-half-even(x[row(r), k] * (127 * (1 / amax))) and
 * scale[r] = amax / 127, every operation rounded to float, with amax =
 * max_k |x[row(r), k]|; row(r) = rows[r] / rows_divisor, or r without `rows`.  q has a row stride of eps_b200_int8_stride(inner) bytes, zeros
 * behind `inner`.  Where 1 / amax could overflow (amax < 2^-120) the row's q and
 * scale are 0; a row holding NaN or infinity has a NaN scale; an entry of `rows`
 * outside x counts as such a row. */
EPS_B200_EXPORT uint64_t eps_b200_int8_stride(uint32_t inner);
EPS_B200_EXPORT int eps_b200_int8_quantize(int32_t device, int32_t type, const void* x,
                                           int64_t x_stride, uint64_t x_rows, uint32_t inner,
                                           const int32_t* rows, uint32_t rows_divisor,
                                           uint64_t count, int8_t* q, float* scale, void* stream,
                                           EpsB200Status* status);
/* out[r, n] = (sum_k q[r, k] * weight[e, n, k]) * scale[r] * weight_scale[e, n]
 *             + bias[e, n]
 * for the rows r of expert e: offsets[e] .. offsets[e + 1] (device, [experts + 1]),
 * or all rows if offsets is NULL (experts == 1).  The sum is exact.  Offsets are
 * read as clamped to [0, rows] and a run that ends before it begins as empty; rows
 * of no run are not written.  q, weight and out 16-byte aligned; q and weight have
 * row strides of eps_b200_int8_stride(inner) with zeros behind `inner` (at most
 * EPS_B200_INT8_INNER, so that the sum fits 32 bits), out is contiguous. */
#define EPS_B200_INT8_INNER 131072u
typedef struct {
  int32_t device;
  int32_t type;                  /* of x (where given) and out */
  uint32_t experts, channels, inner;
  uint32_t rows_divisor;
  uint64_t rows;                 /* < 2^31 */
  const int8_t* weight;          /* [experts, channels, stride] */
  const float* weight_scale;     /* [experts, channels] */
  const float* bias;             /* [experts, channels] or NULL */
  const int32_t* offsets;
  void* out;                     /* [rows, channels] */
  void* workspace;
  uint64_t workspace_bytes;
} EpsB200Int8Product;
EPS_B200_EXPORT uint64_t eps_b200_int8_product_workspace(uint64_t rows, uint32_t experts,
                                                         uint32_t channels, uint32_t inner);
EPS_B200_EXPORT int eps_b200_int8_product(const EpsB200Int8Product* args, const int8_t* q,
                                          const float* scale, void* stream, EpsB200Status* status);
/* quantize and product in one call, q and scale in the workspace of
 * eps_b200_int8_product_workspace() bytes (0 for few rows: then they need none). */
EPS_B200_EXPORT int eps_b200_int8_linear(const EpsB200Int8Product* args, const void* x,
                                         int64_t x_stride, uint64_t x_rows, const int32_t* rows,
                                         void* stream, EpsB200Status* status);

/* ---- One AdamW step over many tensors (decoupled weight decay).
 *   g = gradient * *gradient_scale              (1 if NULL)
 *   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr * weight_decay) - lr / (1 - beta1^step) * m / (sqrt(v / (1 - beta2^step)) + epsilon)
 * all in 32 bits; an epsilon below the smallest normal float counts as that.  A step
 * whose *skip is nonzero changes nothing.  Unlike the store's LazyAdam, epsilon is
 * added after the bias correction and every element moves at every step.
 *
 * The moments of all tensors lie in one buffer each, tensor i from element
 * state_begin[i], a multiple of EPS_B200_ADAMW_BLOCK.  state_bits == 32: float.
 * state_bits == 8: e4m3 values with one float scale per EPS_B200_ADAMW_BLOCK
 * elements (the largest magnitude / 448); `first` holds m rounded to the nearest,
 * `second` sqrt(v) rounded up or down at random, right on average: nearest would
 * hold v still wherever a step moves it by less than half a unit (3 %).  A root
 * above zero stays above zero.  The random bits are a function of seed, step and
 * element, so a step repeats exactly.
 *
 * `master`, if given, holds the parameters in float at the moments' places; they
 * are then updated there and rounded into `parameters`. */
#define EPS_B200_ADAMW_BLOCK 256u

typedef struct {
  void* parameter;
  const void* gradient;
  uint64_t elements;
  uint64_t state_begin;
} EpsB200AdamWTensor;

typedef struct {
  int32_t device;
  int32_t parameter_type, gradient_type;   /* gradients: parameter_type or EPS_B200_F32 */
  int32_t state_bits;                      /* 32 or 8 */
  float* master;
  void *first, *second;
  float *first_scale, *second_scale;       /* state_bits == 8 */
  const float* gradient_scale;             /* device scalar or NULL */
  const int32_t* skip;                     /* device scalar or NULL */
  double learning_rate, beta1, beta2, epsilon, weight_decay;
  uint64_t step;                           /* this step's number, from 1 */
  uint64_t seed;
} EpsB200AdamW;

/* Lays the tensors out for eps_b200_adamw: `plan` (host, eps_b200_adamw_plan_bytes()
 * bytes) is to be copied to the device by the caller and stays valid as long as
 * pointers and sizes do.  *blocks_out receives the plan's block count. */
EPS_B200_EXPORT uint64_t eps_b200_adamw_plan_bytes(const EpsB200AdamWTensor* tensors, uint64_t count);
EPS_B200_EXPORT int eps_b200_adamw_plan(const EpsB200AdamWTensor* tensors, uint64_t count, void* plan,
                                        uint64_t plan_bytes, uint64_t* blocks_out,
                                        EpsB200Status* status);
EPS_B200_EXPORT int eps_b200_adamw(const EpsB200AdamW* args, const void* plan, uint64_t count,
                                   uint64_t blocks, void* stream, EpsB200Status* status);

/* The step for a captured graph.  eps_b200_adamw takes its number by value, and with it
 * the bias corrections, the learning rate and the random bits: every replay would be the
 * same step again.  This one reads them from `clock`, in device memory of the caller's
 * that lives between the calls: the step's number is args->step + taken, and each call or
 * replay adds 1 to taken (a skipped step too).  A learning_rate of 0 or more there takes
 * the place of args->learning_rate; below 0 the latter holds.  The other members are
 * written by the call. */
typedef struct {
  int64_t taken;
  double learning_rate;
  float decay, rate, inverse_root;
  uint32_t key;
} EpsB200AdamWClock;
EPS_B200_EXPORT int eps_b200_adamw_counted(const EpsB200AdamW* args, const void* plan, uint64_t count,
                                           uint64_t blocks, EpsB200AdamWClock* clock, void* stream,
                                           EpsB200Status* status);

/* ---- The norm over many gradients, the factor that clips it, and clipping in place.
 *   u = *gradient_scale                          1 if NULL
 *   norm = |u| sqrt(sum g^2)                     EPS_B200_GRADIENT_L2
 *   norm = |u| max |g|                           EPS_B200_GRADIENT_MAX
 *   scale = u * min(1, max_norm / norm)          u where norm is 0
 * Where norm is not finite (as a float) skip is 1 and scale 0; else skip is 0.  scale
 * and skip are what eps_b200_adamw takes.  With `clip` every gradient becomes
 * gradient * scale, a product in float that is then rounded to the gradient's type, and
 * stays as it is where skip is 1.  Sums are taken in 64 bits (the squares of 16 bytes
 * first in float, where it holds them), in an order that only the sizes, the gradients'
 * alignment and the GPU decide, so results repeat exactly. */
enum { EPS_B200_GRADIENT_L2 = 0, EPS_B200_GRADIENT_MAX = 1 };

typedef struct {
  void* gradient;
  uint64_t elements;
  int32_t type;                  /* each tensor has its own */
  int32_t reserved;
} EpsB200Gradient;

typedef struct {
  float norm, scale;
  int32_t skip;
} EpsB200GradientResult;

/* Lays the tensors out for eps_b200_gradient_norm, as eps_b200_adamw_plan does for
 * AdamW: `plan` (host, eps_b200_gradient_norm_plan_bytes() bytes) is to be copied to
 * the device by the caller, 16-byte aligned, and *blocks_out receives its block count.
 * Tensors that overlap are refused. */
EPS_B200_EXPORT uint64_t eps_b200_gradient_norm_plan_bytes(const EpsB200Gradient* tensors, uint64_t count);
EPS_B200_EXPORT int eps_b200_gradient_norm_plan(const EpsB200Gradient* tensors, uint64_t count, void* plan,
                                                uint64_t plan_bytes, uint64_t* blocks_out,
                                                EpsB200Status* status);
typedef struct {
  int32_t device;
  int32_t kind, clip;
  int32_t reserved;
  const void* plan;
  uint64_t blocks;
  const float* gradient_scale;   /* device scalar or NULL; no part of result, such as the
                                    scale of the call before, nor of a gradient */
  double max_norm;               /* >= 0; infinity: nothing is clipped */
  EpsB200GradientResult* result; /* device; with gradient_scale, outside the workspace */
  void* workspace;
  uint64_t workspace_bytes;
} EpsB200GradientNorm;
EPS_B200_EXPORT uint64_t eps_b200_gradient_norm_workspace(uint64_t blocks);
EPS_B200_EXPORT int eps_b200_gradient_norm(const EpsB200GradientNorm* args, void* stream, EpsB200Status* status);

/* ---- A loss that balances the experts, and how many entries each has.
 *   s = softmax(logits) or sigmoid(logits)       a row of -inf alone has s = 0
 *   p = s / sum_e s                              s itself if not `normalise` (0 if the
 *                                                sum is 0; a softmax is normalised as it is)
 * A sigmoid counts as 0 where a float hardly tells it from 0, at logits of -88.71 and below
 * (the router's weights end at -88.72).
 * over the tokens whose mask is not 0 (all without a mask), n of them:
 *   counts[e] = entries of chosen[t, :] that are e; entries outside [0, experts) count for none
 *   mass[e] = sum_t p[t, e]
 *   loss = weight * experts / (top_k * n^2) * sum_e counts[e] * mass[e]     0 if n is 0
 * What masked tokens hold is read by no sum.  Sums over tokens are taken in an order
 * that only the sizes, the logits' alignment and stride and the GPU decide, in float over
 * 64 rows a lane at most and in 64 bits beyond, so their error does not grow with the
 * tokens.  Of several ranks with a batch each, counts,
 * mass and counted add up to those of the joint batch; backward takes the sums. */
typedef struct {
  int32_t device;
  int32_t type;                  /* of logits, add and dlogits */
  int32_t score, normalise;
  uint32_t experts, top_k;       /* at most EPS_B200_ROUTE_EXPERTS and EPS_B200_ROUTE_TOP_K */
  uint64_t tokens;               /* tokens * top_k < 2^31 */
  float weight;
  int32_t reserved;
  const void* logits;            /* [tokens, experts] */
  int64_t logits_stride;
  const uint8_t* mask;           /* [tokens] or NULL */
} EpsB200BalanceLoss;

EPS_B200_EXPORT uint64_t eps_b200_balance_loss_workspace(uint64_t tokens, uint32_t experts);
EPS_B200_EXPORT int eps_b200_balance_loss(const EpsB200BalanceLoss* args, const int32_t* chosen,
                                          float* loss, int32_t* counts, float* mass, int32_t* counted,
                                          void* workspace, uint64_t workspace_bytes,
                                          void* stream, EpsB200Status* status);
/* dlogits = *dloss * (the loss's gradient) + add, rounded once; masked tokens get `add`
 * alone.  dloss NULL: 1; add NULL: 0; dlogits may be `add` or the logits themselves, and
 * must not overlap them otherwise.  The counts take no gradient. */
EPS_B200_EXPORT int eps_b200_balance_loss_backward(const EpsB200BalanceLoss* args, const int32_t* counts,
                                                   const int32_t* counted, const float* dloss,
                                                   const void* add, int64_t add_stride,
                                                   void* dlogits, int64_t dlogits_stride,
                                                   void* stream, EpsB200Status* status);

/* ---- Low-rank adapters of many requests at once, beside a layer that they share.
 *   a = ids[t];  out[t] = base[t] + scale[a] * up[a] (down[a] x[t])
 * An id outside [0, adapters) is no adapter: out[t] is base[t].  base NULL: 0; out may
 * be base itself, and must overlap nothing else that is read.  down [adapters, R, K'] and
 * up [adapters, channels, R] are contiguous and 16-byte aligned; inner, channels and strides are below
 * 2^30.  R = eps_b200_low_rank_rank(rank)
 * and K' = eps_b200_low_rank_inner(inner), and zeros behind `rank` and `inner`.  All
 * have one type.  `workspace` holds eps_b200_low_rank_workspace() bytes (0 for few rows).
 * Products are exact and sums are held in 32 bits; down[a] x[t] is
 * kept to 16 bits of mantissa or more (24 with float, where infinity, NaN or a magnitude
 * from 3.38e38 on in x[t], down, up or a sum makes what it enters NaN).  A row's result
 * does not depend on the other rows' values (on the numbers of rows and of adapters it does,
 * by a rounding: sums are shared out by them). */
#define EPS_B200_LOW_RANK 128u             /* most ranks */
#define EPS_B200_LOW_RANK_ADAPTERS 16384u  /* most adapters */
typedef struct {
  int32_t device;
  int32_t type;
  uint32_t adapters, rank, inner, channels;
  uint64_t rows;                 /* < 2^31 */
  const void *down, *up;
  const float* scale;            /* [adapters] or NULL: 1 */
  const int32_t* ids;            /* [rows] */
  const void *x, *base;          /* [rows, inner], [rows, channels] */
  void* out;                     /* [rows, channels] */
  int64_t x_stride, base_stride, out_stride;
  void* workspace;
  uint64_t workspace_bytes;
} EpsB200LowRank;
EPS_B200_EXPORT uint64_t eps_b200_low_rank_rank(uint32_t rank);
EPS_B200_EXPORT uint64_t eps_b200_low_rank_inner(uint32_t inner);
EPS_B200_EXPORT uint64_t eps_b200_low_rank_workspace(uint64_t rows, uint32_t adapters);
EPS_B200_EXPORT int eps_b200_low_rank(const EpsB200LowRank* args, void* stream, EpsB200Status* status);

#ifdef __cplusplus
}
#endif
#endif /* EPS_B200_DENSE_H */
