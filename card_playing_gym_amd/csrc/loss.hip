// The clipped policy loss of an update on the device (gfx950): forward and gradient over rows of
// policy logits, with an entropy bonus and a KL term towards a reference policy.
//
// A row's legal entries are those its mask keeps and whose logit is above -inf; p is the softmax over
// them.  With x = z - max, S = sum e^x and T = sum e^x x over the legal entries:
//   log p_j = x_j - log S,   H = log S - T / S          (both terms of H are positive: no cancellation)
//   r = exp(log p_a - old),  l = -min(r A, clamp(r, lo, hi) A) + beta K - c H
//   K = sum p_j (log p_j - log q_j) from the reference's logits, or e^d - d - 1 with
//   d = log q_a - log p_a from the reference's log-probability of the action,
//   dl/dz_j = p_j (c (log p_j + H) + beta (log p_j - log q_j - K) - A') + [j = a] A'
// where A' = dl / d log p_a, -r A where the unclipped product is the smaller (or r is inside), plus
// beta (1 - e^d) with the second K.  The gradient of the sum of w l over `normalizer` is written in the
// same pass, for an upstream gradient of 1; a backward call with another one forms it again from the
// inputs, so it is rounded once whatever the upstream scale.
//
// Bound by HBM: every logit (mask byte, reference logit) is read once and every gradient written once.
// A row stays in registers between the passes over it: its maximum, its sums, its gradient.
//
// The row's scalars are formed in fp64: the ends of the clip range are borders where the gradient jumps,
// and a ratio off by fp32's 1e-6 would cross one in a few of a million rows.  A lane's partial sums over
// its entries are fp32, joined in fp64.
#include <cmath>

#include "common.h"

namespace cg {
namespace {

constexpr int MAX_BLOCKS = 2048;  // and partial sums of the loss
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LOWEST = -1e30f;  // in place of the log-probability of an entry with p = 0 where p multiplies it

struct Scalar {
  float value;
  const float *at;  // NULL: value
};
__device__ __forceinline__ double read(const Scalar &s) { return double(s.at ? *s.at : s.value); }

struct LossArgs {
  const void *logits, *ref_logits;
  const uint8_t *mask;
  const int64_t *actions;
  const float *old, *advantages, *weights, *ref;
  int64_t ld_logits, ld_ref, ld_mask;
  int32_t rows, width;
  double lo, hi;
  Scalar normalizer, entropy_coef, kl_coef;
  float *log_probs, *entropy, *kl;  // NULL in a backward call
  void *grad;                       // NULL: none
  double *partials;
  float *loss;
  const float *upstream;  // of a backward call
  int32_t written;        // the gradient for an upstream of 1 is in place
};

// ---- a group of G lanes that share a row: reductions that leave the result in every lane ---------------

template <int CONTROL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CONTROL, 0xf, 0xf, false));
}
template <int CONTROL>
__device__ __forceinline__ double dpp(double x) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CONTROL, 0xf, 0xf, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(x), CONTROL, 0xf, 0xf, false));
}
struct Add {
  __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};
struct Most {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// Within a wave: the lane's neighbour, the pair's, the quad's (mirrored halves of eight), the other eight
// of the row of 16, the other rows.
template <int G, typename X, typename Op>
__device__ __forceinline__ X lanes_join(X x, Op op) {
  x = op(x, dpp<0xB1>(x));   // quad_perm [1, 0, 3, 2]
  x = op(x, dpp<0x4E>(x));   // quad_perm [2, 3, 0, 1]
  x = op(x, dpp<0x141>(x));  // row_half_mirror
  if constexpr (G > 8) x = op(x, dpp<0x128>(x));  // row_ror:8
  if constexpr (G > 16) {
    x = op(x, __shfl_xor(x, 16, 64));
    x = op(x, __shfl_xor(x, 32, 64));
  }
  return x;
}

// Over several waves through LDS.  Each reduction of a row has a slot of its own, so a slot is written
// again only behind another's barrier, which every wave reaches after its reads.
template <int G, int N, typename X, typename Op>
__device__ __forceinline__ void join(X (&x)[N], X *slot, Op op) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = lanes_join<(G < 64 ? G : 64)>(x[i], op);
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) slot[i * W + (threadIdx.x >> 6)] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      X s = slot[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) s = op(s, slot[i * W + w]);
      x[i] = s;
    }
  }
}

template <int G>
struct Slots {
  static constexpr int W = G > 64 ? G / 64 : 1;
  float tops[2 * W];
  double sums[3 * W], gaps[W];
};

// ---- entries --------------------------------------------------------------------------------------------

template <typename T>
constexpr int VEC = 16 / sizeof(T);

// VEC entries of a row from entry i on, -inf for those past its end or (mask) not legal.  Rows may start
// anywhere: 16 bytes are loaded wherever they begin.  The vector over the row's end is loaded as the
// row's last VEC entries, of which the vector before has the first.
template <typename T>
__device__ __forceinline__ void load_entries(float *z, const T *row, const uint8_t *legal, int i, int width) {
  constexpr int V = VEC<T>;
  if (i >= width) {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = -INFINITY;
    return;
  }
  if (width < V) {
    for (int k = 0; k < V; ++k) {
      z[k] = -INFINITY;
      if (k < width && (!legal || legal[k])) z[k] = to_f32(row[k]);
    }
    return;
  }
  const int at = i + V <= width ? i : width - V, seen = i - at;
  T q[V];
  __builtin_memcpy(q, row + at, sizeof q);
  uint8_t b[V];
  if (legal) __builtin_memcpy(b, legal + at, sizeof b);
  float f[V];
#pragma unroll
  for (int k = 0; k < V; ++k) f[k] = !legal || b[k] ? to_f32(q[k]) : -INFINITY;
  if (seen == 0) {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = f[k];
  } else {
    // entry i + k is f[k + seen]
#pragma unroll
    for (int k = 0; k < V; ++k) {
      z[k] = -INFINITY;
#pragma unroll
      for (int s = 1; s < V; ++s)
        if (k + s < V && seen == s) z[k] = f[k + s];
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_entries(T *row, const float *g, int i, int width) {
  constexpr int V = VEC<T>;
  if (i + V <= width) {
    T q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) q[k] = from_f32<T>(g[k]);
    __builtin_memcpy(row + i, q, sizeof q);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (i + k < width) row[i + k] = from_f32<T>(g[k]);
  }
}

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// ---- a row's scalars ---------------------------------------------------------------------------------------

struct RowSums {
  float top, ref_top;
  double s, t, ref_s;  // sum e^x, sum e^x x, and the reference's sum e^y
};
// The gradient's coefficients: e (base + slope x + pull (z - y - shift)), plus `own` at the action.
struct RowCoefs {
  float base, slope, pull, shift, own;
};
struct RowScalars {
  double log_p, entropy, kl, value;  // value: weight times the row's loss
  RowCoefs c;
  bool live;
};

// gap(shift): sum of e (z - y - shift), of the whole group (called by all of it).
template <bool REF, typename Gap>
__device__ __forceinline__ RowScalars row_scalars(const LossArgs &a, int64_t row, float action_logit, double weight,
                                                  const RowSums &q, double scale, const Gap &gap) {
  RowScalars o;
  o.live = weight != 0 && q.s != 0;
  const double log_s = log(q.s), c = read(a.entropy_coef), beta = read(a.kl_coef);
  o.log_p = (double(action_logit) - double(q.top)) - log_s;
  o.entropy = log_s - q.t / q.s;
  const double adv = a.advantages[row], r = exp(o.log_p - double(a.old[row]));
  const double bounded = r < a.lo ? a.lo : r > a.hi ? a.hi : r;  // (NaN stays)
  const double whole = r * adv, part = bounded * adv;
  double value = -(part < whole ? part : whole) - c * o.entropy;
  double own = r == bounded || whole < part ? -whole : 0;
  if (whole != whole) own = value = whole;
  double shift = 0, base = c * (o.entropy - log_s);
  o.kl = 0;
  if constexpr (REF) {
    shift = (double(q.top) - double(q.ref_top)) + (log_s - log(q.ref_s));
    const double k = gap(float(shift)) / q.s;
    o.kl = k;
    value += beta * k;
    base -= beta * k;
  } else if (a.ref) {
    const double d = double(a.ref[row]) - o.log_p, rise = expm1(d);
    o.kl = rise == INFINITY ? rise : rise - d;
    value += beta * o.kl;
    own -= beta * rise;
  }
  const double f = weight * scale;
  o.value = weight * value;
  o.c.own = float(f * own);
  o.c.base = float(f * (base - own) / q.s);
  o.c.slope = float(f * c / q.s);
  o.c.pull = REF ? float(f * beta / q.s) : 0.f;
  o.c.shift = float(shift);
  return o;
}

// x = z - top and its exponential.  The product of an entry of p = 0 with its x is 0, never 0 * inf.
struct Entry {
  float e, x;
};
__device__ __forceinline__ Entry entry_of(float z, float top) {
  const float x = z - top;
  return Entry{exp_of(x), fmaxf(x, LOWEST)};  // (a NaN is kept by e)
}
template <bool REF>
__device__ __forceinline__ float gap_of(float e, float z, float y, float shift) {
  return REF && e > 0 ? (z - y) - shift : 0.f;
}
template <bool REF>
__device__ __forceinline__ float grad_of(float z, float y, float top, const RowCoefs &c) {
  const Entry n = entry_of(z, top);
  float u = fmaf(c.slope, n.x, c.base);
  if (REF) u = fmaf(c.pull, gap_of<REF>(n.e, z, y, c.shift), u);
  return n.e * u;
}

__device__ __forceinline__ void report(const LossArgs &a, int64_t row, const RowScalars &o) {
  a.log_probs[row] = o.live ? float(o.log_p) : 0.f;
  a.entropy[row] = o.live ? float(o.entropy) : 0.f;
  if (a.kl) a.kl[row] = o.live ? float(o.kl) : 0.f;
}

// The block's sum of `value` over its threads, to its partial sum, or the loss where it is the only one.
__device__ __forceinline__ void block_loss(const LossArgs &a, double value) {
  __shared__ double sums[16];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) value += __shfl_xor(value, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = value;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double s = 0;
  for (int w = 0; w < int(blockDim.x >> 6); ++w) s += sums[w];
  if (gridDim.x == 1)
    *a.loss = float(s / read(a.normalizer));
  else
    a.partials[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void loss_kernel(const LossArgs a, int count) {
  double s = 0;
  for (int k = threadIdx.x; k < count; k += 256) s += a.partials[k];
  block_loss(a, s);  // (of one block)
}

// Whether this call has nothing to do: a backward whose gradient is in place already.
__device__ __forceinline__ bool done(const LossArgs &a) { return a.upstream && a.written && *a.upstream == 1.0f; }

__device__ __forceinline__ double scale_of(const LossArgs &a) {
  return (a.upstream ? double(*a.upstream) : 1.0) / read(a.normalizer);
}

// The action's logit; NaN for an action outside the row, -inf for one that is not legal.
template <typename T>
__device__ __forceinline__ float logit_of(const LossArgs &a, int64_t row, int64_t action) {
  if (action < 0 || action >= a.width) return NAN;
  if (a.mask && !a.mask[row * a.ld_mask + action]) return -INFINITY;
  return to_f32(static_cast<const T *>(a.logits)[row * a.ld_logits + action]);
}

// ---- rows in registers: E entries a lane, G lanes a row, 256 / G rows a block at a time (one from 256 on) -----

template <typename T, int G, int E, bool REF>
__global__ __launch_bounds__(G > 256 ? G : 256) void rows_kernel(const LossArgs a) {
  constexpr int V = VEC<T>, C = E / V, THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  const int lane = threadIdx.x % G;
  const double scale = scale_of(a);
  double value = 0;
  // every thread of the block takes every turn: lanes of rows past the end have nothing live
  for (int64_t first = int64_t(blockIdx.x) * ROWS; first < a.rows; first += int64_t(gridDim.x) * ROWS) {
    const int64_t mine = first + threadIdx.x / G;
    const bool in = mine < a.rows;
    const int64_t row = in ? mine : a.rows - 1;
    const double weight = !in ? 0.0 : a.weights ? double(a.weights[row]) : 1.0;
    const int width = weight != 0 ? a.width : 0;  // rows without weight are not read
    const int64_t action = a.actions[row];
    const T *logits = static_cast<const T *>(a.logits) + row * a.ld_logits;
    const T *ref = static_cast<const T *>(a.ref_logits) + (REF ? row * a.ld_ref : 0);
    const uint8_t *legal = a.mask ? a.mask + row * a.ld_mask : nullptr;
    float z[E], y[REF ? E : 1];
#pragma unroll
    for (int c = 0; c < C; ++c) load_entries(z + c * V, logits, legal, (c * G + lane) * V, width);
    if constexpr (REF) {
#pragma unroll
      for (int c = 0; c < C; ++c) load_entries(y + c * V, ref, legal, (c * G + lane) * V, width);
    }
    const float action_logit = width ? logit_of<T>(a, row, action) : 0.f;
    RowSums q;
    float tops[REF ? 2 : 1];
    tops[0] = z[0];
#pragma unroll
    for (int k = 1; k < E; ++k) tops[0] = fmaxf(tops[0], z[k]);
    if constexpr (REF) {
      tops[1] = y[0];
#pragma unroll
      for (int k = 1; k < E; ++k) tops[1] = fmaxf(tops[1], y[k]);
    }
    join<G>(tops, slots.tops, Most{});
    q.top = tops[0] > -INFINITY ? tops[0] : 0.f;
    q.ref_top = REF && tops[REF ? 1 : 0] > -INFINITY ? tops[REF ? 1 : 0] : 0.f;
    float s = 0, t = 0, rs = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const Entry n = entry_of(z[k], q.top);
      s += n.e;
      t = fmaf(n.e, n.x, t);
      if (REF) rs += exp_of(y[REF ? k : 0] - q.ref_top);
    }
    double sums[REF ? 3 : 2];
    sums[0] = s, sums[1] = t;
    if constexpr (REF) sums[2] = rs;
    join<G>(sums, slots.sums, Add{});
    q.s = sums[0], q.t = sums[1], q.ref_s = REF ? sums[REF ? 2 : 0] : 0;
    const RowScalars o = row_scalars<REF>(a, row, action_logit, weight, q, scale, [&](float shift) {
      float g = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float e = exp_of(z[k] - q.top);
        g = fmaf(e, gap_of<REF>(e, z[k], y[REF ? k : 0], shift), g);
      }
      double gaps[1] = {g};
      join<G>(gaps, slots.gaps, Add{});
      return gaps[0];
    });
    if (!in) continue;  // (all lanes of a group; the reductions are behind)
    if (lane == 0 && a.log_probs) {
      if (o.live) value += o.value;
      report(a, row, o);
    }
    if (a.grad) {
      T *grad = static_cast<T *>(a.grad) + row * int64_t(a.width);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int i = (c * G + lane) * V;
        if (i >= a.width) break;
        float g[V];
#pragma unroll
        for (int k = 0; k < V; ++k)
          g[k] = o.live ? grad_of<REF>(z[c * V + k], y[REF ? c * V + k : 0], q.top, o.c) : 0.f;
        store_entries(grad, g, i, a.width);
      }
      // The action's own term, by the lane that has just written that entry.
      if (o.live && action >= 0 && action < a.width && action / V % G == lane) {
        const float yr = REF && action_logit > -INFINITY ? to_f32(ref[REF ? action : 0]) : 0.f;
        grad[action] = from_f32<T>(grad_of<REF>(action_logit, yr, q.top, o.c) + o.c.own);
      }
    }
  }
  if (a.log_probs) block_loss(a, value);
}

// ---- rows of any width: a block a row, read again for each pass ----------------------------------------------

template <typename T, bool REF>
__global__ __launch_bounds__(1024) void long_rows_kernel(const LossArgs a) {
  constexpr int V = VEC<T>, G = 1024;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  const double scale = scale_of(a);
  double value = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const double weight = a.weights ? double(a.weights[row]) : 1.0;
    const int width = weight != 0 ? a.width : 0;
    const int64_t action = a.actions[row];
    const T *logits = static_cast<const T *>(a.logits) + row * a.ld_logits;
    const T *ref = static_cast<const T *>(a.ref_logits) + (REF ? row * a.ld_ref : 0);
    const uint8_t *legal = a.mask ? a.mask + row * a.ld_mask : nullptr;
    const float action_logit = width ? logit_of<T>(a, row, action) : 0.f;
    const auto each = [&](const auto &visit) {  // visit(first entry, logits, reference logits)
      for (int64_t i = int64_t(threadIdx.x) * V; i < width; i += G * V) {
        float z[V], y[V];
        load_entries(z, logits, legal, int(i), width);
        if (REF) load_entries(y, ref, legal, int(i), width);
        visit(int(i), z, y);
      }
    };
    RowSums q;
    float tops[REF ? 2 : 1];
    tops[0] = tops[REF ? 1 : 0] = -INFINITY;
    each([&](int, const float *z, const float *y) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        tops[0] = fmaxf(tops[0], z[k]);
        if (REF) tops[REF ? 1 : 0] = fmaxf(tops[REF ? 1 : 0], y[k]);
      }
    });
    join<G>(tops, slots.tops, Most{});
    q.top = tops[0] > -INFINITY ? tops[0] : 0.f;
    q.ref_top = REF && tops[REF ? 1 : 0] > -INFINITY ? tops[REF ? 1 : 0] : 0.f;
    double sums[REF ? 3 : 2] = {};
    each([&](int, const float *z, const float *y) {
      float s = 0, t = 0, rs = 0;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const Entry n = entry_of(z[k], q.top);
        s += n.e;
        t = fmaf(n.e, n.x, t);
        if (REF) rs += exp_of(y[k] - q.ref_top);
      }
      sums[0] += s, sums[1] += t;
      if (REF) sums[REF ? 2 : 0] += rs;
    });
    join<G>(sums, slots.sums, Add{});
    q.s = sums[0], q.t = sums[1], q.ref_s = REF ? sums[REF ? 2 : 0] : 0;
    const RowScalars o = row_scalars<REF>(a, row, action_logit, weight, q, scale, [&](float shift) {
      double gaps[1] = {};
      each([&](int, const float *z, const float *y) {
        float g = 0;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float e = exp_of(z[k] - q.top);
          g = fmaf(e, gap_of<REF>(e, z[k], y[k], shift), g);
        }
        gaps[0] += g;
      });
      join<G>(gaps, slots.gaps, Add{});
      return gaps[0];
    });
    if (threadIdx.x == 0 && a.log_probs) {
      if (o.live) value += o.value;
      report(a, row, o);
    }
    if (!a.grad) continue;
    T *grad = static_cast<T *>(a.grad) + row * int64_t(a.width);
    if (o.live) {
      each([&](int i, const float *z, const float *y) {
        float g[V];
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] = grad_of<REF>(z[k], y[k], q.top, o.c);
        store_entries(grad, g, i, a.width);
      });
      if (action >= 0 && action < a.width && action / V % G == threadIdx.x) {
        const float yr = REF && action_logit > -INFINITY ? to_f32(ref[REF ? action : 0]) : 0.f;
        grad[action] = from_f32<T>(grad_of<REF>(action_logit, yr, q.top, o.c) + o.c.own);
      }
    } else {
      const float zero[V] = {};
      for (int64_t i = int64_t(threadIdx.x) * V; i < a.width; i += G * V) store_entries(grad, zero, int(i), a.width);
    }
  }
  if (a.log_probs) block_loss(a, value);
}

// ---- host side ---------------------------------------------------------------------------------------------------

struct Launch {
  void (*kernel)(LossArgs);
  int rows, threads;  // rows a block takes at a time
};

template <typename T, bool REF>
Launch launch_of(int width) {
  if (width <= 64) return {rows_kernel<T, 8, 8, REF>, 32, 256};
  if (width <= 128) return {rows_kernel<T, 16, 8, REF>, 16, 256};
  if (width <= 256) return {rows_kernel<T, 16, 16, REF>, 16, 256};
  if (width <= 512) return {rows_kernel<T, 64, 8, REF>, 4, 256};
  if (width <= 1024) return {rows_kernel<T, 64, 16, REF>, 4, 256};
  if (width <= 2048) return {rows_kernel<T, 256, 8, REF>, 1, 256};
  if (width <= 4096) return {rows_kernel<T, 256, 16, REF>, 1, 256};
  if (width <= 8192) return {rows_kernel<T, 256, 32, REF>, 1, 256};
  if (width <= 16384) return {rows_kernel<T, 1024, 16, REF>, 1, 1024};
  if (width <= 32768) return {rows_kernel<T, 1024, 32, REF>, 1, 1024};
  return {long_rows_kernel<T, REF>, 1, 1024};
}

template <typename T>
Launch launch_of(int width, bool ref) {
  return ref ? launch_of<T, true>(width) : launch_of<T, false>(width);
}

Launch launch_of(const cg_policy_loss &p) {
  const bool ref = p.reference_logits != nullptr;
  return p.dtype == CG_F32    ? launch_of<float>(p.width, ref)
         : p.dtype == CG_BF16 ? launch_of<bf16>(p.width, ref)
                              : launch_of<f16>(p.width, ref);
}

int grid_of(const cg_policy_loss &p, const Launch &l) {
  const int64_t blocks = (int64_t(p.rows) + l.rows - 1) / l.rows;
  return int(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS);
}

Scalar scalar(const cg_scalar &s) { return Scalar{s.value, s.device}; }

LossArgs args_of(const cg_policy_loss *loss) {
  CG_REQUIRE(loss != nullptr, CG_ERR_INVALID, "loss is NULL");
  const cg_policy_loss &p = *loss;
  dtype_size(p.dtype);
  CG_REQUIRE(p.rows >= 0 && p.width > 0, CG_ERR_INVALID, "rows must be non-negative, width positive");
  CG_REQUIRE(p.rows == 0 || (p.logits && p.actions && p.old_log_probs && p.advantages), CG_ERR_INVALID,
             "logits, actions, old_log_probs and advantages are required");
  CG_REQUIRE(!(p.reference_logits && p.reference_log_probs), CG_ERR_INVALID,
             "reference_logits and reference_log_probs exclude each other");
  CG_REQUIRE(p.ld_logits >= 0 && p.ld_mask >= 0 && p.ld_reference >= 0, CG_ERR_INVALID, "row strides must be non-negative");
  LossArgs a{};
  a.logits = p.logits, a.ref_logits = p.reference_logits, a.mask = p.mask, a.actions = p.actions;
  a.old = p.old_log_probs, a.advantages = p.advantages, a.weights = p.weights, a.ref = p.reference_log_probs;
  a.ld_logits = p.ld_logits, a.ld_ref = p.ld_reference, a.ld_mask = p.ld_mask;
  a.rows = p.rows, a.width = p.width;
  a.lo = p.clip_low, a.hi = p.clip_high;
  a.normalizer = scalar(p.normalizer), a.entropy_coef = scalar(p.entropy_coef), a.kl_coef = scalar(p.kl_coef);
  return a;
}

}  // namespace
}  // namespace cg

using namespace cg;

extern "C" {

size_t cg_policy_loss_workspace_size(void) { return MAX_BLOCKS * sizeof(double); }

int cg_policy_loss_forward(const cg_policy_loss *loss, float *value, float *log_probs, float *entropy, float *kl,
                           void *grad, void *workspace, size_t workspace_size, void *stream) {
  return guarded([&] {
    LossArgs a = args_of(loss);
    CG_REQUIRE(value && workspace, CG_ERR_INVALID, "value and workspace are required");
    CG_REQUIRE(workspace_size >= cg_policy_loss_workspace_size(), CG_ERR_INVALID, "workspace too small");
    CG_REQUIRE(a.rows == 0 || (log_probs && entropy), CG_ERR_INVALID, "log_probs and entropy are required");
    CG_REQUIRE(a.rows == 0 || !kl == !(a.ref || a.ref_logits), CG_ERR_INVALID, "kl goes with a reference");
    a.partials = static_cast<double *>(workspace);
    a.loss = value;
    int blocks = 0;
    if (a.rows > 0) {
      a.log_probs = log_probs, a.entropy = entropy, a.kl = kl, a.grad = grad;
      const Launch l = launch_of(*loss);
      blocks = grid_of(*loss, l);
      l.kernel<<<blocks, l.threads, 0, as_stream(stream)>>>(a);
      CG_LAUNCHED();
    }
    if (blocks != 1) {
      loss_kernel<<<1, 256, 0, as_stream(stream)>>>(a, blocks);
      CG_LAUNCHED();
    }
  });
}

int cg_policy_loss_backward(const cg_policy_loss *loss, const float *upstream, int32_t written, void *grad,
                            void *stream) {
  return guarded([&] {
    LossArgs a = args_of(loss);
    CG_REQUIRE(upstream, CG_ERR_INVALID, "upstream is required");
    if (a.rows == 0) return;
    CG_REQUIRE(grad, CG_ERR_INVALID, "grad is required");
    a.grad = grad, a.upstream = upstream, a.written = written;
    const Launch l = launch_of(*loss);
    l.kernel<<<grid_of(*loss, l), l.threads, 0, as_stream(stream)>>>(a);
    CG_LAUNCHED();
  });
}

}  // extern "C"
