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
// A row stays in registers between the passes over it: its maximum, its sums, its gradient.  (Not all of it where
// a lane has 64 entries beside a reference's 64: 16-bit rows of over 16384 entries with reference logits keep up to
// 32 registers of a lane in scratch memory, bf16 4096 x 32768 320 us beside 169 for its bytes at a copy's rate.)
//
// The row's scalars are formed in fp64: the ends of the clip range are borders where the gradient jumps,
// and a ratio off by fp32's 1e-6 would cross one in a few of a million rows.  A lane's partial sums over
// its entries are fp32, joined in fp64.
#include "rows.h"

namespace cg {
namespace {

// Logits and gradient of this many bytes go past the caches (256 MB of Infinity Cache); below, whatever made the
// logits or takes the gradient may find them there.  us kept and past them: fp32 4096 x 16384 (512 MB) 102 and 98,
// 8192 x 16384 205 and 201; bf16, whose time is arithmetic, 4096 x 32768 128-133 and 127-129.
constexpr int64_t STREAM_BYTES = 512 << 20;
constexpr int MAX_BLOCKS = 2048;  // and partial sums of the loss
// The least x = z - top that p = e^x is multiplied by: e^x is 0 from -104 on.  No lower, so that the coefficient
// of x may be as large as 2^120 before the product is infinite, which times p = 0 is NaN.
constexpr float LOWEST = -128.f;

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
  double *parts;          // of split rows: SPLIT_PARTS for each segment
  int32_t splits, segment;  // segments of a row, and entries of one
  int32_t streams;        // the logits and their gradient go past the caches (rows of 512 lanes and more)
};

template <int G>
struct Slots {
  static constexpr int W = G > 64 ? G / 64 : 1;
  float tops[2 * W];
  double sums[3 * W], gaps[W];
};

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

// What a row is beside its logits.
struct RowInputs {
  int64_t action;
  float weight, old, advantage, ref;
};
__device__ __forceinline__ RowInputs row_inputs(const LossArgs &a, int64_t row) {
  return RowInputs{a.actions[row], a.weights ? a.weights[row] : 1.f, a.old[row], a.advantages[row], a.ref ? a.ref[row] : 0.f};
}
struct Coefs {  // of the whole launch
  double entropy, kl, scale;
};

// log p - log q is z - y less this.
__device__ __forceinline__ double shift_of(const RowSums &q, double log_s) {
  return (double(q.top) - double(q.ref_top)) + (log_s - log_of(q.ref_s));
}

// gap(shift): sum of e (z - y - shift), of the whole group (called by all of it).
template <bool REF, typename Gap>
__device__ __forceinline__ RowScalars row_scalars(const LossArgs &a, const RowInputs &in, float action_logit,
                                                  const RowSums &q, const Coefs &k, const Gap &gap) {
  RowScalars o;
  o.live = in.weight != 0 && q.s != 0;
  const double log_s = log_of(q.s), inv = reciprocal(q.s), c = k.entropy, beta = k.kl;
  double base = 0, kl = 0;
  o.c.shift = 0;
  if constexpr (REF) {
    const double shift = shift_of(q, log_s);
    o.c.shift = float(shift);
    kl = gap(o.c.shift) * inv - (shift - double(o.c.shift));  // (p sums to 1)
  }
  o.log_p = (double(action_logit) - double(q.top)) - log_s;
  o.entropy = log_s - q.t * inv;
  base = c * (o.entropy - log_s);
  const double adv = in.advantage, r = exp_of(o.log_p - double(in.old));
  const double bounded = r < a.lo ? a.lo : r > a.hi ? a.hi : r;  // (NaN stays)
  const double whole = r * adv, part = bounded * adv;
  double value = -(part < whole ? part : whole) - c * o.entropy;
  double own = r == bounded || whole < part ? -whole : 0;
  if (whole != whole) own = value = whole;
  double rise = 0;
  if (!REF && a.ref) {
    const double d = double(in.ref) - o.log_p;
    rise = exp_of(d) - 1;
    kl = rise == INFINITY ? rise : rise - d;
  }
  if (beta != 0) {  // (with a coefficient of 0 a reference is reported only, whatever it holds)
    value += beta * kl;
    own -= beta * rise;
    if (REF) base -= beta * kl;
  }
  o.kl = kl;
  const double weight = in.weight, f = weight * k.scale;
  o.value = weight * value;
  // The entries of a row that does not count have e = 0: with these the gradient is 0 without asking.
  o.c.own = float(f * own);
  o.c.base = o.live ? float(f * (base - own) * inv) : 0.f;
  o.c.slope = o.live ? float(f * c * inv) : 0.f;
  o.c.pull = REF && o.live ? float(f * beta * inv) : 0.f;
  o.c.shift = o.live ? o.c.shift : 0.f;
  return o;
}

// A lane's sum of exponentials: in fp64 where the logarithms of two rows' sums are subtracted, to a tenth
// of what either is.
template <bool REF>
struct SumType {
  using type = float;
};
template <>
struct SumType<true> {
  using type = double;
};
template <bool REF>
using Sum = typename SumType<REF>::type;

// x = z - top and its exponential.  The product of an entry of p = 0 with its x is 0, never 0 * inf.
struct Entry {
  float e, x;
};
template <bool FINE = false>
__device__ __forceinline__ Entry entry_of(float z, float top) {
  const float x = z - top;
  return Entry{exp_of<FINE>(x), fmaxf(x, LOWEST)};  // (a NaN is kept by e)
}
template <bool REF>
__device__ __forceinline__ float gap_of(float e, float z, float y, float shift) {
  return REF && e > 0 ? (z - y) - shift : 0.f;
}
template <bool REF>
__device__ __forceinline__ float grad_of(float z, float y, float top, const RowCoefs &c) {
  const Entry n = entry_of(z, top);
  float u = fmaf(c.slope, n.x, c.base);
  // (finite: a reference's 0 where p is not, or its NaN, is the KL's to tell, and none of a pull of 0)
  if (REF) u = fmaf(c.pull, fminf(gap_of<REF>(n.e, z, y, c.shift), 3e38f), u);
  return n.e * u;
}

__device__ __forceinline__ void report(const LossArgs &a, int64_t row, const RowScalars &o) {
  a.log_probs[row] = o.live ? float(o.log_p) : 0.f;
  a.entropy[row] = o.live ? float(o.entropy) : 0.f;
  if (a.kl) a.kl[row] = o.live ? float(o.kl) : 0.f;
}

__device__ __forceinline__ Coefs coefs_of(const LossArgs &a) {
  return Coefs{read(a.entropy_coef), read(a.kl_coef), (a.upstream ? double(*a.upstream) : 1.0) / read(a.normalizer)};
}

// The action's logit; NaN for an action outside the row, -inf for one that is not legal.
template <typename T>
__device__ __forceinline__ float logit_of(const LossArgs &a, int64_t row, int64_t action) {
  if (action < 0 || action >= a.width) return NAN;
  if (a.mask && !a.mask[row * a.ld_mask + action]) return -INFINITY;
  return to_f32(static_cast<const T *>(a.logits)[row * a.ld_logits + action]);
}

// ---- rows in registers: E entries a lane, G lanes a row, 256 / G rows a block at a time (one from 256 on) -----

// The waves of a SIMD that the registers have to leave room for.
template <typename T, int G, int E, bool REF, int W = Entries<T, E>::WORDS * (REF ? 2 : 1)>
constexpr int ROOM = G == 1024 ? (W <= 16 ? 8 : 4) : W <= 16 ? 6 : W < 32 ? 5 : 4;

// S: the type in which entries are kept (T, or float where rows are shorter than a load).
template <typename T, int G, int E, bool REF, typename S = T>
__global__ __launch_bounds__((G > 256 ? G : 256), (ROOM<S, G, E, REF>)) void rows_kernel(const LossArgs a) {
  constexpr int V = E == 1 ? 1 : VEC<T>, C = E / V, THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  const Coefs coefs = coefs_of(a);
  double value = 0;
  const int in_block = G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : int(threadIdx.x / G);
  const auto row_of = [&](int64_t first) { return min(first + in_block, int64_t(a.rows) - 1); };
  int64_t first = int64_t(blockIdx.x) * ROWS;
  RowInputs next = row_inputs(a, row_of(first));
  // every thread of the block takes every turn: lanes of rows past the end have nothing live
  for (; first < a.rows; first += int64_t(gridDim.x) * ROWS) {
    int lane = threadIdx.x % G;
    asm volatile("" : "+v"(lane));  // (what follows from it alone stays here: 60 masks, else, around the loop)
    const bool in = first + in_block < a.rows;
    const int64_t row = row_of(first);
    RowInputs inputs = next;
    next = row_inputs(a, row_of(first + int64_t(gridDim.x) * ROWS));
    if (!in) inputs.weight = 0;
    const T *logits = static_cast<const T *>(a.logits) + row * a.ld_logits;
    const T *ref = static_cast<const T *>(a.ref_logits) + (REF ? row * a.ld_ref : 0);
    const uint8_t *legal = a.mask ? a.mask + row * a.ld_mask : nullptr;
    Entries<S, E> z;
    Entries<S, REF ? E : V> y;
    float action_logit = 0;
    const bool streams = G >= 512 && a.streams;
    if (inputs.weight != 0) {  // rows without weight are not read
      load_entries<G, C, V>(z.w, logits, legal, lane * V, a.width, streams);
      if constexpr (REF) load_entries<G, C, V>(y.w, ref, legal, lane * V, a.width, streams);
      action_logit = logit_of<T>(a, row, inputs.action);
    } else {
      z.clear();
      if constexpr (REF) y.clear();
    }
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
    z.forget();
    if constexpr (REF) y.forget();
    Sum<REF> s = 0, rs = 0;
    float t = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const Entry n = entry_of<REF>(z[k], q.top);
      s += n.e;
      t = fmaf(n.e, n.x, t);
      if constexpr (REF) rs += exp_of<true>(y[k] - q.ref_top);
    }
    double sums[REF ? 3 : 2];
    sums[0] = s, sums[1] = t;
    if constexpr (REF) sums[2] = rs;
    join<G>(sums, slots.sums, Add{});
    q.s = sums[0], q.t = sums[1], q.ref_s = REF ? sums[REF ? 2 : 0] : 0;
    z.forget();
    if constexpr (REF) y.forget();
    const RowScalars o = row_scalars<REF>(a, inputs, action_logit, q, coefs, [&](float shift) {
      float g = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float e = exp_of<true>(z[k] - q.top);
        g = fmaf(e, gap_of<REF>(e, z[k], y[REF ? k : 0], shift), g);
      }
      double gaps[1] = {g};
      join<G>(gaps, slots.gaps, Add{});
      return gaps[0];
    });
    z.forget();
    if constexpr (REF) y.forget();
    if (!in) continue;  // (all lanes of a group; the reductions are behind)
    if (lane == 0 && a.log_probs) {
      if (o.live) value += o.value;
      report(a, row, o);
    }
    if (a.grad) {
      T *grad = static_cast<T *>(a.grad) + row * int64_t(a.width);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float g[V];
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] = grad_of<REF>(z[c * V + k], y[REF ? c * V + k : 0], q.top, o.c);
        store_entries<V>(grad, g, (c * G + lane) * V, a.width, (c + 1) * G * V <= a.width, streams);
      }
      // The action's own term, by the lane that has just written that entry.
      const int64_t action = inputs.action;
      if (o.live && action >= 0 && action < a.width && action / V % G == lane) {
        const float yr = REF && action_logit > -INFINITY ? to_f32(ref[REF ? action : 0]) : 0.f;
        grad[action] = from_f32<T>(grad_of<REF>(action_logit, yr, q.top, o.c) + o.c.own);
      }
    }
  }
  if (a.log_probs) block_loss(a, value);
}

// ---- passes over a row, or a segment of one, that is read again for each --------------------------------------
//
// each(visit): calls visit(first entry, logits, reference logits) for this thread's vectors.

template <int G, int V, bool REF, typename Each>
__device__ __forceinline__ void row_sums(const Each &each, Slots<G> &slots, RowSums &q) {
  float tops[REF ? 2 : 1];
  tops[0] = tops[REF ? 1 : 0] = -INFINITY;
  each([&](int, const auto &z, const auto &y) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      tops[0] = fmaxf(tops[0], z[k]);
      if constexpr (REF) tops[1] = fmaxf(tops[1], y[k]);
    }
  });
  join<G>(tops, slots.tops, Most{});
  q.top = tops[0] > -INFINITY ? tops[0] : 0.f;
  q.ref_top = REF && tops[REF ? 1 : 0] > -INFINITY ? tops[REF ? 1 : 0] : 0.f;
  double sums[REF ? 3 : 2] = {};
  each([&](int, const auto &z, const auto &y) {
    Sum<REF> s = 0, rs = 0;
    float t = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const Entry n = entry_of<REF>(z[k], q.top);
      s += n.e;
      t = fmaf(n.e, n.x, t);
      if constexpr (REF) rs += exp_of<true>(y[k] - q.ref_top);
    }
    sums[0] += s, sums[1] += t;
    if constexpr (REF) sums[2] += rs;
  });
  join<G>(sums, slots.sums, Add{});
  q.s = sums[0], q.t = sums[1], q.ref_s = REF ? sums[REF ? 2 : 0] : 0;
}

template <int G, int V, typename Each>
__device__ __forceinline__ double gap_sum(const Each &each, Slots<G> &slots, const RowSums &q, float shift) {
  double gaps[1] = {};
  each([&](int, const auto &z, const auto &y) {
    float g = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float e = exp_of<true>(z[k] - q.top);
      g = fmaf(e, gap_of<true>(e, z[k], y[k], shift), g);
    }
    gaps[0] += g;
  });
  join<G>(gaps, slots.gaps, Add{});
  return gaps[0];
}

// The gradient of entries [begin, end) of a row, by `threads` threads.
template <typename T, bool REF, typename Each>
__device__ __forceinline__ void row_grads(const LossArgs &a, T *grad, const T *ref, int64_t action, float action_logit,
                                          float top, const RowScalars &o, const Each &each, int begin, int end,
                                          int threads) {
  constexpr int V = VEC<T>;
  if (o.live) {
    each([&](int i, const auto &z, const auto &y) {
      float g[V];
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = grad_of<REF>(z[k], REF ? y[k] : 0.f, top, o.c);
      store_entries<V>(grad, g, i, a.width, false);
    });
    if (action >= begin && action < end && int(action - begin) / V % threads == int(threadIdx.x)) {
      const float yr = REF && action_logit > -INFINITY ? to_f32(ref[REF ? action : 0]) : 0.f;
      grad[action] = from_f32<T>(grad_of<REF>(action_logit, yr, top, o.c) + o.c.own);
    }
  } else {
    const float zero[V] = {};
    for (int64_t i = begin + int64_t(threadIdx.x) * V; i < end; i += threads * V)
      store_entries<V>(grad, zero, int(i), a.width, false);
  }
}

// ---- rows of any width: a block a row -------------------------------------------------------------------------

template <typename T, bool REF>
__global__ __launch_bounds__(1024, 4) void long_rows_kernel(const LossArgs a) {
  constexpr int V = VEC<T>, G = 1024;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  const Coefs coefs = coefs_of(a);
  double value = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const RowInputs inputs = row_inputs(a, row);
    const int width = inputs.weight != 0 ? a.width : 0;
    const T *logits = static_cast<const T *>(a.logits) + row * a.ld_logits;
    const T *ref = static_cast<const T *>(a.ref_logits) + (REF ? row * a.ld_ref : 0);
    const uint8_t *legal = a.mask ? a.mask + row * a.ld_mask : nullptr;
    const float action_logit = width ? logit_of<T>(a, row, inputs.action) : 0.f;
    const auto each = [&](const auto &visit) {
      for (int64_t i = int64_t(threadIdx.x) * V; i < width; i += G * V) {
        Entries<T, V> z, y;
        load_entries<1, 1, V>(z.w, logits, legal, int(i), width);
        if constexpr (REF) load_entries<1, 1, V>(y.w, ref, legal, int(i), width);
        visit(int(i), z, y);
      }
    };
    RowSums q;
    row_sums<G, V, REF>(each, slots, q);
    const RowScalars o = row_scalars<REF>(a, inputs, action_logit, q, coefs,
                                          [&](float shift) { return gap_sum<G, V>(each, slots, q, shift); });
    if (threadIdx.x == 0 && a.log_probs) {
      if (o.live) value += o.value;
      report(a, row, o);
    }
    if (!a.grad) continue;
    T *grad = static_cast<T *>(a.grad) + row * int64_t(a.width);
    row_grads<T, REF>(a, grad, ref, inputs.action, action_logit, q.top, o, each, 0, a.width, G);
  }
  if (a.log_probs) block_loss(a, value);
}

// ---- a few long rows: a block a segment of a row, the segments joined by every block of the next launch ---------

constexpr int MOST_SPLITS = 64;  // a lane each
constexpr int SPLIT_PARTS = 6;   // top, S, T, the reference's top and S, and the sum of the KL's terms

// The whole row's sums from its segments', scaled from their tops to the row's.
template <bool REF>
__device__ __forceinline__ RowSums joined_sums(const LossArgs &a, const double *parts) {
  const int s = threadIdx.x & 63;
  const bool in = s < a.splits;
  const double *p = parts + SPLIT_PARTS * (in ? s : 0);
  RowSums q;
  const auto part = [&](double top, double sum, float &whole) {  // the segment's factor
    const float mine = in && sum != 0 ? float(top) : -INFINITY;
    whole = lanes_join<64>(mine, Most{});
    whole = whole > -INFINITY ? whole : 0.f;
    return in && sum != 0 ? exp_of(top - double(whole)) : 0.0;
  };
  const double f = part(p[0], p[1], q.top);
  q.s = lanes_join<64>(f != 0 ? f * p[1] : 0.0, Add{});
  q.t = lanes_join<64>(f != 0 ? f * (p[2] + (p[0] - double(q.top)) * p[1]) : 0.0, Add{});
  q.ref_top = 0, q.ref_s = 0;
  if constexpr (REF) {
    const double g = part(p[3], p[4], q.ref_top);
    q.ref_s = lanes_join<64>(g != 0 ? g * p[4] : 0.0, Add{});
  }
  return q;
}

// STEP 0: a segment's sums; 1: its part of the exact KL; 2: its gradient, and the row's numbers.
template <typename T, bool REF, int STEP>
__global__ __launch_bounds__(256) void split_rows_kernel(const LossArgs a) {
  constexpr int V = VEC<T>, G = 256;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  const int row = blockIdx.x / a.splits, segment = blockIdx.x % a.splits;
  const RowInputs inputs = row_inputs(a, row);
  const int begin = segment * a.segment, end = min(begin + a.segment, a.width);
  const T *logits = static_cast<const T *>(a.logits) + row * a.ld_logits;
  const T *ref = static_cast<const T *>(a.ref_logits) + (REF ? row * a.ld_ref : 0);
  const uint8_t *legal = a.mask ? a.mask + row * a.ld_mask : nullptr;
  const bool counts = inputs.weight != 0;
  double *parts = a.parts + int64_t(row) * a.splits * SPLIT_PARTS, *mine = parts + segment * SPLIT_PARTS;
  const auto each = [&](const auto &visit) {
    if (!counts) return;
    for (int i = begin + int(threadIdx.x) * V; i < end; i += G * V) {
      Entries<T, V> z, y;
      load_entries<1, 1, V>(z.w, logits, legal, i, a.width);
      if constexpr (REF) load_entries<1, 1, V>(y.w, ref, legal, i, a.width);
      visit(i, z, y);
    }
  };
  if constexpr (STEP == 0) {
    RowSums q;
    row_sums<G, V, REF>(each, slots, q);
    if (threadIdx.x == 0) {
      mine[0] = q.top, mine[1] = q.s, mine[2] = q.t;
      if (REF) mine[3] = q.ref_top, mine[4] = q.ref_s;
    }
  } else {
    const RowSums q = joined_sums<REF>(a, parts);
    if constexpr (STEP == 1) {
      const double g = gap_sum<G, V>(each, slots, q, float(shift_of(q, log_of(q.s))));
      if (threadIdx.x == 0) mine[5] = g;
    } else {
      const float action_logit = counts ? logit_of<T>(a, row, inputs.action) : 0.f;
      const RowScalars o = row_scalars<REF>(a, inputs, action_logit, q, coefs_of(a), [&](float) {
        const int s = threadIdx.x & 63;
        return lanes_join<64>(s < a.splits ? parts[SPLIT_PARTS * s + 5] : 0.0, Add{});
      });
      if (segment == 0 && threadIdx.x == 0 && a.log_probs) {
        a.partials[row] = o.live ? o.value : 0.0;
        report(a, row, o);
      }
      if (!a.grad) return;
      T *grad = static_cast<T *>(a.grad) + int64_t(row) * a.width;
      row_grads<T, REF>(a, grad, ref, inputs.action, action_logit, q.top, o, each, begin, end, G);
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------

struct Launch {
  void (*kernel)(LossArgs);
  int rows, threads;  // rows a block takes at a time
};

// Segments of a row: 1 (none) unless rows are long and leave most CUs without one.  A pass over bf16 rows with
// the backward that has nothing to do, as a block a row and as segments, us: 9 x 50001 beside a reference's
// 41 and 23, alone 20 and 13.5; 64 x 50001 beside one 43 and 35; but 64 x 30000 13.8 and 15.4, 9 x 9000
// 10.6 and 14.1, 128 x 50001 22.6 and 25.
int splits_of(const cg_policy_loss &p) {
  if (p.rows > 64 || p.rows == 0 || p.width <= 32768) return 1;
  const int wanted = (512 + p.rows - 1) / p.rows, most = p.width / 2048;
  const int splits = wanted < most ? wanted : most;
  return splits < MOST_SPLITS ? splits : MOST_SPLITS;
}

size_t parts_bytes(const cg_policy_loss &p) {
  const int splits = splits_of(p);
  return splits > 1 ? size_t(p.rows) * splits * SPLIT_PARTS * sizeof(double) : 0;
}

template <typename T, bool REF>
void launch_splits(LossArgs a, const cg_policy_loss &p, hipStream_t stream) {
  const int splits = splits_of(p);
  a.segment = ((p.width + splits - 1) / splits + VEC<T> - 1) / VEC<T> * VEC<T>;
  a.splits = (p.width + a.segment - 1) / a.segment;
  const int blocks = p.rows * a.splits;
  split_rows_kernel<T, REF, 0><<<blocks, 256, 0, stream>>>(a);
  CG_LAUNCHED();
  if constexpr (REF) {
    split_rows_kernel<T, REF, 1><<<blocks, 256, 0, stream>>>(a);
    CG_LAUNCHED();
  }
  split_rows_kernel<T, REF, 2><<<blocks, 256, 0, stream>>>(a);
  CG_LAUNCHED();
}

template <typename T, int G, int E, bool REF, typename S = T>
Launch launch_as() {
  return {rows_kernel<T, G, E, REF, S>, G > 256 ? 1 : 256 / G, G > 256 ? G : 256};
}

// Lanes and entries a lane by width: few lanes a row keep the row's scalars, which each of them forms, few; up to
// 32 entries (64 of 16 bits where rows are wide) leave room for the waves that hide the loads.  us of a pass:
//   257 to 1024 entries, half as many lanes from 8193 rows on: 16384 x 512 fp32 15.0 and 16.4, bf16 13.8 and 15.2,
//   32768 x 1024 bf16 34.5 and 42.6, but 1024 x 512 bf16 6.4 and 5.8, with a reference 10.0 and 7.9.  Between 4096
//   and 8192 rows 512 entries are even, 1024 would gain up to 2 of 16.
//   A wave a row up to 2048, a block a row beyond: 4096 x 2048 bf16 14.8 and 20.1, fp32 16.5 and 20.8; 4096 x 4096
//   fp32 36 and 29, with a reference 174 and 51, but bf16 20.9 and 25.5, with a reference 47.0 and 49.5; 256 x 4096
//   bf16 8.3 and 6.3.
template <typename T, bool REF>
Launch launch_of(int width, int rows) {
  if (width < VEC<T>) return launch_as<T, 8, 1, REF, float>();
  if (width <= 32) return launch_as<T, 4, 8, REF>();
  if (width <= 64) return launch_as<T, 4, 16, REF>();
  if (width <= 96) return launch_as<T, 4, 24, REF>();
  if (width <= 128) return launch_as<T, 4, 32, REF>();
  if (width <= 192) return launch_as<T, 8, 24, REF>();
  if (width <= 256) return launch_as<T, 8, 32, REF>();
  if (width <= 512) return rows <= 8192 ? launch_as<T, 32, 16, REF>() : launch_as<T, 16, 32, REF>();
  if (width <= 1024) return rows <= 8192 ? launch_as<T, 64, 16, REF>() : launch_as<T, 32, 32, REF>();
  if (width <= 2048) return launch_as<T, 64, 32, REF>();
  if (width <= 4096) return launch_as<T, 256, 16, REF>();
  if (width <= 8192) return launch_as<T, 256, 32, REF>();
  if (width <= 16384) return launch_as<T, 512, 32, REF>();
  if constexpr (sizeof(T) == 2) {
    if (width <= 32768) return launch_as<T, 512, 64, REF>();
    if (width <= 65536) return launch_as<T, 1024, 64, REF>();
  } else if (width <= 32768) {
    return launch_as<T, 1024, 32, REF>();
  }
  return {long_rows_kernel<T, REF>, 1, 1024};
}

template <typename T>
Launch launch_of(const cg_policy_loss &p, bool ref) {
  return ref ? launch_of<T, true>(p.width, p.rows) : launch_of<T, false>(p.width, p.rows);
}

Launch launch_of(const cg_policy_loss &p) {
  const bool ref = p.reference_logits != nullptr;
  return p.dtype == CG_F32    ? launch_of<float>(p, ref)
         : p.dtype == CG_BF16 ? launch_of<bf16>(p, ref)
                              : launch_of<f16>(p, ref);
}

// Returns the number of partial sums of the loss that are written (by one block for all rows: the loss itself).
int launch_rows(const LossArgs &a, const cg_policy_loss &p, hipStream_t stream) {
  if (splits_of(p) > 1) {
    const auto of = [&](auto type) {
      using T = decltype(type);
      if (p.reference_logits)
        launch_splits<T, true>(a, p, stream);
      else
        launch_splits<T, false>(a, p, stream);
    };
    if (p.dtype == CG_F32)
      of(float{});
    else if (p.dtype == CG_BF16)
      of(bf16{});
    else
      of(f16{});
    return p.rows;
  }
  const Launch l = launch_of(p);
  const int64_t blocks = (int64_t(p.rows) + l.rows - 1) / l.rows;
  // Blocks of 512 lanes and more fit a CU twice at most: as many as fit walk the rows, each row's inputs loaded
  // a turn ahead (4096 x 32768: 131 us with 2048 blocks, 128 with 512).
  const int most = l.threads >= 512 ? 512 : MAX_BLOCKS;
  const int grid = int(blocks < most ? blocks : most);
  l.kernel<<<grid, l.threads, 0, stream>>>(a);
  CG_LAUNCHED();
  return grid;
}

LossArgs args_of(const cg_policy_loss *loss) {
  CG_REQUIRE(loss != nullptr, CG_ERR_INVALID, "loss is NULL");
  const cg_policy_loss &p = *loss;
  dtype_size(p.dtype);
  CG_REQUIRE(p.rows >= 0 && p.width > 0, CG_ERR_INVALID, "rows must be non-negative, width positive");
  CG_REQUIRE(p.width <= 1 << 30, CG_ERR_UNSUPPORTED, "policy loss: rows wider than 2^30");
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
  a.streams = int64_t(p.rows) * p.width >= STREAM_BYTES / (2 * dtype_size(p.dtype));
  a.normalizer = scalar(p.normalizer), a.entropy_coef = scalar(p.entropy_coef), a.kl_coef = scalar(p.kl_coef);
  return a;
}

}  // namespace
}  // namespace cg

using namespace cg;

extern "C" {

size_t cg_policy_loss_workspace_size(const cg_policy_loss *loss) {
  return loss ? MAX_BLOCKS * sizeof(double) + parts_bytes(*loss) : 0;
}

int cg_policy_loss_forward(const cg_policy_loss *loss, float *value, float *log_probs, float *entropy, float *kl,
                           void *grad, void *workspace, size_t workspace_size, void *stream) {
  return guarded([&] {
    LossArgs a = args_of(loss);
    CG_REQUIRE(value && workspace, CG_ERR_INVALID, "value and workspace are required");
    CG_REQUIRE(workspace_size >= cg_policy_loss_workspace_size(loss), CG_ERR_INVALID, "workspace too small");
    CG_REQUIRE(a.rows == 0 || (log_probs && entropy), CG_ERR_INVALID, "log_probs and entropy are required");
    CG_REQUIRE(a.rows == 0 || !kl == !(a.ref || a.ref_logits), CG_ERR_INVALID, "kl goes with a reference");
    a.partials = static_cast<double *>(workspace);
    a.parts = a.partials + MAX_BLOCKS;
    a.loss = value;
    int sums = 0;
    if (a.rows > 0) {
      a.log_probs = log_probs, a.entropy = entropy, a.kl = kl, a.grad = grad;
      sums = launch_rows(a, *loss, as_stream(stream));
    }
    if (sums != 1 || splits_of(*loss) > 1) {
      loss_kernel<LossArgs><<<1, 256, 0, as_stream(stream)>>>(a, sums);
      CG_LAUNCHED();
    }
  });
}

size_t cg_policy_loss_backward_workspace_size(const cg_policy_loss *loss) { return loss ? parts_bytes(*loss) : 0; }

int cg_policy_loss_backward(const cg_policy_loss *loss, const float *upstream, int32_t written, void *grad,
                            void *workspace, size_t workspace_size, void *stream) {
  return guarded([&] {
    LossArgs a = args_of(loss);
    CG_REQUIRE(upstream, CG_ERR_INVALID, "upstream is required");
    if (a.rows == 0) return;
    CG_REQUIRE(grad, CG_ERR_INVALID, "grad is required");
    const size_t need = cg_policy_loss_backward_workspace_size(loss);
    CG_REQUIRE(need == 0 || (workspace && workspace_size >= need), CG_ERR_INVALID, "workspace too small");
    a.parts = static_cast<double *>(workspace);
    a.grad = grad, a.upstream = upstream, a.written = written;
    launch_rows(a, *loss, as_stream(stream));
  });
}

}  // extern "C"
