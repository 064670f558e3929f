// The distillation loss towards a record of another policy's top entries (gfx950): forward and gradient over rows
// of logits in one pass.
//
// A row's legal entries are those its mask keeps and whose logit is above -inf; p = softmax(z / T) over them.  The
// record R holds entries k with the logs of the teacher's q_k, and may hold the log of q_r, what the teacher has
// outside.  With p_r p's mass outside R and Q the sum of q:
//   KL = sum_R q_k (log q_k - log p_k) + q_r (log q_r - log p_r),
//   dKL/dz_j = (Q p_j - q_j) / T in R,  p_j (Q - q_r / p_r) / T outside;
// without q_r, q is made to sum to 1 over R and the second term is not there.  The loss is the sum of w KL over `normalizer`.
//
// Entries in R are set aside: a bit each in LDS, by which the lanes that hold the row leave them out, and a lane
// each for their terms, in fp64.  So p_r is a sum of its own, measured from its own largest entry, and not 1 minus what
// R has; and the gradient outside R is e^((z - m_r) / T) times one number a row, whose two terms nearly cancel where the policies
// agree and are therefore subtracted in fp64.
//
// Every logit (mask byte) is read once and every gradient written once; a row stays in registers between its maximum,
// its sum and its gradient.  Wide rows are bound by VALU instructions beside HBM (29.5 an entry of 16 bits, two of
// them exponentials; bf16 4096 x 32768 140 us, its bytes 107), narrow ones by the record's terms and the row's
// scalars.  The forward writes the gradient for an upstream of 1; a backward with another one forms it again from the
// inputs, so it is rounded once whatever the scale.
#include "rows.h"

namespace cg {
namespace {

constexpr int MAX_WIDTH = 1 << 18;
constexpr int MAX_TOP = 256;
// Logits and gradient of this many bytes go past the caches (256 MB of Infinity Cache); below, whatever made the logits
// or takes the gradient may find them there.  us kept and past them: fp32 2048 x 32768 163 and 139, bf16 4096 x 32768, whose
// time is arithmetic, even.
constexpr int64_t STREAM_BYTES = 512 << 20;

struct DistillArgs {
  const void *logits;
  const uint8_t *mask;
  const int64_t *indices;  // [rows, k]
  const float *top, *rest;  // [rows, k], and [rows] or NULL
  const float *weights;
  int64_t ld_logits, ld_mask;
  int32_t rows, width, k;
  double inverse;     // 1 / T
  float fast, slow;   // log2(e) / T rounded down, and the rest of it: both above 0, so that -inf stays -inf
  float scale;        // log2(e) / T to the nearest
  Scalar normalizer;
  float *kl;   // NULL in a backward call
  void *grad;  // NULL: none
  double *partials;
  float *loss;
  const float *upstream;  // of a backward call
  int32_t written;        // the gradient for an upstream of 1 is in place
  int32_t streams;        // the logits and their gradient go past the caches (rows of 512 lanes and more)
};

// e^((z - from) / T) for z <= from (-inf: 0).  The scale's second part keeps its rounding, which is the same for all
// entries, out of their sum; what the rounding of the product leaves differs from one to the next.
__device__ __forceinline__ float exp_from(const DistillArgs &a, float z, float from) {
  const float d = z - from;
  return __builtin_amdgcn_exp2f(fmaf(d, a.fast, d * a.slow));
}

// For a gradient of 16 bits, whose own rounding is 2^-8 or 2^-11 of it: the scale's rounding, |x| 2^-24 of the exponential
// (x = (z - from) / T, 104 at most before it is 0), is a 79th of fp16's at most.  One instruction less of five:
// 4096 x 32768 bf16 143 and 140 us.  Values and sums have exp_from in every type.
__device__ __forceinline__ float exp_near(const DistillArgs &a, float z, float from) {
  return __builtin_amdgcn_exp2f((z - from) * a.scale);
}

// ---- the record's entries in a row -------------------------------------------------------------------------

// Bit i % 32 of word i / 32 is set for entries in R.  A word more than the row has, so that two side by side can be read.
template <int CAPACITY>
struct Bits {
  static constexpr int WORDS = (CAPACITY + 31) / 32 + 1;
  uint32_t w[WORDS];
  // Bits i to i + 31, i a multiple of nothing.
  __device__ __forceinline__ uint32_t from(int i) const {
    return __builtin_amdgcn_alignbit(w[(i >> 5) + 1], w[i >> 5], i & 31);
  }
};

// This lane's entries of R.  A group of 64 lanes or more loads them once, beside the row; in narrower ones, whose rows
// have few words to wait for, they would take more registers than the row does.
template <int G, typename T>
struct Record {
  static constexpr int N = G < 64 ? 0 : G < MAX_TOP ? MAX_TOP / G : 1;
  const DistillArgs &a;
  const int64_t *indices;
  const float *top;
  const T *logits;
  const uint8_t *legal;
  int lane, index[N > 0 ? N : 1];  // -1: none; -2: not of the row
  float log_q[N > 0 ? N : 1], z[N > 0 ? N : 1];

  __device__ __forceinline__ Record(const DistillArgs &a, int64_t r, int lane, const T *logits, const uint8_t *legal, bool counts)
      : a(a), indices(a.indices + r * a.k), top(a.top + r * a.k), logits(logits), legal(legal), lane(lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = lane + i * G;
      index[i] = -1, log_q[i] = z[i] = -INFINITY;
      if (!counts || k >= a.k) continue;
      index[i] = in_row(indices[k]);
      log_q[i] = top[k];
    }
  }
  __device__ __forceinline__ int in_row(int64_t i) const { return i >= 0 && i < a.width ? int(i) : i == -1 ? -1 : -2; }
  // The entry's logit, -inf where it is not legal.
  __device__ __forceinline__ float logit(int i) const { return !legal || legal[i] ? to_f32(logits[i]) : -INFINITY; }
  __device__ __forceinline__ void load_logits() {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (index[i] >= 0) z[i] = logit(index[i]);
  }
  // visit(index, log q, logit) for those in the row.
  template <typename Visit>
  __device__ __forceinline__ void each(const Visit &visit) const {
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (index[i] >= 0) visit(index[i], log_q[i], z[i]);
    } else {
      for (int k = lane; k < a.k; k += G) {
        const int i = in_row(indices[k]);
        if (i >= 0) visit(i, top[k], logit(i));
      }
    }
  }
  // Marks R, of a row that counts.  Returns whether this lane's indices are in the row, and there once.
  template <typename B>
  __device__ __forceinline__ bool mark(B &bits, bool counts) const {
    const int words = min((a.width >> 5) + 2, B::WORDS);  // (of vectors that begin before the row's end, and one more)
    for (int i = lane; i < words; i += G) bits.w[i] = 0;
    group_sync<G>();
    bool good = true;
    const auto set = [&](int i) {
      if (i == -2) good = false;
      if (i < 0) return;
      const uint32_t bit = 1u << (i & 31);
      if (atomicOr(&bits.w[i >> 5], bit) & bit) good = false;
    };
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) set(index[i]);
    } else if (counts) {
      for (int k = lane; k < a.k; k += G) set(in_row(indices[k]));
    }
    group_sync<G>();
    return good;
  }
};

// ---- a row's scalars -----------------------------------------------------------------------------------------

// Sums over R: e^((z - m) / T), q, q log q and q (z - m) / T.  Without q_r, q is measured from its largest.
struct TopSums {
  double s, q, own, cross;
};

struct RowScalars {
  double kl, value;
  float outer;         // the gradient's factor of e outside R
  double inner, pull;  // in R: inner e^((z - m) / T) - pull q
  bool live;
};

// top, rest_top: the row's largest entry, and the largest outside R; rest: the sum outside, from rest_top.
__device__ __forceinline__ RowScalars row_scalars(const DistillArgs &a, int64_t r, float weight, float top, float rest_top,
                                                  double rest, const TopSums &t, bool good) {
  RowScalars o;
  const double gap = rest > 0 ? (double(rest_top) - double(top)) * a.inverse : 0.0;
  const double lower = rest > 0 ? exp_of(gap) : 0.0;
  double s = t.s + (rest > 0 ? rest * lower : rest);  // (rest: NaN stays)
  // s is 0 where nothing is legal.  (Without q_r the largest q counts as 1: they sum to 0 where the record has nothing, and
  // the row has no term whatever its logits.)
  o.live = weight != 0 && s != 0 && (a.rest || t.q != 0 || !good);
  if (!good) s = NAN;
  const double log_s = log_of(s);
  double mass = t.q, outer = 0;
  if (a.rest) {
    const double log_q = weight != 0 ? a.rest[r] : -INFINITY, q = exp_of(log_q);
    mass += q;
    o.kl = t.own - t.cross + t.q * log_s;
    if (!(q <= 0)) {
      const double log_p = rest > 0 ? gap + log_of(rest) - log_s : -INFINITY;
      o.kl += q * (log_q - log_p);
      if (rest > 0) outer = q * reciprocal(rest);
    }
    o.pull = 1;
  } else {
    const double inv = t.q > 0 ? reciprocal(t.q) : 0;
    o.kl = t.q > 0 ? (t.own - t.cross) * inv - log_of(t.q) + log_s : NAN;
    mass = t.q > 0 ? 1 : NAN;
    o.pull = inv;
  }
  const double f = double(weight) * (a.upstream ? double(*a.upstream) : 1.0) / read(a.normalizer) * a.inverse;
  o.inner = f * mass * reciprocal(s);
  o.pull *= f;
  o.outer = float(o.inner * lower - f * outer);
  o.value = double(weight) * o.kl;
  return o;
}

template <int G>
struct Slots {
  static constexpr int W = G > 64 ? G / 64 : 1;
  float tops[3 * W];
  double sums[6 * W];
};

// From a row's entries outside R to its numbers and its gradient: what every kernel does with a row.
// each(visit): visit(first entry, entries, inside) for this lane's vectors, those in R as -inf.  pass(): between passes.
template <int G, int V, typename T, typename Each, typename Pass>
__device__ __forceinline__ void distill_row(const DistillArgs &a, int64_t r, int lane, float weight, bool good,
                                            const Record<G, T> &record, Slots<G> &slots, bool in, const Each &each, const Pass &pass, double &value) {
  float tops[3] = {-INFINITY, -INFINITY, -INFINITY};  // of z outside R, in it, and of log q
  if (weight != 0) {
    each([&](int, const auto &z, bool) {
#pragma unroll
      for (int k = 0; k < V; ++k) tops[0] = fmaxf(tops[0], z(k));
    });
    record.each([&](int, float log_q, float z) {
      tops[1] = fmaxf(tops[1], z);
      tops[2] = fmaxf(tops[2], log_q);
    });
  }
  join<G>(tops, slots.tops, Most{});
  pass();
  const float rest_top = tops[0] > -INFINITY ? tops[0] : 0.f;
  const float most = fmaxf(tops[0], tops[1]), top = most > -INFINITY ? most : 0.f;
  // Without q_r, only the differences of the log q count.
  const float base = !a.rest && tops[2] > -INFINITY ? tops[2] : 0.f;
  double sums[6] = {};  // the rest, then TopSums, then whether the record is in order
  if (weight != 0) {
    each([&](int, const auto &z, bool) {
      float s = 0;  // (of a vector's 4 or 8, each off by (3 |x| + 4) 2^-24: 8 roundings more, then float64)
#pragma unroll
      for (int k = 0; k < V; ++k) s += exp_from(a, z(k), rest_top);
      sums[0] += s;
    });
    record.each([&](int, float log_q, float z) {
      const double x = (double(z) - double(top)) * a.inverse, l = double(log_q) - double(base), q = exp_of(l);
      sums[1] += exp_of(x);
      sums[2] += q;
      if (!(q <= 0)) sums[3] += q * l, sums[4] += q * x;
    });
  }
  sums[5] = good ? 0 : 1;
  join<G>(sums, slots.sums, Add{});
  pass();
  const RowScalars o = row_scalars(a, r, weight, top, rest_top, sums[0], TopSums{sums[1], sums[2], sums[3], sums[4]},
                                   sums[5] == 0);
  if (in && lane == 0 && a.kl) {
    if (o.live) value += o.value;
    a.kl[r] = o.live ? float(o.kl) : 0.f;
  }
  if (!a.grad) return;
  T *grad = static_cast<T *>(a.grad) + r * int64_t(a.width);
  if (in && o.live) {
    each([&](int i, const auto &z, bool inside) {
      float g[V];
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = o.outer * (sizeof(T) == 2 ? exp_near(a, z(k), rest_top) : exp_from(a, z(k), rest_top));
      store_entries<V>(grad, g, i, a.width, inside, G >= 512 && a.streams);
    });
  } else if (in) {  // (their logits may be NaN: no product with them is 0)
    const float zeros[V] = {};
    each([&](int i, const auto &, bool inside) { store_entries<V>(grad, zeros, i, a.width, inside, G >= 512 && a.streams); });
  }
  group_sync<G>();  // (the zeros just written at R's entries come first)
  if (in && o.live) {
    record.each([&](int i, float log_q, float z) {
      if (z == -INFINITY) return;
      const double x = (double(z) - double(top)) * a.inverse;
      grad[i] = from_f32<T>(float(o.inner * exp_of(x) - o.pull * exp_of(double(log_q) - double(base))));
    });
  }
}

// ---- rows in registers: E entries a lane, G lanes a row, 256 / G rows a block (one from 256 on) -----------------
//
// A block takes its rows and ends: in a loop over rows the compiler keeps what is the same for all of them in registers,
// which the row needs (bf16 4096 x 32768, 512 blocks in a loop: 311 us).

// S: the type in which entries are kept (T, or float where rows are shorter than a load).
template <typename T, int G, int E, typename S = T>
__global__ __launch_bounds__((G > 256 ? G : 256), 4) void rows_kernel(const DistillArgs a) {
  constexpr int V = E == 1 ? 1 : VEC<T>, C = E / V, THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  __shared__ Bits<G * E> bits[ROWS];
  double value = 0;
  const int in_block = threadIdx.x / G, lane = threadIdx.x % G;
  const int64_t first = int64_t(blockIdx.x) * ROWS + in_block;
  const bool in = first < a.rows;  // (lanes of rows past the end have nothing live)
  const int64_t r = in ? first : int64_t(a.rows) - 1;
  const float weight = in ? a.weights ? a.weights[r] : 1.f : 0.f;
  const T *logits = static_cast<const T *>(a.logits) + r * a.ld_logits;
  const uint8_t *legal = a.mask ? a.mask + r * a.ld_mask : nullptr;
  Record<G, T> record(a, r, lane, logits, legal, weight != 0);
  Entries<S, E> z;
  bool good = true;
  if (weight != 0) {  // rows without weight are not read
    load_entries<G, C, V>(z.w, logits, legal, lane * V, a.width, G >= 512 && a.streams);
  } else {
    z.clear();
  }
  // (groups of a wave go through their barriers together, weight or not)
  record.load_logits();
  if (weight != 0 || G <= 64) good = record.mark(bits[in_block], weight != 0);
  if (weight != 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = V == 1 ? lane : min((c * G + lane) * V, a.width - V);
      const uint32_t set = at < a.width ? bits[in_block].from(at) & ((1u << V) - 1) : 0;
      if (set == 0) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const uint32_t part = Entries<S, E>::PER == 1 ? ~0u : k % 2 ? 0xffff0000u : 0xffffu;
        uint32_t &w = z.w[(c * V + k) / Entries<S, E>::PER];
        if (set >> k & 1) w = (w & ~part) | (NEGATIVE_INFINITY<S> & part);
      }
    }
  }
  const auto each = [&](const auto &visit) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      visit((c * G + lane) * V, [&](int k) { return z[c * V + k]; }, (c + 1) * G * V <= a.width);
  };
  distill_row<G, V>(a, r, lane, weight, good, record, slots, in, each, [&] { z.forget(); }, value);
  if (a.kl) block_loss(a, value);
}

// ---- rows of any width, read again for each pass: a block a row ---------------------------------------------------

template <typename T>
__global__ __launch_bounds__(1024) void long_rows_kernel(const DistillArgs a) {
  constexpr int V = VEC<T>, G = 1024;
  if (done(a)) return;
  __shared__ Slots<G> slots;
  __shared__ Bits<MAX_WIDTH> bits;
  double value = 0;
  const int lane = threadIdx.x;
  const int64_t r = blockIdx.x;
  const float weight = a.weights ? a.weights[r] : 1.f;
  const T *logits = static_cast<const T *>(a.logits) + r * a.ld_logits;
  const uint8_t *legal = a.mask ? a.mask + r * a.ld_mask : nullptr;
  Record<G, T> record(a, r, lane, logits, legal, weight != 0);
  record.load_logits();
  const bool good = weight != 0 ? record.mark(bits, true) : true;
  const auto each = [&](const auto &visit) {
    for (int i = lane * V; i < a.width; i += G * V) {
      Entries<T, V> z;
      z.clear();
      uint32_t set = 0;
      if (weight != 0) {
        load_entries<1, 1, V>(z.w, logits, legal, i, a.width);
        set = bits.from(min(i, a.width - V));
      }
      visit(i, [&](int k) { return set >> k & 1 ? -INFINITY : z[k]; }, false);
    }
  };
  distill_row<G, V>(a, r, lane, weight, good, record, slots, true, each, [] {}, value);
  if (a.kl) block_loss(a, value);
}

// ---- host side ---------------------------------------------------------------------------------------------------

struct Launch {
  void (*kernel)(DistillArgs);
  int rows, threads;  // rows a block takes
};

template <typename T, int G, int E, typename S = T>
Launch launch_as() {
  return {rows_kernel<T, G, E, S>, G > 256 ? 1 : 256 / G, G > 256 ? G : 256};
}

// The fewest lanes that hold a row: more have less to do each in the row's joins and its record, and rows wait for both.
// us of forward and backward as chosen and with the next more lanes, k 16 and k 32:
//   65536 x 32 bf16  27  40 and  41  48     16384 x 2048 bf16  58  59 and 156 (k 32)     2048 x 16384 fp32 65 and 118
//   65536 x 128 bf16 44  51 and  73  74      4096 x 8192 bf16      55 and  85            1024 x 32768 bf16 47 and  83
//   65536 x 512 bf16 81  82 and 125 125      2048 x 16384 bf16     53 and  72             512 x 65536 bf16 54 and  60
// fp16, k 16: 26 and 38, 40 and 73, 74 and 153, 52 and 141; 4096 x 8192 50 and 82, 2048 x 16384 50 and 68, 1024 x 32768
// 44 and 79, 512 x 65536 51 and 59.
// (Records of nearly all of a narrow row would have more: 131072 x 32 fp32, k 32, 193 and 79.)
template <typename T>
Launch launch_of(int width) {
  if (width < VEC<T>) return launch_as<T, 8, 1, float>();
  if (width <= 32) return launch_as<T, 4, 8>();
  if (width <= 128) return launch_as<T, 16, 8>();
  if (width <= 512) return launch_as<T, 32, 16>();
  if (width <= 2048) return launch_as<T, 64, 32>();
  if (width <= 8192) return launch_as<T, 256, 32>();
  if (width <= 16384) return launch_as<T, 512, 32>();
  if constexpr (sizeof(T) == 2) {
    if (width <= 32768) return launch_as<T, 512, 64>();
    if (width <= 65536) return launch_as<T, 1024, 64>();
  } else if (width <= 32768) {
    return launch_as<T, 1024, 32>();
  }
  return {long_rows_kernel<T>, 1, 1024};
}

Launch launch_of(const cg_policy_rows &p) {
  return p.dtype == CG_F32 ? launch_of<float>(p.width) : p.dtype == CG_BF16 ? launch_of<bf16>(p.width) : launch_of<f16>(p.width);
}

// Each block's sum of the loss is a partial sum of it (one block's the loss itself).
int64_t blocks_of(const cg_policy_rows &p) {
  const Launch l = launch_of(p);
  return (int64_t(p.rows) + l.rows - 1) / l.rows;
}

void launch_rows(const DistillArgs &a, const cg_policy_rows &p, hipStream_t stream) {
  const Launch l = launch_of(p);
  const int64_t blocks = blocks_of(p);
  CG_REQUIRE(blocks * l.threads < int64_t(1) << 32, CG_ERR_UNSUPPORTED, "more rows than a launch has threads for");
  l.kernel<<<unsigned(blocks), l.threads, 0, stream>>>(a);
  CG_LAUNCHED();
}

DistillArgs args_of(const cg_distill_loss *loss) {
  CG_REQUIRE(loss != nullptr, CG_ERR_INVALID, "loss is NULL");
  const cg_distill_loss &p = *loss;
  const cg_policy_rows &q = p.rows;
  dtype_size(q.dtype);
  CG_REQUIRE(q.rows >= 0 && q.width > 0, CG_ERR_INVALID, "rows must be non-negative, width positive");
  CG_REQUIRE(q.width <= MAX_WIDTH, CG_ERR_UNSUPPORTED, "distill_loss: rows wider than 2^18");
  CG_REQUIRE(p.k > 0 && p.k <= MAX_TOP, CG_ERR_INVALID, "k must be from 1 to 256");
  CG_REQUIRE(p.temperature >= 1e-30 && p.temperature <= 1e30, CG_ERR_INVALID, "temperature must be from 1e-30 to 1e30");
  CG_REQUIRE(q.rows == 0 || (q.logits && p.indices && p.log_probs), CG_ERR_INVALID,
             "logits, indices and log_probs are required");
  CG_REQUIRE(q.ld_logits >= 0 && q.ld_mask >= 0, CG_ERR_INVALID, "row strides must be non-negative");
  DistillArgs a{};
  a.logits = q.logits, a.mask = q.mask, a.indices = p.indices, a.top = p.log_probs, a.rest = p.log_rest;
  a.weights = p.weights;
  a.ld_logits = q.ld_logits, a.ld_mask = q.ld_mask;
  a.rows = q.rows, a.width = q.width, a.k = p.k;
  a.inverse = 1 / p.temperature;
  const double c = 1.44269504088896340736 / p.temperature;
  a.fast = float(c);
  if (double(a.fast) >= c) a.fast = nextafterf(a.fast, 0.f);
  a.slow = float(c - double(a.fast));
  a.scale = float(c);
  a.normalizer = scalar(p.normalizer);
  a.streams = int64_t(q.rows) * q.width >= STREAM_BYTES / (2 * dtype_size(q.dtype));
  return a;
}

}  // namespace
}  // namespace cg

using namespace cg;

extern "C" {

size_t cg_distill_loss_workspace_size(const cg_distill_loss *loss) {
  return loss && loss->rows.rows > 0 && loss->rows.width > 0 ? blocks_of(loss->rows) * sizeof(double) : sizeof(double);
}

int cg_distill_loss_forward(const cg_distill_loss *loss, float *value, float *kl, void *grad, void *workspace,
                            size_t workspace_size, void *stream) {
  return guarded([&] {
    DistillArgs a = args_of(loss);
    CG_REQUIRE(value && workspace, CG_ERR_INVALID, "value and workspace are required");
    CG_REQUIRE(workspace_size >= cg_distill_loss_workspace_size(loss), CG_ERR_INVALID, "workspace too small");
    CG_REQUIRE(a.rows == 0 || kl, CG_ERR_INVALID, "kl is required");
    a.partials = static_cast<double *>(workspace);
    a.loss = value, a.kl = kl, a.grad = grad;
    const int64_t sums = a.rows > 0 ? blocks_of(loss->rows) : 0;
    if (sums > 0) launch_rows(a, loss->rows, as_stream(stream));
    if (sums != 1) {
      // (us of 256 lanes a load at a time, and of these: 4096 sums 6.3 and 4.8, 32768 33 and 6.4, 262144 355 and 45)
      loss_kernel<DistillArgs, 1024><<<1, 1024, 0, as_stream(stream)>>>(a, int(sums));
      CG_LAUNCHED();
    }
  });
}

int cg_distill_loss_backward(const cg_distill_loss *loss, const float *upstream, int32_t written, void *grad,
                             void *stream) {
  return guarded([&] {
    DistillArgs a = args_of(loss);
    CG_REQUIRE(upstream, CG_ERR_INVALID, "upstream is required");
    if (a.rows == 0) return;
    CG_REQUIRE(grad, CG_ERR_INVALID, "grad is required");
    a.grad = grad, a.upstream = upstream, a.written = written;
    launch_rows(a, loss->rows, as_stream(stream));
  });
}

}  // extern "C"
