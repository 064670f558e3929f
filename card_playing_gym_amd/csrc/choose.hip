// Answers of a policy straight from its logits (gfx950): sampling under a temperature, top-k, top-p and
// min-p from given uniforms, and the record of a row's top entries that a distillation loss learns from.
//
// A row's legal entries are those its mask keeps and whose logit is above -inf.  With m the largest,
// d = (z - m) / T and w = e^d; their order puts larger logits first and, of equal ones, the lower index.
//   sampling: of the order's first k (their weights sum to S) those before which less than top_p S is summed
//     up, of these those of w >= min_p, the first always; S' is the sum of what is kept, the action the
//     first entry of the order whose running sum exceeds u S', its log-probability d - log S'.
//   record: the first k of the order with d - log S over the whole row, and the log of the others' share.
//
// An action is decided at borders between running sums, so it must not depend on the order or the rounding of
// additions.  A weight is an integer, 2^scale e^d to the nearest from a polynomial within 2^-44 of e^d, and sums of a
// row are exact 64-bit integers (scale + log2 width <= 62): the same whatever lanes and waves add up.  Every filter
// keeps a beginning of the order, so S' is the least of their sums, and sampling comes down to
// finding the entry at a given place in the order's running sum.
//
// F(v) = sum of the weights of entries above v falls as v rises, and changes at entries only: the entry at place P is
// among those of the least v with F(v) <= P, found by halving the range of v, its ties by halving their index.
#include "rows.h"

namespace cg {
namespace {

constexpr int MAX_WIDTH = 1 << 18;
constexpr int MAX_TOP = 256;

// What every row has alike, or of its own.
template <typename X, typename Y>
struct Control {
  X value;
  const Y *at;  // NULL: value
  __device__ __forceinline__ X of(int64_t row) const { return at ? X(at[row]) : value; }
};

struct ChooseArgs {
  const void *logits;
  const uint8_t *mask;
  int64_t ld_logits, ld_mask;
  int32_t rows, width;
  // sampling
  const double *uniforms;
  Control<double, float> temperature, top_p, min_p;
  Control<int64_t, int64_t> top_k;
  int32_t scale;  // a weight of 1 is 2^scale
  int64_t *actions;
  // the record
  int32_t k;
  int64_t *indices;
  float *log_rest;
  float *log_probs;
};

// ---- a row's group of lanes: a wave, or a block ----------------------------------------------------------------

template <int G>
struct Shared {
  static constexpr int W = G > 64 ? G / 64 : 1;
  uint64_t slots[2][W];
};

template <int G>
struct Group {
  Shared<G> &shared;
  int turn = 0;
  __device__ __forceinline__ explicit Group(Shared<G> &s) : shared(s) {}
  static __device__ __forceinline__ int lane() { return threadIdx.x % G; }

  __device__ __forceinline__ void sync() const {
    if constexpr (G > 64) {
      __syncthreads();
    } else {  // the wave's LDS writes to its own reads
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
  // Joins x over the group, the result in every lane.  Slots are used in turn: one is written again only behind the
  // next join's barrier, which every wave reaches after its reads.
  template <typename X, typename Op>
  __device__ __forceinline__ X join(X x, Op op) {
    x = lanes_join<(G < 64 ? G : 64)>(x, op);
    if constexpr (G > 64) {
      constexpr int W = G / 64;
      X *slot = reinterpret_cast<X *>(shared.slots[turn]);
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = x;
      __syncthreads();
      x = lanes_join<W>(slot[threadIdx.x % W], op);
    }
    return x;
  }
};

// ---- a row's entries: in registers, or read again for every pass ---------------------------------------------
//
// each(visit): visit(index of entry 0, z) for this lane's vectors, z(k) the k-th logit, -inf where it is not legal.

// S: the type in which entries are kept (T, or float where rows are shorter than a load).
template <typename T, int G, int E, typename S = T>
struct Held {
  static constexpr int V = E == 1 ? 1 : VEC<T>, C = E / V;
  Entries<S, E> z;
  int width;
  __device__ __forceinline__ Held(const T *row, const uint8_t *legal, int width) : width(width) {
    load_entries<G, C, V>(z.w, row, legal, int(threadIdx.x % G) * V, width);
  }
  template <typename Visit>
  __device__ __forceinline__ void each(const Visit &visit) const {
    const int first = int(threadIdx.x % G) * V;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = V == 1 ? first : min(first + c * G * V, width - V);
      visit(at, [&](int k) { return z[c * V + k]; });
    }
  }
  // A row whose largest entry is +inf: these share everything.
  __device__ __forceinline__ void unbounded() {
    constexpr int PER = Entries<S, E>::PER;
    constexpr uint32_t NONE = NEGATIVE_INFINITY<S>;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const uint32_t part = PER == 1 ? ~0u : k % 2 ? 0xffff0000u : 0xffffu;
      const bool is = z[k] == INFINITY;
      uint32_t &w = z.w[k / PER];
      w = (w & ~part) | (is ? 0u : NONE & part);
    }
  }
};

template <typename T, int G>
struct Read {
  static constexpr int V = VEC<T>;
  const T *row;
  const uint8_t *legal;
  int width;
  bool infinite = false;
  __device__ __forceinline__ Read(const T *row, const uint8_t *legal, int width) : row(row), legal(legal), width(width) {}
  template <typename Visit>
  __device__ __forceinline__ void each(const Visit &visit) const {
    for (int i = int(threadIdx.x % G) * V; i < width; i += G * V) {
      Entries<T, V> q;
      load_entries<1, 1, V>(q.w, row, legal, i, width);
      visit(min(i, width - V), [&](int k) { return infinite ? (q[k] == INFINITY ? 0.f : -INFINITY) : q[k]; });
    }
  }
  __device__ __forceinline__ void unbounded() { infinite = true; }
};

// ---- order, weights --------------------------------------------------------------------------------------------

// Floats in their order as integers; -0 is 0.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// Integer weights: 2^scale e^((z - top) / T).
struct Weights {
  double top, c;  // c = log2(e) / T, finite: the top weighs 1
  double magic;   // 1.5 * 2^(52 - scale): a sum with it has the weight in its low bits, to the nearest
  __device__ __forceinline__ Weights(float top, double temperature, int scale)
      : top(top), c(fmin(1.44269504088896340736 / temperature, 1e300)), magic(__builtin_amdgcn_ldexp(1.5, 52 - scale)) {}
  // 2^t = 2^k 2^f, |f| <= 1/2: 2^f = 1 + f g(f), g interpolated at the nodes of Chebyshev's polynomial of degree 9;
  // off by 2^-44.6 of it at most, and 1 at 0.
  __device__ __forceinline__ uint64_t operator()(float z) const {
    const double t = fmax((double(z) - top) * c, -64.0);  // (a NaN of -inf and c = 0 too: a weight of 0 from -63 on)
    const double k = __builtin_rint(t), f = t - k;
    double p = 1.0202923985536321e-07;
    p = fma(p, f, 1.3255228630225242e-06);
    p = fma(p, f, 1.5252687853419455e-05);
    p = fma(p, f, 0.00015403455837972657);
    p = fma(p, f, 0.0013333558177508053);
    p = fma(p, f, 0.009618129159415947);
    p = fma(p, f, 0.055504108664767154);
    p = fma(p, f, 0.24022650695813);
    p = fma(p, f, 0.6931471805599454);
    p = fma(p, f, 1.0);
    const double sum = __builtin_amdgcn_ldexp(p, int(k)) + magic;
    return __builtin_bit_cast(uint64_t, sum) - __builtin_bit_cast(uint64_t, magic);
  }
};

// The sum of the weights above v; their count.
template <typename Row, int G>
__device__ __forceinline__ uint64_t mass_above(const Row &row, Group<G> &group, const Weights &weight, float v) {
  uint64_t s = 0;
  row.each([&](int, const auto &z) {
#pragma unroll
    for (int k = 0; k < Row::V; ++k)
      if (z(k) > v) s += weight(z(k));
  });
  return group.join(s, Plus{});
}
template <typename Row, int G>
__device__ __forceinline__ int count_above(const Row &row, Group<G> &group, float v) {
  int n = 0;
  row.each([&](int, const auto &z) {
#pragma unroll
    for (int k = 0; k < Row::V; ++k) n += z(k) > v;
  });
  return group.join(n, Plus{});
}

// The least v up to `top` at which of(v) < limit; of(v) falls as v rises, of(-inf) >= limit, of(top) = 0.
// value: of(v) there.
template <typename X, typename Of>
__device__ __forceinline__ float least_value(float top, X limit, const Of &of, X &value) {
  uint32_t lo = key_of(-INFINITY), hi = key_of(top);
  value = 0;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const X x = of(of_key(mid));
    if (x < limit)
      hi = mid, value = x;
    else
      lo = mid;
  }
  return of_key(hi);
}

// The index of entry number r (from 0) of those equal to v.
template <typename Row, int G>
__device__ __forceinline__ int tie(const Row &row, Group<G> &group, float v, int r) {
  int lo = -1, hi = row.width - 1;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    int n = 0;
    row.each([&](int at, const auto &z) {
#pragma unroll
      for (int k = 0; k < Row::V; ++k) n += z(k) == v && at + k <= mid;
    });
    if (group.join(n, Plus{}) > r)
      hi = mid;
    else
      lo = mid;
  }
  return hi;
}

// The row's largest entry, -inf where none is legal; nan: one of them is.
template <typename Row, int G>
__device__ __forceinline__ float row_top(Row &row, Group<G> &group, bool &nan) {
  float top = -INFINITY;
  int bad = 0;
  row.each([&](int, const auto &z) {
#pragma unroll
    for (int k = 0; k < Row::V; ++k) {
      top = fmaxf(top, z(k));
      bad |= z(k) != z(k);
    }
  });
  if (bad) top = NAN;
  // (the larger of two, NaN where one is)
  top = group.join(top, [](float a, float b) { return a > b || a != a ? a : b; });
  nan = top != top;
  if (top == INFINITY) {
    row.unbounded();
    top = 0;
  }
  return top;
}

// ---- sampling ----------------------------------------------------------------------------------------------------

template <typename Row, int G>
__device__ __forceinline__ void sample_row(const ChooseArgs &a, int64_t r, Row &row, Group<G> &group) {
  const double temperature = a.temperature.of(r), p = a.top_p.of(r), least = a.min_p.of(r), u = a.uniforms[r];
  const int64_t most = a.top_k.of(r);
  bool nan;
  const float top = row_top(row, group, nan);
  int64_t action = -1;
  float log_prob = 0;
  if (nan || !(temperature >= 0)) {
    log_prob = NAN;
  } else if (top > -INFINITY) {
    if (temperature == 0) {
      action = tie(row, group, top, 0);
    } else {
      const Weights weight(top, temperature, a.scale);
      const uint64_t one = uint64_t(1) << a.scale;
      uint64_t total = mass_above(row, group, weight, -INFINITY);
      if (most > 0 && most < a.width && most < count_above(row, group, -INFINITY)) {
        int above;
        const float v = least_value(top, int(most), [&](float x) { return count_above(row, group, x); }, above);
        total = mass_above(row, group, weight, v) + (most - above) * weight(v);
      }
      const auto mass = [&](float x) { return mass_above(row, group, weight, x); };
      uint64_t kept = total;
      if (p < 1) {
        const uint64_t limit = p > 0 ? uint64_t(ceil(p * double(total))) : 1;
        uint64_t above;
        const float v = least_value(top, limit > 0 ? limit : 1, mass, above);
        const uint64_t w = weight(v);
        kept = min(kept, above + (limit - above + w - 1) / w * w);
      }
      if (least > 0) {
        const double x = ceil(least * double(one));
        const uint64_t bound = x < double(one) ? uint64_t(x) : one;
        uint64_t s = 0;
        row.each([&](int, const auto &z) {
#pragma unroll
          for (int k = 0; k < Row::V; ++k) {
            const uint64_t w = weight(z(k));
            s += w >= bound ? w : 0;
          }
        });
        s = group.join(s, Plus{});
        kept = min(kept, least > 1 ? one : s);
      }
      // The entry at place u S' (as integers: the first running sum above it); the last one for a u of 1 or NaN.
      const double at = u * double(kept);
      uint64_t place = at > 0 ? at < double(kept) ? uint64_t(at) : kept - 1 : u != u ? kept - 1 : 0;
      place = min(place, kept - 1);
      uint64_t above;
      const float v = least_value(top, place + 1, mass, above);
      const uint64_t w = weight(v);
      action = tie(row, group, v, int((place - above) / w));
      log_prob = float((double(v) - double(top)) / temperature - (log_of(double(kept)) - a.scale * 0.69314718055994530942));
    }
  }
  if (group.lane() == 0) {
    a.actions[r] = action;
    a.log_probs[r] = log_prob;
  }
}

// ---- the record --------------------------------------------------------------------------------------------------

struct Top {
  float z;
  int index;
  // Whether this stands before o in the order.
  __device__ __forceinline__ bool before(const Top &o) const { return z > o.z || (z == o.z && index < o.index); }
};

template <typename Row, int G>
__device__ __forceinline__ void top_row(const ChooseArgs &a, int64_t r, Row &row, Group<G> &group, Top *list, int *count) {
  const double temperature = a.temperature.of(r);
  const int lane = group.lane();
  float *log_probs = a.log_probs + r * a.k;
  int64_t *indices = a.indices + r * a.k;
  bool nan;
  const float top = row_top(row, group, nan);
  int held = 0;
  double log_total = 0;
  float log_rest = nan ? NAN : -INFINITY;
  if (!nan && top > -INFINITY) {
    const int legal = count_above(row, group, -INFINITY);
    held = min(a.k, legal);
    // Entries above v, and those equal to it up to index `last`.
    float v = -INFINITY;
    int last = -1;
    if (held < legal) {
      int above;
      v = least_value(top, held, [&](float x) { return count_above(row, group, x); }, above);
      last = tie(row, group, v, held - above - 1);
    }
    if (lane == 0) *count = 0;
    group.sync();
    const auto in = [&](float z, int i) { return z > v || (z == v && i <= last); };
    float next = -INFINITY;  // the largest of the others
    row.each([&](int at, const auto &z) {
#pragma unroll
      for (int k = 0; k < Row::V; ++k) {
        if (z(k) == -INFINITY) continue;
        if (in(z(k), at + k))
          list[atomicAdd(count, 1)] = Top{z(k), at + k};
        else
          next = fmaxf(next, z(k));
      }
    });
    next = group.join(next, Most{});
    const float from = next > -INFINITY ? next : 0.f;
    const double c = 1.44269504088896340736 / temperature;
    const float fast = float(c), rest = float(c - double(fast));
    // e^((z - from) / T), with what the rounding of the product cuts off
    double s = 0;
    row.each([&](int at, const auto &z) {
#pragma unroll
      for (int k = 0; k < Row::V; ++k) {
        if (z(k) == -INFINITY || in(z(k), at + k)) continue;
        const float d = z(k) - from, t = d * fast;
        s += __builtin_amdgcn_exp2f(t) * (1 + fmaf(d, rest, fmaf(d, fast, -t)) * 0.69314718f);
      }
    });
    s = group.join(s, Add{});
    group.sync();
    double in_list = 0;
    for (int i = lane; i < held; i += G) in_list += exp_of((double(list[i].z) - double(top)) / temperature);
    in_list = group.join(in_list, Add{});
    const double gap = (double(from) - double(top)) / temperature;
    log_total = log_of(in_list + (s > 0 ? s * exp_of(gap) : 0.0));
    if (s > 0) log_rest = float(gap + log_of(s) - log_total);
    for (int i = lane; i < held; i += G) {
      const Top mine = list[i];
      int rank = 0;
      for (int j = 0; j < held; ++j) rank += list[j].before(mine);
      log_probs[rank] = float((double(mine.z) - double(top)) / temperature - log_total);
      indices[rank] = mine.index;
    }
  }
  for (int i = held + lane; i < a.k; i += G) {
    log_probs[i] = nan ? NAN : -INFINITY;
    indices[i] = -1;
  }
  if (lane == 0) a.log_rest[r] = log_rest;
}

// ---- kernels -------------------------------------------------------------------------------------------------------

template <typename T, int G, typename Row, bool RECORD>
__global__ __launch_bounds__((G > 256 ? G : 256)) void choose_kernel(const ChooseArgs a) {
  constexpr int ROWS = G > 256 ? 1 : 256 / G;
  __shared__ Shared<G> shared[ROWS];
  __shared__ Top list[RECORD ? ROWS : 1][RECORD ? MAX_TOP : 1];
  __shared__ int count[ROWS];
  const int in_block = G < 256 ? __builtin_amdgcn_readfirstlane(threadIdx.x / G) : 0;
  const int64_t r = int64_t(blockIdx.x) * ROWS + in_block;
  if (r >= a.rows) return;  // (whole groups; a group's barriers are its own wave's, or its own block's)
  Group<G> group(shared[in_block]);
  Row row(static_cast<const T *>(a.logits) + r * a.ld_logits, a.mask ? a.mask + r * a.ld_mask : nullptr, a.width);
  if constexpr (RECORD)
    top_row(a, r, row, group, list[in_block], &count[in_block]);
  else
    sample_row(a, r, row, group);
}

struct Launch {
  void (*kernel)(ChooseArgs);
  int rows, threads;  // rows a block takes
};

template <typename T, int G, int E, bool RECORD, typename S = T>
Launch launch_as() {
  return {choose_kernel<T, G, Held<T, G, E, S>, RECORD>, G > 256 ? 1 : 256 / G, G > 256 ? G : 256};
}

template <typename T, bool RECORD>
Launch launch_of(int width) {
  if (width < VEC<T>) return launch_as<T, 64, 1, RECORD, float>();
  if (width <= 512) return launch_as<T, 64, 8, RECORD>();
  if (width <= 1024) return launch_as<T, 64, 16, RECORD>();
  if (width <= 4096) return launch_as<T, 256, 16, RECORD>();
  if (width <= 8192) return launch_as<T, 256, 32, RECORD>();
  if (width <= 16384) return launch_as<T, 512, 32, RECORD>();
  if constexpr (sizeof(T) == 2) {
    if (width <= 32768) return launch_as<T, 512, 64, RECORD>();
    if (width <= 65536) return launch_as<T, 1024, 64, RECORD>();
  } else if (width <= 32768) {
    return launch_as<T, 1024, 32, RECORD>();
  }
  return {choose_kernel<T, 1024, Read<T, 1024>, RECORD>, 1, 1024};
}

template <bool RECORD>
void launch(const ChooseArgs &a, int dtype, hipStream_t stream) {
  const Launch l = dtype == CG_F32    ? launch_of<float, RECORD>(a.width)
                   : dtype == CG_BF16 ? launch_of<bf16, RECORD>(a.width)
                                      : launch_of<f16, RECORD>(a.width);
  l.kernel<<<unsigned((int64_t(a.rows) + l.rows - 1) / l.rows), l.threads, 0, stream>>>(a);
  CG_LAUNCHED();
}

ChooseArgs args_of(const cg_policy_rows *p, const char *who) {
  CG_REQUIRE(p != nullptr, CG_ERR_INVALID, "rows is NULL");
  dtype_size(p->dtype);
  CG_REQUIRE(p->rows >= 0 && p->width > 0, CG_ERR_INVALID, "rows must be non-negative, width positive");
  CG_REQUIRE(p->width <= MAX_WIDTH, CG_ERR_UNSUPPORTED, std::string(who) + ": rows wider than 2^18");
  CG_REQUIRE(p->rows == 0 || p->logits, CG_ERR_INVALID, "logits are required");
  CG_REQUIRE(p->ld_logits >= 0 && p->ld_mask >= 0, CG_ERR_INVALID, "row strides must be non-negative");
  ChooseArgs a{};
  a.logits = p->logits, a.mask = p->mask;
  a.ld_logits = p->ld_logits, a.ld_mask = p->ld_mask;
  a.rows = p->rows, a.width = p->width;
  return a;
}

}  // namespace
}  // namespace cg

using namespace cg;

extern "C" {

int cg_sample_logits(const cg_policy_rows *rows, const double *uniforms, const cg_sample_controls *controls,
                     int64_t *actions, float *log_probs, void *stream) {
  return guarded([&] {
    ChooseArgs a = args_of(rows, "sample_logits");
    CG_REQUIRE(controls, CG_ERR_INVALID, "controls are required");
    const cg_sample_controls &c = *controls;
    CG_REQUIRE(c.temperatures || (c.temperature >= 0 && c.temperature < INFINITY), CG_ERR_INVALID,
               "temperature must be finite and not negative");
    if (a.rows == 0) return;
    CG_REQUIRE(uniforms && actions && log_probs, CG_ERR_INVALID, "uniforms, actions and log_probs are required");
    a.uniforms = uniforms, a.actions = actions, a.log_probs = log_probs;
    a.temperature = {c.temperature, c.temperatures};
    a.top_p = {c.top_p, c.top_ps}, a.min_p = {c.min_p, c.min_ps};
    a.top_k = {c.top_k, c.top_ks};
    int bits = 0;
    while (1 << bits < a.width) ++bits;
    a.scale = min(50, 62 - bits);
    launch<false>(a, rows->dtype, as_stream(stream));
  });
}

int cg_top_logits(const cg_policy_rows *rows, int32_t k, double temperature, float *log_probs, int64_t *indices,
                  float *log_rest, void *stream) {
  return guarded([&] {
    ChooseArgs a = args_of(rows, "top_logits");
    CG_REQUIRE(k > 0 && k <= MAX_TOP, CG_ERR_INVALID, "k must be from 1 to 256");
    CG_REQUIRE(temperature >= 1e-30 && temperature <= 1e30, CG_ERR_INVALID, "temperature must be from 1e-30 to 1e30");
    if (a.rows == 0) return;
    CG_REQUIRE(log_probs && indices && log_rest, CG_ERR_INVALID, "log_probs, indices and log_rest are required");
    a.k = k, a.log_probs = log_probs, a.indices = indices, a.log_rest = log_rest;
    a.temperature = {temperature, nullptr};
    launch<true>(a, rows->dtype, as_stream(stream));
  });
}

}  // extern "C"
