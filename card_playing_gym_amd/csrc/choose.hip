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
// row are exact 64-bit integers (scale + log2 width <= 62): the same whatever lanes and waves add up.  That is chosen
// over float64 weights, whose sums would go by the order of the atomics: an entry is off by 2^-44 of its weight and by half
// of 2^-scale of the largest, 2^-51 in rows of up to 4096 entries and 2^-45 in the widest, where a uniform number of
// 2^-53 steps would meet an entry of less (which is never drawn) once in 2^45 draws.  Every filter
// keeps a beginning of the order, so S' is the least of their sums, and sampling comes down to
// finding the entry at a given place in the order's running sum.
//
// Finding that entry, or the k-th: a histogram of the row's weights (or of ones) in LDS, over bins of equal width in z, says
// which bin the place falls into and what is summed up before it.  The entries of that bin, a few dozen, go into a
// list, where each one adds up what stands before it.  A bin of more entries than the list has room for is cut into
// bins again, between its least and its largest entry; one of equal entries is decided by halving the range of their indices
// (and one of entries that differ by less than 1e-38 by halving the range of their values before).
// The first k of a row with k up to the lanes of its group need no histogram: at least k entries are as large as the k-th
// largest of the lanes' own maxima, and not many more, so these are the list.
//
// A row is read from HBM once (what its bytes take: bf16 4096 x 32768 53 us) and looked through in LDS, so wide rows
// are bound by VALU instructions: 8 an entry for its load and the maximum, 25 for its weight and the histogram, up to
// 9 for each entry that is looked for.  us there: greedy 43, the record of 64 entries 101 to 113, no filter 159,
// top_p 198 to 206.  Few rows are bound by the latency of passes and barriers (256 x 32768 with every filter 38),
// rows of up to 64 entries by their scalars.  These are of normal logits.  Where many entries have few values, atomics to
// the same bin wait for each other and a bin has more entries than the list: with all entries equal no filter takes 818 us
// there, top_p 1230 and the record 988 (16 values 757, 1143 and 946); at 4096 x 512 22, 25 and 26 (normal 12, 15 and 17).
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

struct Least {
  template <typename X>
  __device__ __forceinline__ X operator()(X a, X b) const {
    return a < b ? a : b;
  }
};
struct Largest {
  template <typename X>
  __device__ __forceinline__ X operator()(X a, X b) const {
    return a > b ? a : b;
  }
};

// The sum over a wave's lanes up to and with this one: within rows of 16 lanes, then rows 0 and 2 into the next, then the
// lower half into the upper.
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ uint64_t from_lower(uint64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(x)), CONTROL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(x >> 32)), CONTROL, ROWS, 0xf, false);
  return uint64_t(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_running_sum(uint64_t x) {
  x += from_lower<0x111>(x);       // row_shr:1
  x += from_lower<0x112>(x);       // row_shr:2
  x += from_lower<0x114>(x);       // row_shr:4
  x += from_lower<0x118>(x);       // row_shr:8
  x += from_lower<0x142, 0xa>(x);  // row_bcast:15
  x += from_lower<0x143, 0xc>(x);  // row_bcast:31
  return x;
}

// An entry in a list: its place in the order as a number (larger ones first), and its weight.
struct Item {
  uint64_t key, weight;
};

template <int G>
struct Shared {
  static constexpr int W = G > 64 ? G / 64 : 1;
  static constexpr int BINS = G > 64 ? 1024 : 256, LIST = G > 64 ? 512 : 256, JOINED = G > 256 ? LIST : 0;
  uint64_t slots[2][W];
  union {  // (the bins are in registers when a list is made)
    uint64_t bins[BINS];
    struct {
      Item list[LIST];
      uint64_t before[JOINED > 0 ? JOINED : 1];
      int rank[JOINED > 0 ? JOINED : 1];
    };
  };
  uint64_t found[2];
  int count;
};

template <int G>
struct Group {
  Shared<G> &shared;
  int turn = 0;
  __device__ __forceinline__ explicit Group(Shared<G> &s) : shared(s) {}
  static __device__ __forceinline__ int lane() { return threadIdx.x % G; }

  __device__ __forceinline__ void sync() const { group_sync<G>(); }
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
  // The sum over the lanes before this one, and over all.
  __device__ __forceinline__ uint64_t sum_before(uint64_t x, uint64_t &all) {
    const uint64_t upto = wave_running_sum(x);
    uint64_t before = upto - x;
    all = __shfl(upto, 63, 64);
    if constexpr (G > 64) {
      constexpr int W = G / 64;
      uint64_t *slot = shared.slots[turn];
      turn ^= 1;
      if ((threadIdx.x & 63) == 63) slot[threadIdx.x >> 6] = upto;
      __syncthreads();
      all = 0;
      const int wave = threadIdx.x >> 6;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        before += w < wave ? slot[w] : 0;
        all += slot[w];
      }
    }
    return before;
  }
};

// ---- a row's entries: in LDS, or read again for every pass ----------------------------------------------------
//
// A row is looked through several times, each time with little to do for most entries: from LDS that costs a fifth of
// what the entries' weights cost, while kept in registers they take most of what a lane has, and code of their number.
// each(visit): visit(index of entry 0, z) for this lane's vectors, z(k) the k-th logit, -inf where it is not legal.  A
// lane reads what it has written: no barrier stands between.

// NaN where one is.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <typename Row>
__device__ __forceinline__ float largest_of(const Row &row) {
  float most = -INFINITY;
  row.each([&](int, const auto &z) {
#pragma unroll
    for (int k = 0; k < Row::V; ++k) most = larger(most, z(k));
  });
  return most;
}

// The vector from entry i on, -inf for those that are not legal; a row's last one is its last V entries, of which those
// that the one before has count as -inf.
template <typename T, int V>
__device__ __forceinline__ void load_vector(uint32_t *w, const T *row, const uint8_t *legal, int i, int width) {
  if constexpr (V == 2) {
    const int at = min(i, width - 2);
    const bool first = at == i && (!legal || legal[at]), second = !legal || legal[at + 1];
    __builtin_memcpy(w, row + at, 2 * sizeof(T));
    constexpr uint32_t NONE = NEGATIVE_INFINITY<T>;
    if constexpr (sizeof(T) == 4) {
      w[0] = first ? w[0] : NONE;
      w[1] = second ? w[1] : NONE;
    } else {
      w[0] = first ? w[0] : (w[0] & 0xffff0000u) | (NONE & 0xffffu);
      w[0] = second ? w[0] : (w[0] & 0xffffu) | (NONE & 0xffff0000u);
    }
  } else if (i + V <= width) {
    __builtin_memcpy(w, row + i, 16);
    if (legal) {
      uint32_t b[V / 4];
      __builtin_memcpy(b, legal + i, V);
#pragma unroll
      for (int j = 0; j < V / 4; ++j) bar<T>(w + (sizeof(T) == 4 ? 4 : 2) * j, b[j]);
    }
  } else {
    load_entries<1, 1, V>(w, row, legal, i, width);
  }
}

// Vectors are 16 bytes, or two entries where rows have fewer bytes than 16 for each lane: us a pass with either, bf16
// 32768 x 256 (the 32 largest) 163 and 54, 65536 x 77 (top_p) 121 and 107, but 16384 x 1000 (masked) 37 and 57.
template <typename T, int G, int BYTES>
struct InLds {
  static constexpr int V = BYTES > 16 * G ? VEC<T> : 2, SIZE = V * int(sizeof(T)), VECTORS = BYTES / SIZE;
  static constexpr int BATCH = VECTORS / G < 8 ? VECTORS / G : 8;
  struct alignas(SIZE) Vector {
    uint32_t w[SIZE / 4];
  };
  Vector *held;
  int width, vectors;
  float most = -INFINITY;  // of this lane's entries, as they came
  __device__ __forceinline__ InLds(Vector *held, const T *row, const uint8_t *legal, int width)
      : held(held), width(width), vectors((width + V - 1) / V) {
    const int lane = threadIdx.x % G;
    for (int first = 0; first < vectors; first += G * BATCH) {
      Entries<T, V> q[BATCH];
#pragma unroll
      for (int c = 0; c < BATCH; ++c) {
        const int from = first + c * G;  // (the same for all lanes, as is whether all of theirs are whole)
        if (!legal && (from + G) * V <= width)
          __builtin_memcpy(q[c].w, row + int64_t(from) * V + lane * V, SIZE);
        else
          load_vector<T, V>(q[c].w, row, legal, min(from + lane, vectors - 1) * V, width);
      }
#pragma unroll
      for (int c = 0; c < BATCH; ++c)
        if (first + c * G + lane < vectors) {
          __builtin_memcpy(&held[first + c * G + lane], q[c].w, SIZE);
#pragma unroll
          for (int k = 0; k < V; ++k) most = larger(most, q[c][k]);
        }
    }
  }
  __device__ __forceinline__ float largest() const { return most; }
  __device__ __forceinline__ int at(int j) const { return min(j * V, width - V); }
  template <typename Visit>
  __device__ __forceinline__ void each(const Visit &visit) const {
#pragma unroll 1
    for (int j = threadIdx.x % G; j < vectors; j += G) {
      Entries<T, V> q;
      __builtin_memcpy(q.w, &held[j], SIZE);
      visit(at(j), [&](int k) { return q[k]; });
    }
  }
  // A row whose largest entry is +inf: these share everything.
  __device__ __forceinline__ void unbounded() {
    for (int j = threadIdx.x % G; j < vectors; j += G) {
      Entries<T, V> q;
      __builtin_memcpy(q.w, &held[j], SIZE);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const uint32_t part = sizeof(T) == 4 ? ~0u : k % 2 ? 0xffff0000u : 0xffffu;
        uint32_t &w = q.w[k / Entries<T, V>::PER];
        w = (w & ~part) | (q[k] == INFINITY ? 0u : NEGATIVE_INFINITY<T> & part);
      }
      __builtin_memcpy(&held[j], q.w, SIZE);
    }
  }
};

template <typename T, int G>
struct Read {
  static constexpr int V = VEC<T>, BATCH = 4;
  const T *row;
  const uint8_t *legal;
  int width;
  bool infinite = false;
  __device__ __forceinline__ Read(const T *row, const uint8_t *legal, int width) : row(row), legal(legal), width(width) {}
  template <typename Visit>
  __device__ __forceinline__ void each(const Visit &visit) const {
    const int vectors = (width + V - 1) / V;
    for (int first = threadIdx.x % G; first < vectors; first += G * BATCH) {
      Entries<T, V> q[BATCH];
#pragma unroll
      for (int c = 0; c < BATCH; ++c) load_vector<T, V>(q[c].w, row, legal, min(first + c * G, vectors - 1) * V, width);
#pragma unroll
      for (int c = 0; c < BATCH; ++c)
        if (first + c * G < vectors) {
          const int at = min((first + c * G) * V, width - V);
          visit(at, [&](int k) { return infinite ? (q[c][k] == INFINITY ? 0.f : -INFINITY) : q[c][k]; });
        }
    }
  }
  __device__ __forceinline__ float largest() const { return largest_of(*this); }
  __device__ __forceinline__ void unbounded() { infinite = true; }
};

// ---- order, weights --------------------------------------------------------------------------------------------

// Floats in their order as integers; -0 is 0.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// A constant in scalar registers: from vector registers the compiler copies it for each use.
__device__ __forceinline__ double scalar_of(double c) {
  int lo = __double2loint(c), hi = __double2hiint(c);
  asm("" : "+s"(lo), "+s"(hi));
  return __hiloint2double(hi, lo);
}

// Integer weights: 2^scale e^((z - top) / T).
struct Weights {
  double top, c;  // c = log2(e) / T, finite: the top weighs 1
  double magic;   // 1.5 * 2^(52 - scale): a sum with it has the weight in its low bits, to the nearest
  double reach;   // 60 octaves
  double g[9];
  // 2^t = 2^k 2^f, |f| <= 1/2: 2^f = 1 + f g(f), g interpolated at the nodes of Chebyshev's polynomial of degree 9;
  // off by 2^-44.6 of it at most, and 1 at 0.
  __device__ __forceinline__ Weights(float top, double temperature, int scale)
      : top(top), c(fmin(1.44269504088896340736 / temperature, 1e300)), magic(__builtin_amdgcn_ldexp(1.5, 52 - scale)),
        reach(60 * 0.69314718055994530942 * temperature),
        g{scalar_of(0.6931471805599454), scalar_of(0.24022650695813), scalar_of(0.055504108664767154),
          scalar_of(0.009618129159415947), scalar_of(0.0013333558177508053), scalar_of(0.00015403455837972657),
          scalar_of(1.5252687853419455e-05), scalar_of(1.3255228630225242e-06), 1.0202923985536321e-07} {
    asm("" : "+v"(g[8]));  // (one operand of an instruction may be scalar)
  }
  // Of any z; 0 below 2^-64.
  __device__ __forceinline__ uint64_t operator()(float z) const { return z >= least() ? near(z) : 0; }
  // Of z >= least().
  __device__ __forceinline__ uint64_t near(float z) const {
    const double d = double(z) - top;
    // (adding 1.5 * 2^52 rounds to whole numbers, k's low bits the sum's)
    const double whole = fma(d, c, 6755399441055744.0), f = fma(d, c, 6755399441055744.0 - whole);
    double p = fma(g[8], f, g[7]);
    p = fma(p, f, g[6]);
    p = fma(p, f, g[5]);
    p = fma(p, f, g[4]);
    p = fma(p, f, g[3]);
    p = fma(p, f, g[2]);
    p = fma(p, f, g[1]);
    p = fma(p, f, g[0]);
    p = fma(p, f, 1.0);
    const double sum = __hiloint2double(__double2hiint(p) + (__double2loint(whole) << 20), __double2loint(p)) + magic;
    int high = __double2hiint(sum) - __double2hiint(magic);  // (magic's low word is 0)
    asm("" : "+v"(high));  // (or the compiler makes a subtraction of both words of it)
    return uint64_t(uint32_t(high)) << 32 | uint32_t(__double2loint(sum));
  }
  // All that weigh anything are as large (2^scale e^d is below 1/2 from t = -52 on), and t >= -64.
  __device__ __forceinline__ float least() const {
    const double z = top - reach;
    float x = z > -0x1.fffffep127 ? float(z) : -0x1.fffffep127f;
    return (double(x) - top) * c < -64.0 ? of_key(key_of(x) + 1) : x;  // (one step, where z was rounded down)
  }
};

// An entry's place in the order as a number: larger ones come first.
__device__ __forceinline__ uint64_t place_of(float z, int index) { return uint64_t(key_of(z)) << 32 | uint32_t(~index); }
__device__ __forceinline__ float value_at(uint64_t place) { return of_key(uint32_t(place >> 32)); }
__device__ __forceinline__ int index_at(uint64_t place) { return int(~uint32_t(place)); }

// A row's largest entry, -inf where none is legal and NaN where one of them is; of this lane's entries: `mine`.
template <typename Row, int G>
__device__ __forceinline__ float row_top(Row &row, Group<G> &group, float &mine) {
  mine = row.largest();
  float top = group.join(mine, larger);
  if (top == INFINITY) {
    row.unbounded();
    mine = largest_of(row);
    top = group.join(mine, larger);
  }
  return top;
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

template <typename Row, int G>
__device__ __forceinline__ int first_index(const Row &row, Group<G> &group, float v) {
  int first = row.width;
  row.each([&](int at, const auto &z) {
#pragma unroll
    for (int k = 0; k < Row::V; ++k) first = min(first, z(k) == v ? at + k : row.width);
  });
  return group.join(first, Least{});
}

// A value that at least n <= G of the row's entries are as large as, and not many more: near the n-th largest of
// the lanes' maxima.  -inf where fewer lanes have an entry.
template <int G>
__device__ __forceinline__ float bound_of_top(Group<G> &group, float top, float mine, int n) {
  constexpr int W = G / 64;
  float tops[W];
  if constexpr (G > 64) {
    float *all = reinterpret_cast<float *>(group.shared.bins);
    all[threadIdx.x] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) tops[w] = all[w * 64 + (threadIdx.x & 63)];
    __syncthreads();  // (the bins are used next)
  } else {
    tops[0] = mine;
  }
  const auto count = [&](float v) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) c += __popcll(__ballot(tops[w] >= v));
    return c;
  };
  float lo = INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) lo = fminf(lo, tops[w] == -INFINITY ? INFINITY : tops[w]);
  lo = lanes_join<64>(lo, Least{});
  if (lo == INFINITY || count(lo) < n) return -INFINITY;
  float hi = top;
  for (int turn = 0; turn < 40; ++turn) {  // (lo: at least n are as large)
    const float mid = 0.5f * lo + 0.5f * hi;
    if (!(mid > lo && mid < hi)) break;
    const int c = count(mid);
    if (c >= n) {
      lo = mid;
      if (c <= n + n / 8) break;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// The entries for which in(z, index) holds into the list.  Returns how many there are, of which those past the list's
// room are not in it.  after(): behind each of this lane's vectors.
template <typename Row, int G, typename In, typename After>
__device__ __forceinline__ int gather(const Row &row, Group<G> &group, const In &in, const After &after) {
  Shared<G> &s = group.shared;
  if constexpr (G == 64) {  // (a wave counts for itself)
    int n = 0;
    row.each([&](int at, const auto &z) {
#pragma unroll
      for (int k = 0; k < Row::V; ++k) {
        const bool is = in(z(k), at + k);
        const uint64_t all = __ballot(is);
        const int slot = n + __builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0));
        if (is && slot < Shared<G>::LIST) s.list[slot].key = place_of(z(k), at + k);
        n += __popcll(all);
      }
      after();
    });
    group.sync();
    return __builtin_amdgcn_readfirstlane(n);  // (lane 0 takes every turn that any takes)
  }
  if (group.lane() == 0) s.count = 0;
  group.sync();
  row.each([&](int at, const auto &z) {
    bool is[Row::V], any = false;
#pragma unroll
    for (int k = 0; k < Row::V; ++k) any |= is[k] = in(z(k), at + k);
    after();
    if (!any) return;
#pragma unroll
    for (int k = 0; k < Row::V; ++k) {
      if (!is[k]) continue;
      const int slot = atomicAdd(&s.count, 1);
      if (slot < Shared<G>::LIST) s.list[slot].key = place_of(z(k), at + k);
    }
  });
  group.sync();
  return s.count;
}
template <typename Row, int G, typename In>
__device__ __forceinline__ int gather(const Row &row, Group<G> &group, const In &in) {
  return gather(row, group, in, [] {});
}

// This lane's items of a list, their weights (weight(z)), and what stands before each.  In blocks of 512 lanes and more
// every wave adds up a part of the list for all of its items: the one or two waves that have them would be waited for
// (bf16 4096 x 32768 by top_p 216 and 207 us).  In narrower ones the room that the joining takes is worth more.
template <int G>
struct Mine {
  static constexpr int N = Shared<G>::LIST / G > 0 ? Shared<G>::LIST / G : 1;
  Item item[N];
  uint64_t before[N];
  int rank[N];
  bool in[N];
  template <typename Weight>
  __device__ __forceinline__ Mine(Group<G> &group, int n, const Weight &weight) {
    Shared<G> &s = group.shared;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = group.lane() + i * G;
      in[i] = at < n;
      item[i] = Item{0, 0};
      before[i] = 0;
      rank[i] = 0;
      if (in[i]) {
        item[i].key = s.list[at].key;
        s.list[at].weight = item[i].weight = weight(value_at(item[i].key));
        if constexpr (Shared<G>::JOINED > 0) s.before[at] = 0, s.rank[at] = 0;
      }
    }
    group.sync();
    if constexpr (Shared<G>::JOINED > 0) {
      constexpr int W = G / 64;
      const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = n * wave / W, last = n * (wave + 1) / W;
      for (int at = threadIdx.x & 63; at < n; at += 64) {
        const uint64_t key[1] = {s.list[at].key};
        uint64_t sum[1] = {0};
        int ahead[1] = {0};
        add_up<1>(s, key, first, last, sum, ahead);
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.before[at]), sum[0]);
        atomicAdd(&s.rank[at], ahead[0]);
      }
      group.sync();
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in[i]) before[i] = s.before[group.lane() + i * G], rank[i] = s.rank[group.lane() + i * G];
    } else {
      if (int(threadIdx.x % G) / 64 * 64 >= n) return;  // (waves without items)
      uint64_t key[N];
#pragma unroll
      for (int i = 0; i < N; ++i) key[i] = item[i].key;
      if (n <= G)
        add_up<1>(s, key, 0, n, before, rank);
      else if (n <= 2 * G)
        add_up<(N < 2 ? N : 2)>(s, key, 0, n, before, rank);
      else
        add_up<N>(s, key, 0, n, before, rank);
    }
  }
  template <int USED>
  static __device__ __forceinline__ void add_up(const Shared<G> &s, const uint64_t *key, int first, int last, uint64_t *sum,
                                                int *count) {
#pragma unroll 4
    for (int j = first; j < last; ++j) {
      const Item other = s.list[j];
#pragma unroll
      for (int i = 0; i < USED; ++i) {
        const bool ahead = other.key > key[i];
        sum[i] += ahead ? other.weight : 0;
        count[i] += ahead;
      }
    }
  }
};

// ---- the entry at a place of the running sum over the order ------------------------------------------------------

// Bins of equal width from `from` downwards, the last one for all below (and what float32 cannot tell from there).  A
// range of one value is one bin; of any other, its ends are in different ones, unless it is shorter than 1 / 1e38.
struct Bins {
  float from, scale, last, width;
  Bins() = default;
  __device__ __forceinline__ Bins(float from, float end, int n) : from(from), last(float(n - 1)) {
    const float half = 0.5f * from - 0.5f * end;  // (the whole may be above float32's largest)
    scale = half > 0 ? fminf(0.5f * last / half, 1e38f) : 0;
    width = 1 / scale;
  }
  __device__ __forceinline__ float at(float z) const { return fminf((from - z) * scale, last); }
  __device__ __forceinline__ bool in(int b, float z) const {
    const float x = at(z);
    return x >= float(b) && x < float(b + 1);
  }
  // A little more than the range of a bin's values: the roundings of at() and of these lines are 7 of 2^-24 together.
  __device__ __forceinline__ void range(int b, float &low, float &high) const {
    low = -INFINITY, high = INFINITY;
    if (scale == 0) return;
    const float near = float(b) * width, far = float(b + 1) * width;
    const float slack = 9 * 0x1p-24f * (fabsf(from) + far) + 0x1p-146f;
    high = from - near + slack;
    if (float(b) < last) low = from - far - slack;
  }
};

struct Entry {
  uint64_t place;  // in the order, as place_of
  uint64_t upto;   // the running sum with it
};

// The histogram of weight.near(z) over the entries of `low` to `high`; WITHIN: some are above `high`.
template <typename Row, int G>
struct Histogram {
  static constexpr int PER = Shared<G>::BINS / G;
  Bins bins;
  float low, high;
  uint64_t value[PER], before, total;  // of this lane's bins

  // The bins end at `end`, or lower.
  template <bool WITHIN = false, typename Weight>
  __device__ __forceinline__ void make(const Row &row, Group<G> &group, const Weight &weight, float from, float end, float least) {
    bins = Bins(from, end, Shared<G>::BINS);
    low = least, high = from;
    Shared<G> &s = group.shared;
    const int lane = group.lane();
    for (int b = lane; b < Shared<G>::BINS; b += G) s.bins[b] = 0;
    group.sync();
    row.each([&](int, const auto &z) {
#pragma unroll
      for (int k = 0; k < Row::V; ++k)
        if (z(k) >= low && !(WITHIN && z(k) > high))
          atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[int(bins.at(z(k)))]), weight.near(z(k)));
    });
    group.sync();
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      value[i] = s.bins[lane * PER + i];
      mine += value[i];
    }
    before = group.sum_before(mine, total);
  }
  // The bin where the running sum reaches `sum` (1 to total), and what is summed up before it.
  __device__ __forceinline__ int locate(Group<G> &group, uint64_t sum, uint64_t &ahead) const {
    Shared<G> &s = group.shared;
    uint64_t b = before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (b < sum && sum <= b + value[i]) {
        s.found[0] = group.lane() * PER + i;
        s.found[1] = b;
      }
      b += value[i];
    }
    group.sync();
    ahead = s.found[1];
    return int(s.found[0]);
  }
  // The sum of the entries above v, v from `low` to `high`.
  template <typename Weight>
  __device__ __forceinline__ uint64_t above(const Row &row, Group<G> &group, const Weight &weight, float v) const {
    Shared<G> &s = group.shared;
    const int bin = int(bins.at(v));
    uint64_t b = before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (group.lane() * PER + i == bin) s.found[0] = b;
      b += value[i];
    }
    float least, most;
    bins.range(bin, least, most);
    most = fminf(most, high);
    const int n = gather(row, group, [&](float z, int) { return z > v && z <= most; });
    const uint64_t ahead = s.found[0];
    uint64_t x = 0;
    if (n <= Shared<G>::LIST) {
      for (int i = group.lane(); i < n; i += G) {
        const float z = value_at(s.list[i].key);
        x += bins.in(bin, z) ? weight.near(z) : 0;
      }
    } else {
      row.each([&](int, const auto &z) {
#pragma unroll
        for (int k = 0; k < Row::V; ++k)
          if (z(k) > v && z(k) <= most && bins.in(bin, z(k))) x += weight.near(z(k));
      });
    }
    return ahead + group.join(x, Plus{});
  }
  // The entry at which the running sum reaches `sum`.
  template <typename Weight>
  __device__ __forceinline__ Entry entry(const Row &row, Group<G> &group, const Weight &weight, uint64_t sum) const {
    Shared<G> &s = group.shared;
    Histogram h = *this;
    for (uint64_t ahead = 0;;) {
      uint64_t more;
      const int bin = h.locate(group, sum - ahead, more);
      ahead += more;
      float least, most;
      h.bins.range(bin, least, most);
      least = fmaxf(least, h.low), most = fminf(most, h.high);
      const Bins bins = h.bins;
      const int n = gather(row, group, [&](float z, int) { return z >= least && z <= most; });
      if (n <= Shared<G>::LIST) {
        // (those of the bins beside it weigh nothing here)
        const Mine<G> mine(group, n, [&](float z) { return bins.in(bin, z) ? weight.near(z) : 0; });
#pragma unroll
        for (int i = 0; i < Mine<G>::N; ++i) {
          const uint64_t b = ahead + mine.before[i];
          if (mine.in[i] && b < sum && sum <= b + mine.item[i].weight) {
            s.found[0] = mine.item[i].key;
            s.found[1] = b + mine.item[i].weight;
          }
        }
        group.sync();
        const Entry e{s.found[0], s.found[1]};
        group.sync();
        return e;
      }
      // Too many: bins within the bin, from its largest entry to its least.
      float lowest = INFINITY, largest = -INFINITY;
      row.each([&](int, const auto &z) {
#pragma unroll
        for (int k = 0; k < Row::V; ++k) {
          const bool is = z(k) >= least && z(k) <= most && bins.in(bin, z(k));
          lowest = fminf(lowest, is ? z(k) : INFINITY);
          largest = fmaxf(largest, is ? z(k) : -INFINITY);
        }
      });
      lowest = group.join(lowest, Least{});
      largest = group.join(largest, Largest{});
      if (Bins(largest, lowest, Shared<G>::BINS).at(lowest) < 1) {
        // Equal entries, or closer to each other than float32's reciprocals reach (numbers below its least normal one):
        // the value by halving its range, `over` the sum of those above, then the entry by halving the indices.
        uint32_t lo = key_of(lowest), hi = key_of(largest);
        uint64_t over = 0;
        while (lo < hi) {
          const uint32_t mid = hi - (hi - lo) / 2;
          uint64_t x = 0;
          row.each([&](int, const auto &z) {
#pragma unroll
            for (int k = 0; k < Row::V; ++k)
              if (z(k) <= largest && key_of(z(k)) >= mid) x += weight.near(z(k));
          });
          x = group.join(x, Plus{});
          if (x >= sum - ahead)
            lo = mid;
          else
            hi = mid - 1, over = x;
        }
        ahead += over;
        const float v = of_key(lo);
        const uint64_t w = weight.near(v), r = (sum - 1 - ahead) / w;
        return Entry{place_of(v, tie(row, group, v, int(r))), ahead + (r + 1) * w};
      }
      h.template make<true>(row, group, weight, largest, lowest, lowest);
    }
  }
};

// Counts.
struct One {
  __device__ __forceinline__ uint64_t operator()(float) const { return 1; }
  __device__ __forceinline__ uint64_t near(float) const { return 1; }
};

// Where a histogram may end: half as far again below the least of the lanes' maxima as the row's largest is above
// it.  A lane's maximum is the largest of what it has, so little is below; what is goes into the last bin.
template <int G>
__device__ __forceinline__ float low_end(Group<G> &group, float top, float mine) {
  const float least = group.join(mine == -INFINITY ? INFINITY : mine, Least{});
  return fmaxf(least - 1.5f * (top - least), -0x1.fffffep127f);
}

// The next number below z (below 0, not -0, which equals it).
__device__ __forceinline__ float below(float z) {
  const uint32_t k = key_of(z);
  return z == -INFINITY ? z : of_key(k == 0x80000000u ? k - 2 : k - 1);
}

// ---- sampling ----------------------------------------------------------------------------------------------------

// The largest k for which the lanes' maxima say where a row's first k end, and the list holds them.  Of a wave's 64
// lanes half: beyond, the list has more entries than the wave lanes (4096 x 512 fp32, k 50: 30 us, with the histogram 16).
template <int G>
constexpr int SHORT = G == 64 ? 32 : Shared<G>::LIST / 2;

// A row's controls.
struct Controls {
  double temperature, p, least, u;
  int64_t most;
  uint64_t one;  // the weight of 1
  __device__ __forceinline__ Controls(const ChooseArgs &a, int64_t r)
      : temperature(a.temperature.of(r)), p(a.top_p.of(r)), least(a.min_p.of(r)), u(a.uniforms[r]), most(a.top_k.of(r)),
        one(uint64_t(1) << a.scale) {}
  // min_p as the least weight that is kept: 1 without, the first entry's at most.
  __device__ __forceinline__ uint64_t bound() const {
    if (!(least > 0)) return 1;
    const double x = ceil(least * double(one));
    return x < double(one) ? uint64_t(x) : one;
  }
  // top_p as a sum: entries before which less than this is summed up are kept.
  __device__ __forceinline__ uint64_t limit(uint64_t total) const {
    const double x = ceil(p * double(total));
    return x > 1 ? uint64_t(x) : 1;
  }
  // The running sum that the answer's is the first to reach: u of what is kept, and a unit more; the last one's for a u
  // of 1 or NaN.
  __device__ __forceinline__ uint64_t target(uint64_t kept) const {
    const double x = u * double(kept);
    const uint64_t place = x > 0 ? x < double(kept) ? uint64_t(x) : kept - 1 : u != u ? kept - 1 : 0;
    return (place < kept ? place : kept - 1) + 1;
  }
  __device__ __forceinline__ float log_share(float z, float top, uint64_t kept, int scale) const {
    return float((double(z) - double(top)) / temperature - log_of(__builtin_amdgcn_ldexp(double(kept), -scale)));  // (0 for the whole)
  }
};

template <typename Row, int G>
__device__ __forceinline__ void sample_row(const ChooseArgs &a, int64_t r, Row &row, Group<G> &group) {
  Shared<G> &s = group.shared;
  const Controls c(a, r);
  const int64_t most = c.most;
  float mine;
  const float top = row_top(row, group, mine);
  const auto answer = [&](int64_t action, float log_prob) { a.actions[r] = action, a.log_probs[r] = log_prob; };
  if (top != top || !(c.temperature >= 0)) {
    if (group.lane() == 0) answer(-1, NAN);
    return;
  }
  if (top == -INFINITY) {
    if (group.lane() == 0) answer(-1, 0);
    return;
  }
  if (c.temperature == 0) {
    const int first = first_index(row, group, top);
    if (group.lane() == 0) answer(first, 0);
    return;
  }
  const Weights weight(top, c.temperature, a.scale);
  const uint64_t bound = c.bound();
  const bool limited = most > 0 && most < a.width;
  if (limited && most <= SHORT<G>) {
    const float under = below(bound_of_top(group, top, mine, int(most)));
    const int n = gather(row, group, [&](float z, int) { return z > under; });
    if (n <= Shared<G>::LIST) {
      const Mine<G> list(group, n, weight);
      const int last = most < n ? int(most) - 1 : n - 1;
      const auto each = [&](const auto &visit) {
#pragma unroll
        for (int i = 0; i < Mine<G>::N; ++i)
          if (list.in[i]) visit(list.item[i], list.before[i], list.rank[i]);
      };
      each([&](const Item &item, uint64_t before, int rank) {
        if (rank == last) s.found[0] = before + item.weight;
      });
      group.sync();
      uint64_t kept = s.found[0];
      if (c.p < 1) {
        const uint64_t limit = c.limit(kept);
        each([&](const Item &item, uint64_t before, int) {
          if (before < limit && limit <= before + item.weight) s.found[1] = before + item.weight;
        });
        group.sync();
        kept = s.found[1];
      }
      if (bound > 1) {
        uint64_t upto = 0;
        each([&](const Item &item, uint64_t before, int) {
          if (item.weight >= bound) upto = Largest{}(upto, before + item.weight);
        });
        kept = min(kept, c.least > 1 ? c.one : group.join(upto, Largest{}));
      }
      const uint64_t sum = c.target(kept);
      each([&](const Item &item, uint64_t before, int) {
        if (before < sum && sum <= before + item.weight) answer(index_at(item.key), c.log_share(value_at(item.key), top, kept, a.scale));
      });
      return;
    }
  }
  const float end = low_end(group, top, mine);
  Histogram<Row, G> h;
  float after = INFINITY;  // the first k: entries above the k-th's value, and this many of those equal to it
  int ties = 0;
  if (limited) {
    h.make(row, group, One{}, top, end, -0x1.fffffep127f);
    if (uint64_t(most) < h.total) {
      after = value_at(h.entry(row, group, One{}, uint64_t(most)).place);
      int above = 0;
      row.each([&](int, const auto &z) {
#pragma unroll
        for (int k = 0; k < Row::V; ++k) above += z(k) > after;
      });
      ties = int(most) - group.join(above, Plus{});
    }
  }
  const float lowest = weight.least();
  h.make(row, group, weight, top, fmaxf(end, lowest), lowest);
  uint64_t kept = h.total;
  if (after >= lowest && after < INFINITY) kept = h.above(row, group, weight, after) + ties * weight.near(after);
  if (c.p < 1) {
    const uint64_t limit = c.limit(kept);
    if (limit < kept) kept = h.entry(row, group, weight, limit).upto;
  }
  if (bound > 1) {
    // The largest value whose weight is not kept, by halving, near where the logarithm says it is.
    const uint32_t near = key_of(float(double(top) + log_of(c.least) * c.temperature));
    uint32_t lo = key_of(lowest), hi = key_of(top);
    if (weight.near(lowest) < bound) {
      if (near - 4 > lo && near < hi && weight.near(of_key(near - 4)) < bound) lo = near - 4;
      if (near > lo && near + 4 < hi && weight.near(of_key(near + 4)) >= bound) hi = near + 4;
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (weight.near(of_key(mid)) < bound)
          lo = mid;
        else
          hi = mid;
      }
      kept = min(kept, h.above(row, group, weight, of_key(lo)));
    }
  }
  if (c.least > 1) kept = c.one;
  const uint64_t place = h.entry(row, group, weight, c.target(kept)).place;
  if (group.lane() == 0) answer(index_at(place), c.log_share(value_at(place), top, kept, a.scale));
}

// ---- the record --------------------------------------------------------------------------------------------------

// e^((z - base) / T) in float32, -inf's 0.  log2(e) / T in two parts, both above 0: its rounding would be the same for all
// entries, and -inf stays -inf.
struct Share {
  float base, fast, slow;
  __device__ __forceinline__ Share(float base, double inverse) : base(base) {
    const double c = 1.44269504088896340736 * inverse;
    fast = float(c);
    if (double(fast) >= c) fast = __uint_as_float(__float_as_uint(fast) - 1);
    slow = float(c - double(fast));
  }
  __device__ __forceinline__ float operator()(float z) const {
    const float d = z - base;
    return __builtin_amdgcn_exp2f(fmaf(d, fast, d * slow));
  }
};

template <typename Row, int G>
__device__ __forceinline__ void top_row(const ChooseArgs &a, int64_t r, Row &row, Group<G> &group) {
  Shared<G> &s = group.shared;
  const double inverse = 1 / a.temperature.value;
  const int lane = group.lane();
  float *log_probs = a.log_probs + r * a.k;
  int64_t *indices = a.indices + r * a.k;
  float mine;
  const float top = row_top(row, group, mine);
  if (top != top || top == -INFINITY) {
    for (int i = lane; i < a.k; i += G) log_probs[i] = top, indices[i] = -1;
    if (lane == 0) a.log_rest[r] = top;
    return;
  }
  // The list: entries above `under`, or (too many) those up to the k-th, at `under` up to `index`.
  const One one;
  float under = -INFINITY;
  int index = -1, n = Shared<G>::LIST + 1;
  double low = 0;  // those not in the list, from `under`
  if (a.k >= a.width || a.k <= SHORT<G>) {
    // (one more, where the lanes suffice: the largest of the others)
    if (a.k < a.width) under = below(bound_of_top(group, top, mine, min(a.k + 1, G)));
    const Share weigh(under > -INFINITY ? under : 0.f, inverse);
    float sum = 0;  // (of a vector's 2 to 8, each off by (3 |d| + 4) 2^-24: 8 roundings more, then float64)
    n = gather(
        row, group,
        [&](float z, int) {
          const bool is = z > under;
          sum += is ? 0.f : weigh(z);
          return is;
        },
        [&] { low += sum, sum = 0; });
  }
  int ties = 0;  // of the others, those equal to the k-th
  if (n > Shared<G>::LIST) {
    Histogram<Row, G> h;
    h.make(row, group, one, top, low_end(group, top, mine), -0x1.fffffep127f);
    under = -INFINITY;
    if (uint64_t(a.k) < h.total) {
      const uint64_t place = h.entry(row, group, one, uint64_t(a.k)).place;
      under = value_at(place), index = index_at(place);
      row.each([&](int at, const auto &z) {
#pragma unroll
        for (int k = 0; k < Row::V; ++k) ties += z(k) == under && at + k > index;
      });
      ties = group.join(ties, Plus{});
    }
    n = gather(row, group, [&](float z, int i) { return z > under || (z == under && i <= index); });
    if (index >= 0) under = below(under);
  }
  // Into the order, whatever the order in which they came: sums go by it.
  {
    const Mine<G> list(group, n, one);
    group.sync();
#pragma unroll
    for (int i = 0; i < Mine<G>::N; ++i)
      if (list.in[i]) s.list[list.rank[i]] = list.item[i];
    group.sync();
  }
  const int held = min(n, a.k);
  // The others: those behind in the list, those not in it, and ties; `next` is their largest.  Where it is in the list,
  // those not in it were summed up while it was made, measured from `under`: one that is lost so far below is nothing beside
  // `next`.
  float next;
  if (n > a.k) {
    next = value_at(s.list[a.k].key);
  } else if (ties > 0) {
    next = of_key(key_of(under) + 1);
  } else {
    next = -INFINITY;
    row.each([&](int, const auto &z) {
#pragma unroll
      for (int k = 0; k < Row::V; ++k) next = fmaxf(next, z(k) <= under ? z(k) : -INFINITY);
    });
    next = group.join(next, Most{});
  }
  const Share weigh(next > -INFINITY ? next : 0.f, inverse);
  double others = 0, record = 0;
  if (n > a.k) {
    others = low > 0 ? low * exp_of((double(under) - double(next)) * inverse) : 0;
  } else {
    row.each([&](int, const auto &z) {
      float sum = 0;
#pragma unroll
      for (int k = 0; k < Row::V; ++k) sum += z(k) <= under ? weigh(z(k)) : 0.f;
      others += sum;
    });
  }
  if (lane == 0) others += ties;  // (the largest of the others, where there are any)
  for (int i = lane; i < n; i += G) {
    const float z = value_at(s.list[i].key);
    if (i < a.k)
      record += exp_of((double(z) - double(top)) * inverse);
    else
      others += weigh(z);
  }
  const double rest = group.join(others, Add{}), held_sum = group.join(record, Add{});
  const double gap = (double(weigh.base) - double(top)) * inverse;
  const double log_total = log_of(held_sum + (rest > 0 ? rest * exp_of(gap) : 0.0));
  for (int i = lane; i < a.k; i += G) {
    const uint64_t place = i < held ? s.list[i].key : 0;
    log_probs[i] = i < held ? float((double(value_at(place)) - double(top)) * inverse - log_total) : -INFINITY;
    indices[i] = i < held ? index_at(place) : -1;
  }
  if (lane == 0) a.log_rest[r] = rest > 0 ? float(gap + log_of(rest) - log_total) : -INFINITY;
}

// ---- rows of up to 64 entries: a lane an entry, 64 / G rows a wave ---------------------------------------------
//
// A lane counts what stands before its entry, puts it there and takes the entry of its own place: from then on the lanes
// are in the row's order, and its sums are those of the lanes before.  131072 rows of 32 float32 entries, a row a wave and
// entry by entry over lists: 148 us.

// Over the lanes of a group of G, its first one `base` in the wave.
template <int G>
struct Lanes {
  int lane, base;
  __device__ __forceinline__ Lanes() : lane(threadIdx.x % G), base((threadIdx.x & 63) / G * G) {}
  template <typename X>
  __device__ __forceinline__ X at(X x, int i) const {
    return __shfl(x, base + i, 64);
  }
  __device__ __forceinline__ int count(bool is) const {
    return __popcll(__ballot(is) >> base & (G == 64 ? ~0ull : (1ull << G % 64) - 1));
  }
  // The sum over the lanes up to and with this one.
  __device__ __forceinline__ uint64_t running_sum(uint64_t x) const {
    const auto add = [&](uint64_t y, int step) { x += G >= 16 || lane >= step ? y : 0; };
    add(from_lower<0x111>(x), 1);
    add(from_lower<0x112>(x), 2);
    if constexpr (G > 4) add(from_lower<0x114>(x), 4);
    if constexpr (G > 8) add(from_lower<0x118>(x), 8);
    if constexpr (G > 16) x += from_lower<0x142, 0xa>(x);
    if constexpr (G > 32) x += from_lower<0x143, 0xc>(x);
    return x;
  }
};

template <typename T, int G, bool RECORD>
__global__ __launch_bounds__(256) void narrow_kernel(const ChooseArgs a) {
  constexpr int ROWS = 256 / G, PITCH = G + 1;  // (rows side by side start in different banks)
  __shared__ uint64_t places[ROWS * PITCH];
  const Lanes<G> lanes;
  const int lane = lanes.lane;
  const int64_t first = int64_t(blockIdx.x) * ROWS + threadIdx.x / G;
  const bool in = first < a.rows;  // (every lane takes part: rows past the end are the last one again)
  const int64_t r = in ? first : int64_t(a.rows) - 1;
  uint64_t *mine = places + threadIdx.x / G * PITCH;
  float z = -INFINITY;
  if (lane < a.width && (!a.mask || a.mask[r * a.ld_mask + lane]))
    z = to_f32(static_cast<const T *>(a.logits)[r * a.ld_logits + lane]);
  float top = lanes_join<G>(z, larger);
  const bool nan = top != top, none = top == -INFINITY;
  if (top == INFINITY) z = z == INFINITY ? 0.f : -INFINITY, top = 0;
  if (nan || none) z = -INFINITY, top = 0;
  // Into the row's order.
  uint64_t place = place_of(z, lane);
  mine[lane] = place;
  wave_sync();
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < G; ++j) rank += mine[j] > place;  // (all different: an index is in each)
  wave_sync();
  mine[rank] = place;
  wave_sync();
  place = mine[lane];
  z = value_at(place);
  const int legal = lanes.count(z > -INFINITY);
  if constexpr (RECORD) {
    const double inverse = 1 / a.temperature.value;
    const bool held = lane < a.k && lane < legal;
    const float next = lanes.at(z, min(a.k, G - 1));  // the largest of the others, where there are any
    const bool rest_there = a.k < legal;
    const Share weigh(rest_there ? next : 0.f, inverse);
    const double x = (double(z) - double(top)) * inverse;
    const double rest = lanes_join<G>(lane >= a.k && lane < legal ? double(weigh(z)) : 0.0, Add{});
    const double held_sum = lanes_join<G>(held ? exp_of(x) : 0.0, Add{});
    const double gap = (double(weigh.base) - double(top)) * inverse;
    const double log_total = log_of(held_sum + (rest_there ? rest * exp_of(gap) : 0.0));
    const float absent = nan ? NAN : -INFINITY;
    if (!in) return;
    for (int i = lane; i < a.k; i += G) {  // (one turn where k is up to G: those behind are absent)
      const bool there = i == lane && held;
      a.log_probs[r * a.k + i] = there ? float(x - log_total) : absent;
      a.indices[r * a.k + i] = there ? index_at(place) : -1;
    }
    if (lane == 0) a.log_rest[r] = rest_there ? float(gap + log_of(rest) - log_total) : absent;
  } else {
    const Controls c(a, r);
    const bool bad = nan || !(c.temperature >= 0), greedy = c.temperature == 0;
    const Weights weight(top, greedy || bad ? 1.0 : c.temperature, a.scale);
    const uint64_t w = weight(z), upto = lanes.running_sum(w), before = upto - w;
    uint64_t kept = lanes.at(upto, (c.most > 0 && c.most < G ? int(c.most) : G) - 1);
    if (c.p < 1) {
      const uint64_t limit = c.limit(kept);
      kept = min(kept, lanes.at(upto, max(lanes.count(before < limit), 1) - 1));
    }
    const uint64_t bound = c.bound();
    if (bound > 1) kept = min(kept, lanes.at(upto, max(lanes.count(w >= bound), 1) - 1));
    if (c.least > 1) kept = c.one;
    const uint64_t sum = c.target(kept);
    const bool chosen = bad || none || greedy ? lane == 0 : before < sum && sum <= upto;
    if (!in || !chosen) return;
    a.actions[r] = bad || none ? -1 : index_at(place);
    a.log_probs[r] = bad ? NAN : none || greedy ? 0.f : c.log_share(z, top, kept, a.scale);
  }
}

// ---- kernels -------------------------------------------------------------------------------------------------------

// BYTES: of LDS for a row; 0: it is read again for each pass.  The record's blocks of 256 lanes fit a SIMD six times with a
// few registers less than they would take; fp16's then spill 9, and gain as much.  us with four and six waves, the 8 and the
// 128 largest: 8192 x 2048 bf16 48 80 and 44 73, fp16 48 81 and 43 74, fp32 47 80 and 43 74; 32768 x 1500 fp16 179 338 and
// 160 309.  Sampling's would spill 69.
template <typename T, int G, int BYTES, bool RECORD>
__global__ __launch_bounds__((G > 256 ? G : 256), RECORD && G == 256 ? 6 : 4) void choose_kernel(const ChooseArgs a) {
  constexpr int ROWS = G > 256 ? 1 : 256 / G;
  __shared__ Shared<G> shared[ROWS];
  const int in_block = G < 256 ? __builtin_amdgcn_readfirstlane(threadIdx.x / G) : 0;
  const int64_t r = int64_t(blockIdx.x) * ROWS + in_block;
  if (r >= a.rows) return;  // (whole groups; a group's barriers are its own wave's, or its own block's)
  Group<G> group(shared[in_block]);
  const T *logits = static_cast<const T *>(a.logits) + r * a.ld_logits;
  const uint8_t *legal = a.mask ? a.mask + r * a.ld_mask : nullptr;
  const auto run = [&](auto row) {
    if constexpr (RECORD)
      top_row(a, r, row, group);
    else
      sample_row(a, r, row, group);
  };
  if constexpr (BYTES > 0) {
    using Row = InLds<T, G, BYTES>;
    __shared__ typename Row::Vector held[ROWS][Row::VECTORS];
    run(Row(held[in_block], logits, legal, a.width));
  } else {
    run(Read<T, G>(logits, legal, a.width));
  }
}

struct Launch {
  void (*kernel)(ChooseArgs);
  int rows, threads;  // rows a block takes
};

template <typename T, int G, int BYTES, bool RECORD>
Launch launch_as() {
  return {choose_kernel<T, G, BYTES, RECORD>, G > 256 ? 1 : 256 / G, G > 256 ? G : 256};
}

template <typename T, int G, bool RECORD>
Launch narrow_as() {
  return {narrow_kernel<T, G, RECORD>, 256 / G, 256};
}

// The fewest lanes and the least LDS that a row fits: us as chosen and by the next one (no filter, top_p, the 8 largest),
//   131072 x 4 bf16       7.6   8.2   9.0 and  11.8  12.6  11.2     32768 x 1024 bf16  70  93  56 and 189 236 166
//   131072 x 16 fp32       21    22    23 and    40    42    43      8192 x 4096 fp32  70  88  47 and 123 154 130
//   131072 x 64 bf16       92    95    98 and   164   207   164      1024 x 32768 bf16 52  64  35 and  72  86  67
//    65536 x 256 bf16      87   114    83 and   100   129    89       910 x 36864 fp32 84 101  67 and  95 119  76
// Rows of 640 bytes to 1 KB have two entries a lane no longer: 65536 x 160 fp32 so 87 111 81, with them 90 116 86.
// fp16 goes as bf16: 131072 x 64 88 93 95 and 146 193 156, 32768 x 1024 68 90 53 and 191 238 146, 8192 x 8192 96 123 57 and
// 146 190 137, 1024 x 32768 52 63 32 and 71 86 59; 910 x 73728 119 150 80 and, read again, 133 171 78.
template <typename T, bool RECORD>
Launch launch_of(int width) {
  if (width <= 4) return narrow_as<T, 4, RECORD>();
  if (width <= 8) return narrow_as<T, 8, RECORD>();
  if (width <= 16) return narrow_as<T, 16, RECORD>();
  if (width <= 32) return narrow_as<T, 32, RECORD>();
  if (width <= 64) return narrow_as<T, 64, RECORD>();
  const int bytes = width * int(sizeof(T));
  if (bytes < 640) return launch_as<T, 64, 640, RECORD>();
  if (bytes <= 2048) return launch_as<T, 64, 2048, RECORD>();
  if (bytes <= 16384) return launch_as<T, 256, 16384, RECORD>();
  if (bytes <= 65536) return launch_as<T, 512, 65536, RECORD>();
  if (bytes <= 147456) return launch_as<T, 1024, 147456, RECORD>();
  return launch_as<T, 1024, 0, RECORD>();
}

template <bool RECORD>
void launch(const ChooseArgs &a, int dtype, hipStream_t stream) {
  const Launch l = dtype == CG_F32    ? launch_of<float, RECORD>(a.width)
                   : dtype == CG_BF16 ? launch_of<bf16, RECORD>(a.width)
                                      : launch_of<f16, RECORD>(a.width);
  const int64_t blocks = (int64_t(a.rows) + l.rows - 1) / l.rows;
  CG_REQUIRE(blocks * l.threads < int64_t(1) << 32, CG_ERR_UNSUPPORTED, "more rows than a launch has threads for");
  l.kernel<<<unsigned(blocks), l.threads, 0, stream>>>(a);
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
