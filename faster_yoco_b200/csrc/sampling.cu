// Sampling of one token for each row of logits from one uniform number a row: temperature, top-k, top-p, min-p.
//
// With w_i = exp((x_i - max) / T) the candidates, in descending order of x (ties: lowest index), are cut to the first k,
// to the shortest prefix with at least p of the weight left and to w_i >= min_p; the token is the first kept index whose
// running weight in index order passes u times the kept weight.
//
// No sort of the vocabulary. A cluster of 1 to 8 CTAs has a row, each CTA a contiguous slice, each warp a contiguous
// segment of it, so that running weights in index order are sums of segments. Passes over the row (the first from memory,
// the others from L2):
//   1  the largest logit, overall and of each thread
//   2  the weight of each segment, where a filter needs the whole vocabulary's (top-p without top-k, or no filter)
//   3  the candidates above a bound that no cut can pass: k-th largest of a CTA's thread maxima (k elements reach it);
//      (1 - p) Z / V (the tail from the p-cut on weighs at least (1 - p) Z and has at most V elements); min_p. They are
//      usually a few hundred: one CTA ranks them in shared memory, cuts and draws.
//   Otherwise the cut is found by a radix search over the order-preserving 32-bit image of the logits, with histograms of
//   counts (top-k) or weights (top-p) in steps of 11 bits, and the draw goes by segment sums.
//   A CTA's bound for top-k is its own slice's, so a row's list has at least CTAs x k candidates, of which it holds 512:
//   with 8 CTAs (one or 16 rows of 100,288) k = 50 takes 21 and 32 us and k = 64 takes 85 and 122; with 4 (64 rows)
//   k = 100 takes 39 and k = 128 takes 122; with one (256 rows) k = 200 takes 49 and k = 500 takes 223.
//
// Tokens are decided by comparing sums over the whole vocabulary, so weights are evaluated to 2^-48 in 64 bits and
// summed in 64 bits: histograms as integers in a fixed point whose 62 bits the weight of all candidates fills, the rest in
// floating point in a fixed order.
//
// Measured (B200): 64 rows of 100,288 bf16 logits, top-k and top-p, 23 us (0.6 TB/s; the read itself takes 2); 256 rows
// without a filter 73 us, bound by the 64-bit exponentials (about 47 instructions a logit, 12 of them 64-bit at 60 a clock
// and SM); one row with top-p 18 us, bound by cluster barriers (1.5 us each) and latency. CTAs a row at 64 rows: 1 / 2 /
// 4 / 8 take 29 / 24 / 22 / 53 us, at one row 53 / 37 / 26 / 18 us, at 400 rows 62 us with one and 152 with two. A radix
// row takes about 80 us on one CTA: 400 rows of 50,001 with settings of their own take 56 us, or 140 where such a row
// starts last (two seeds of twelve).
#include <ATen/ATen.h>
#include <c10/util/Optional.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common/host.h"
#include "common/ptx.cuh"

namespace fyb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kGranules = 8;        // pieces of a warp's segment whose weights are kept
constexpr int kList = kThreads;     // candidates of the short list: one a thread
constexpr int kGuess = 192;         // elements that a first look at a top-p cut is content with
constexpr int kBinBits = 11;        // of a radix step
constexpr uint32_t kFull = 0xffffffffu;

struct SampleParams {
  const void* logits;
  int64_t ld;                // row stride (elements)
  int V;
  int chunks;                // 8-element chunks of a CTA's slice
  const float* u;
  const float* temperature;  // per row, or null: temperature_all
  const void* top_k;         // per row (int32 or int64), or null
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int64_t top_k_all;
  int top_k_64;
  int64_t* token;
  float* logprob;            // or null
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// order-preserving image of a candidate; 0 for -inf and NaN, which are never drawn. Adding zero turns -0 into +0, which
// compare as equal.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (x > -INFINITY) ? k : 0u;       // false for -inf and for NaN
}

__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// w = 2^(t / 32) for t = 32 log2(e) (x - max) / T <= 0, by a table of 2^(j / 32) and a polynomial on |r| <= 1/2 (the
// table-driven method of P. T. P. Tang, 1989): 2^(r / 32) = 1 + r (c1 + r (c2 + ...)), c_i = (ln 2 / 32)^i / i!; the
// remainder after r^5 is below 2^-48. The table lies in the lanes of the warp (lane j: 2^(j / 32)) and is read by
// shuffles: all lanes call.
struct Weight {
  double top, scale, table;  // largest logit (finite), 32 log2(e) / T, this lane's 2^(lane / 32)
  float half, lowest;        // -max / 2; the (x - max) / 2 of a weight of 2^-1000
  uint32_t kmax;

  __device__ __forceinline__ void init(uint32_t largest, float t) {
    kmax = largest;
    const float topf = value_of(largest);
    top = static_cast<double>(topf);
    scale = 46.166241308446828384 / static_cast<double>(t);
    half = -0.5f * topf;
    lowest = fmaxf(static_cast<float>(-16000.0 / scale), -3.402823466e38f);
  }
  // whether a logit has a weight: not -inf or NaN, not below 2^-1000. It goes by the difference of the logits, halved so
  // that it stays finite: one rounding of what value() evaluates, so that neighbours of the largest are told apart at
  // any temperature (x scale - max scale in 32 bits is off by thousands where max / T is large, and the exponent field
  // of a weight below 2^-1022 wraps).
  __device__ __forceinline__ bool some(float x) const { return fmaf(x, 0.5f, half) >= lowest; }
  // weight of a logit that has one, exactly 1 for the largest; anything for others
  __device__ __forceinline__ double value(float x) const {
    constexpr double kRound = 6755399441055744.0;        // 1.5 x 2^52: adding it rounds to an integer
    constexpr double l = 0.021660849392498290;           // ln 2 / 32
    const double d = static_cast<double>(x) - top;
    const double z = fma(d, scale, kRound);
    const double r = fma(d, scale, kRound - z);
    const int n = __double2loint(z);
    const int lo = __shfl_sync(kFull, __double2loint(table), n);           // (of the index the low five bits count)
    const int hi = __shfl_sync(kFull, __double2hiint(table), n);
    double q = fma(r, l * l * l * l * l / 120, l * l * l * l / 24);
    q = fma(q, r, l * l * l / 6);
    q = fma(q, r, l * l / 2);
    q = fma(q, r, l);
    const double b = __hiloint2double(hi + ((n << 15) & 0xfff00000), lo);
    return fma(b * r, q, b);
  }
  __device__ __forceinline__ double operator()(float x) const {
    const double w = value(x);
    return some(x) ? w : 0.0;
  }
};

// Eight logits of a row: chunk c holds elements 8 c - off .. 8 c - off + 7, where off brings the row to a 16-byte boundary;
// -inf outside the row.
template <typename T>
struct Row {
  const T* x;
  int V, off, chunks;
  bool only_inf = false;     // the largest logit is +inf: these count as 0, all others as -inf

  __device__ __forceinline__ Row(const SampleParams& p, int64_t n)
      : x(reinterpret_cast<const T*>(p.logits) + n * p.ld), V(p.V) {
    off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    chunks = (V + off + 7) / 8;
  }
  __device__ __forceinline__ int index(int c, int j) const { return 8 * c - off + j; }
  __device__ __forceinline__ bool whole(int c) const { return c < chunks && 8 * c >= off && 8 * c - off + 8 <= V; }
  // a chunk as it is stored, and its values: fetch() can run ahead
  struct Raw {
    uint4 a[sizeof(T) / 2];
  };
  __device__ __forceinline__ Raw fetch(int c) const {
    Raw raw{};
    if (whole(c)) {
      const uint4* src = reinterpret_cast<const uint4*>(x + 8 * c - off);
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k) raw.a[k] = src[k];
    }
    return raw;
  }
  __device__ __forceinline__ void load(int c, float (&v)[8]) const { values(c, fetch(c), v); }
  __device__ __forceinline__ void values(int c, const Raw& raw, float (&v)[8]) const {
    const int i = 8 * c - off;
    if (whole(c)) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          v[4 * k] = __uint_as_float(raw.a[k].x), v[4 * k + 1] = __uint_as_float(raw.a[k].y);
          v[4 * k + 2] = __uint_as_float(raw.a[k].z), v[4 * k + 3] = __uint_as_float(raw.a[k].w);
        }
      } else {
        const uint32_t w[4] = {raw.a[0].x, raw.a[0].y, raw.a[0].z, raw.a[0].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 f;
          if constexpr (std::is_same<T, __half>::value)
            f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
          else
            f = unpack_bf16(w[k]);
          v[2 * k] = f.x;
          v[2 * k + 1] = f.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = -INFINITY;
      if (c < chunks) {                  // at the ends of the row
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i + j >= 0 && i + j < V) v[j] = to_float(x[i + j]);
      }
    }
    if (only_inf) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] == INFINITY ? 0.f : -INFINITY;
    }
  }
  // the larger of m and the chunk's largest logit, NaN aside
  __device__ __forceinline__ float max_with(int c, float m) const {
    if constexpr (sizeof(T) == 2) {
      if (whole(c)) {
        const uint4 a = *reinterpret_cast<const uint4*>(x + 8 * c - off);
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2* w = reinterpret_cast<const T2*>(&a);
        const T2 y = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
        return fmaxf(m, fmaxf(to_float(y.x), to_float(y.y)));
      }
    }
    float v[8];
    load(c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, v[j]);
    return m;
  }
};

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(kFull, v); }

// What is kept of a row: everything, weights of at least min_p, or what a cut (and min_p) leaves
enum Mode : int { kAll, kByWeight, kByCut };

struct Cut {
  uint32_t key;         // images above are kept, those below are not
  uint32_t ties;        // how many images equal to `key` are kept (the first ones by index)
};

struct Shared {
  uint32_t warp_best[kWarps];
  uint32_t best, first;                // of this CTA: largest image; ~(lowest index that has the row's largest)
  uint32_t bound;                      // of this CTA
  double part[kWarps][kGranules];      // weight of each granule
  double part_sum[kWarps];
  double sum;                          // of this CTA
  uint32_t count[kWarps];
  uint32_t total_count;                // of this CTA (candidates, or ties)
  bool done;                           // a token was drawn from the list
  uint32_t hist_lo[1 << kBinBits], hist_hi[1 << kBinBits];
  uint64_t scan[kWarps];
  uint64_t found[3];
  // the short list, in the CTA that draws from it
  uint32_t key[kList], idx[kList];
  double w[kList];
  uint32_t listed;                     // candidates met
  uint32_t by_key[kList];              // rank by index, by rank in descending order
  uint32_t by_idx[kList];              // index, by rank by index (as the weights)
};

// What the CTAs of a row know of one another goes through a field of Shared that each writes once before a cluster barrier
// and that is written again only behind another one.
template <typename T>
struct Sampler {
  const SampleParams& p;
  Shared& sh;
  cg::cluster_group cluster;
  Row<T> row;
  Weight weight;
  int rank, ctas, warp, lane;
  int c0, c1, per, iters, step;        // this warp's chunks; chunks and iterations a warp, iterations of a granule
  double unit = 1.0;                   // fixed-point units of a weight of 1

  __device__ __forceinline__ Sampler(const SampleParams& p_, Shared& s, int64_t n)
      : p(p_), sh(s), cluster(cg::this_cluster()), row(p_, n) {
    rank = cluster.block_rank();
    ctas = cluster.num_blocks();
    warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    per = (p.chunks + kWarps - 1) / kWarps;
    iters = (per + 31) / 32;
    step = (iters + kGranules - 1) / kGranules;
    const int end = min((rank + 1) * p.chunks, row.chunks);
    c0 = min(rank * p.chunks + warp * per, end);
    c1 = min(c0 + per, end);
    weight.table = exp2(lane / 32.0);
  }
  __device__ __forceinline__ const Shared& of(int r) const {
    return ctas == 1 ? sh : *cluster.map_shared_rank(&sh, r);
  }
  __device__ __forceinline__ void sync() {
    if (ctas == 1)
      __syncthreads();
    else
      cluster.sync();
  }
  // chunk of this lane at an iteration, or one outside the row
  __device__ __forceinline__ int chunk(int it) const {
    const int c = c0 + it * 32 + lane;
    return c < c1 ? c : row.chunks;
  }

  // largest of a value over the row, through a field of Shared of its own
  __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t Shared::* field) {
    v = warp_max(v);
    __syncthreads();
    if (lane == 0) sh.warp_best[warp] = v;
    __syncthreads();
    v = warp_max(sh.warp_best[lane & (kWarps - 1)]);
    if (ctas == 1) return v;
    if (threadIdx.x == 0) sh.*field = v;
    cluster.sync();
    return warp_max(of(lane & (ctas - 1)).*field);
  }

  // image of the largest logit of this thread
  __device__ __forceinline__ uint32_t largest() {
    float m = -INFINITY;
#pragma unroll 8
    for (int it = 0; it < iters; ++it) m = row.max_with(chunk(it), m);      // 64 KB of a CTA's slice in flight
    return key_of(m);
  }

  // lowest index with the largest image
  __device__ __forceinline__ uint32_t first_of(uint32_t kmax, uint32_t thread_key) {
    uint32_t mine = 0;
    if (thread_key == kmax) {
#pragma unroll 1
      for (int it = 0; it < iters && mine == 0; ++it) {
        float v[8];
        row.load(chunk(it), v);
#pragma unroll
        for (int j = 7; j >= 0; --j)
          if (key_of(v[j]) == kmax) mine = ~static_cast<uint32_t>(row.index(chunk(it), j));
      }
    }
    __syncwarp();
    return ~row_max(mine, &Shared::first);
  }

  // An image that at least k elements of the CTA's slice reach: the k-th largest of its thread maxima (k <= kThreads), bit
  // by bit the largest image that k threads reach, to 18 bits (all that a 16-bit type has but for one of fp16's; a
  // bound that is too low by less than 2^-9 finds a few more candidates).
  __device__ __forceinline__ uint32_t bound_of_k(uint32_t thread_key, int k) {
    uint32_t b = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 14; --bit) {
      const uint32_t t = b | (1u << bit);
      if (__syncthreads_count(thread_key >= t) >= k) b = t;
    }
    return max(b, 1u);
  }
  // the largest of the CTAs' bounds
  __device__ __forceinline__ uint32_t shared_bound(uint32_t b) {
    if (ctas == 1) return b;
    if (threadIdx.x == 0) sh.bound = b;
    cluster.sync();
    return warp_max(of(lane & (ctas - 1)).bound);
  }

  // what is kept: above the cut, and the first of its ties by index; weights of at least min_w
  struct Kept {
    Cut cut;
    double min_w;
  };

  // Weights of what is kept among the eight logits of each lane (w[j] = 0 for the others) and their sum, in index order.
  // tie_rank counts the ties of this warp's segment met so far. All lanes call.
  template <Mode kMode>
  __device__ __forceinline__ double weigh(const float (&v)[8], const Kept& kept, uint32_t& tie_rank, double (&w)[8]) {
    double s = 0.0;
    if constexpr (kMode != kByCut) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double x = weight.value(v[j]);
        w[j] = 0.0;
        if (weight.some(v[j]) && (kMode == kAll || x >= kept.min_w)) {
          w[j] = x;
          s += x;
        }
      }
      return s;
    }
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine += key_of(v[j]) == kept.cut.key ? 1u : 0u;
    uint32_t before = 0;
    if (__any_sync(kFull, mine != 0)) {
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t c = __shfl_up_sync(kFull, inc, o);
        if (lane >= o) inc += c;
      }
      before = tie_rank + inc - mine;
      tie_rank += __shfl_sync(kFull, inc, 31);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = 0.0;
      const uint32_t k = key_of(v[j]);
      bool keep = k > kept.cut.key;
      if (k == kept.cut.key) keep = before++ < kept.cut.ties;
      if (!__any_sync(kFull, keep)) continue;
      const double x = weight(v[j]);
      if (keep && x >= kept.min_w) w[j] = x;
      s += w[j];
    }
    return s;
  }

  // ties of the cut before this warp's segment
  __device__ __forceinline__ uint32_t ties_before(const Cut& cut) {
    uint32_t n = 0;
#pragma unroll 2
    for (int it = 0; it < iters; ++it) {
      float v[8];
      row.load(chunk(it), v);
#pragma unroll
      for (int j = 0; j < 8; ++j) n += key_of(v[j]) == cut.key ? 1u : 0u;
    }
    n = warp_sum(n);
    if (lane == 0) sh.count[warp] = n;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += sh.count[i];
      all += sh.count[i];
    }
    if (ctas > 1) {
      if (threadIdx.x == 0) sh.total_count = all;
      cluster.sync();
      for (int r = 0; r < rank; ++r) before += of(r).total_count;
    }
    return before;
  }

  // weight of every granule; returns the row's
  template <Mode kMode>
  __device__ __forceinline__ double sums(const Kept& kept, uint32_t ties0) {
    uint32_t tie_rank = ties0;
    double mine = 0.0;
#pragma unroll 1
    for (int g = 0; g < kGranules && g * step < iters; ++g) {
      double s = 0.0;
      const int end = min((g + 1) * step, iters);
      typename Row<T>::Raw raw[2] = {row.fetch(chunk(g * step)), row.fetch(chunk(g * step + 1))};
#pragma unroll 1
      for (int it = g * step; it < end; ++it) {
        float v[8];
        double w[8];
        row.values(chunk(it), raw[0], v);
        raw[0] = raw[1];
        raw[1] = row.fetch(chunk(it + 2));       // two chunks are on their way meanwhile
        s += weigh<kMode>(v, kept, tie_rank, w);
      }
      s = warp_sum(s);
      if (lane == 0) sh.part[warp][g] = s;
      mine += s;
    }
    if (lane == 0) sh.part_sum[warp] = mine;
    __syncthreads();
    double s = warp_sum(lane < kWarps ? sh.part_sum[lane] : 0.0);
    if (ctas == 1) return s;
    if (threadIdx.x == 0) sh.sum = s;
    cluster.sync();
    return warp_sum(lane < ctas ? of(lane).sum : 0.0);
  }

  // first of n parts whose running sum (from `before`) passes r, the last with any weight if rounding hides it
  template <typename F>
  __device__ __forceinline__ int pass(int n, F part, double r, double& before) {
    int last = 0;
    double at_last = before;
    for (int i = 0; i < n; ++i) {
      const double s = part(i);
      if (s > 0.0) {
        last = i;
        at_last = before;
      }
      if (before + s > r) return i;
      before += s;
    }
    before = at_last;
    return last;
  }

  // draws by the granules' weights (sums() of the same `kept` came before)
  template <Mode kMode>
  __device__ __forceinline__ void draw(int64_t n, const Kept& kept, uint32_t ties0, double total) {
    const double r = fmin(fmax(static_cast<double>(p.u[n]), 0.0), 1.0 - 0x1p-24) * total;
    double before = 0.0;
    if (ctas > 1 && pass(ctas, [&](int i) { return of(i).sum; }, r, before) != rank) return;
    if (pass(kWarps, [&](int i) { return sh.part_sum[i]; }, r, before) != warp) return;
    const int g = pass((iters + step - 1) / step, [&](int i) { return sh.part[warp][i]; }, r, before);
    uint32_t tie_rank = ties0;
    float v[8];
    double w[8];
    if (kMode == kByCut)                         // ties of the granules before
      for (int it = 0; it < g * step; ++it) {
        row.load(chunk(it), v);
        uint32_t t = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) t += key_of(v[j]) == kept.cut.key ? 1u : 0u;
        tie_rank += warp_sum(t);
      }
    int found = -1;
    double found_w = 0.0;
    for (int it = g * step; it < min((g + 1) * step, iters); ++it) {
      row.load(chunk(it), v);
      const double mine = weigh<kMode>(v, kept, tie_rank, w);
      double inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double c = __shfl_up_sync(kFull, inc, o);
        if (lane >= o) inc += c;
      }
      const uint32_t hit = __ballot_sync(kFull, before + inc > r && mine > 0.0);
      const uint32_t some = __ballot_sync(kFull, mine > 0.0);
      if (some != 0) {
        // the first lane that passes r; none yet: the last one with weight so far
        const int l = hit != 0 ? __ffs(hit) - 1 : 31 - __clz(some);
        const double base = before + __shfl_sync(kFull, inc - mine, l);
        int at = -1;
        double at_w = 0.0;
        if (lane == l) {
          double run = base;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool open = at < 0 || run <= r;
            run += w[j];
            if (w[j] > 0.0 && open) {
              at = row.index(chunk(it), j);
              at_w = w[j];
            }
          }
        }
        found = __shfl_sync(kFull, at, l);
        found_w = __shfl_sync(kFull, at_w, l);
      }
      if (hit != 0) break;
      before += __shfl_sync(kFull, inc, 31);
    }
    if (lane == 0) write(n, found, found_w, total);
  }

  __device__ __forceinline__ void write(int64_t n, int index, double w, double total) const {
    p.token[n] = index;
    if (p.logprob != nullptr) p.logprob[n] = static_cast<float>(log(w / total));
  }

  // Candidates of image >= bound (a CTA's own) to the first CTA's list, in no order; returns how many there are (more than
  // kList: the list is short of some)
  __device__ __forceinline__ uint32_t gather(uint32_t bound, uint32_t thread_key) {
    Shared& to = ctas == 1 ? sh : *cluster.map_shared_rank(&sh, 0);
    const bool has = thread_key >= bound;
    if (__any_sync(kFull, has)) {
      uint32_t where = 0;                        // iterations (mod 32) that have candidates
      if (has && *static_cast<volatile uint32_t*>(&to.listed) <= kList) {
#pragma unroll 8
        for (int it = 0; it < iters; ++it)
          if (key_of(row.max_with(chunk(it), -INFINITY)) >= bound) where |= 1u << (it & 31);
      }
      __syncwarp();
      const uint32_t any = __reduce_or_sync(kFull, where);
#pragma unroll 1
      for (int it = 0; it < iters; ++it) {
        if ((any >> (it & 31) & 1u) == 0) continue;
        float v[8];
        row.load(where >> (it & 31) & 1u ? chunk(it) : row.chunks, v);
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine += key_of(v[j]) >= bound ? 1u : 0u;
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t c = __shfl_up_sync(kFull, inc, o);
          if (lane >= o) inc += c;
        }
        uint32_t at = 0;
        if (lane == 31 && inc > 0) at = atomicAdd(&to.listed, inc);
        at = __shfl_sync(kFull, at, 31);
        if (at > kList) break;                   // too many, whatever follows
        at += inc - mine;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t k = key_of(v[j]);
          if (k >= bound) {
            if (at < kList) {
              to.key[at] = k;
              to.idx[at] = static_cast<uint32_t>(row.index(chunk(it), j));
            }
            ++at;
          }
        }
      }
    }
    sync();
    return to.listed;
  }

  // inclusive sum over the threads of the block before and with this one, in a fixed order; only the first `used` warps
  // have anything but zeros
  template <typename V>
  __device__ __forceinline__ V block_scan(V v, V* scratch, int used = kWarps) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V c = __shfl_up_sync(kFull, v, o);
      if (lane >= o) v += c;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    V before = 0;
#pragma unroll 1
    for (int i = 0; i < min(warp, used); ++i) before += scratch[i];
    return before + v;
  }

  // Cuts and draws from the list of n candidates, which holds everything that can be kept (sure), or all larger images of
  // what it holds: then false if their weight does not reach the share. z: weight of what top_p is a share of, or 0 where
  // that is the first k candidates.
  __device__ __forceinline__ bool draw_list(int64_t n_row, int n, int k, float top_p, double min_w, double z, bool sure) {
    const int t = threadIdx.x, used = (n + 31) / 32;
    const bool have = t < n;
    if (warp < used) {
      const uint32_t key = have ? sh.key[t] : 0u, idx = have ? sh.idx[t] : 0u;
      const double w = weight(have ? value_of(key) : -INFINITY);
      // ranks in descending order (ties are won by the lower index) and by index
      int rank_k = 0, rank_i = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const uint32_t o = sh.key[j], i = sh.idx[j];
        rank_i += i < idx ? 1 : 0;
        rank_k += (o > key || (o == key && i < idx)) ? 1 : 0;
      }
      if (have) {
        sh.by_key[rank_k] = static_cast<uint32_t>(rank_i);
        sh.w[rank_i] = w;
        sh.by_idx[rank_i] = idx;
      }
    }
    __syncthreads();
    // in the order of ranks: thread t looks at the candidate of rank t
    const int first = k > 0 ? min(k, n) : n;
    const int who = have ? static_cast<int>(sh.by_key[t]) : 0;
    const double wr = t < first ? sh.w[who] : 0.0;
    bool keep = t < first && wr >= min_w;
    if (top_p < 1.f) {
      const double inc = block_scan(wr, sh.part_sum, used);
      if (t == kThreads - 1) sh.sum = inc;
      __syncthreads();
      if (!sure && sh.sum < static_cast<double>(top_p) * z) return false;
      keep = keep && (t == 0 || inc - wr < static_cast<double>(top_p) * (z > 0.0 ? z : sh.sum));
    }
    __syncthreads();
    if (have && !keep) sh.w[who] = 0.0;
    __syncthreads();
    // in index order
    const double wi = have ? sh.w[t] : 0.0;
    const double run = block_scan(wi, sh.part_sum, used);
    if (t == kThreads - 1) sh.sum = run;
    __syncthreads();
    const double total = sh.sum;
    const double r = fmin(fmax(static_cast<double>(p.u[n_row]), 0.0), 1.0 - 0x1p-24) * total;
    // first with run > r; rounding cannot hide the last one, whose running sum is `total` itself
    const uint32_t m = __ballot_sync(kFull, wi > 0.0 && run > r);
    if (lane == 0) sh.count[warp] = m;
    __syncthreads();
    if (t == 0) {
#pragma unroll 1
      for (int i = 0; i < used; ++i) {
        if (sh.count[i] == 0) continue;
        const int at = 32 * i + __ffs(sh.count[i]) - 1;
        write(n_row, static_cast<int>(sh.by_idx[at]), sh.w[at], total);
        break;
      }
    }
    return true;
  }

  __device__ __forceinline__ uint64_t fixed(double w) const { return static_cast<uint64_t>(__double2ll_rn(w * unit)); }
  // a unit in which weights of `total` (1 or more) together take 62 bits: what V of them lose by rounding is below 2^-62 V of
  // the total, however many the small ones are (V weights of 1 would leave 2^-40 for one of 2^22 logits)
  __device__ __forceinline__ void set_unit(double total) {
    const int e = (__double2hiint(total) >> 20) - 1022;        // total < 2^e
    unit = __hiloint2double((1023 + 62 - e) << 20, 0);
  }

  // The image at which the amount of larger and equal images first reaches `target`: 1 for each candidate that the cut
  // keeps, or its fixed-point weight. Steps of kBinBits over the images from `low` (> 0) up, which hold the answer.
  // above: the amount of larger images; at: the amount of that image.
  template <bool kWeights>
  __device__ uint32_t radix_find(const Cut& cut, uint32_t low, double target, uint64_t& above, uint64_t& at) {
    uint32_t base = low;
    int bits = 32 - __clz(weight.kmax - low);
    above = 0;
    at = 0;
    do {
      const int s = max(bits - kBinBits, 0);
      const int bins = 1 << (bits - s);
      __syncthreads();
      for (int i = threadIdx.x; i < bins; i += kThreads) sh.hist_lo[i] = sh.hist_hi[i] = 0;
      __syncthreads();
      auto add = [&](uint32_t bin, uint64_t a) {
        const uint32_t lo = static_cast<uint32_t>(a);
        uint32_t hi = static_cast<uint32_t>(a >> 32);
        const uint32_t old = atomicAdd(&sh.hist_lo[bin], lo);
        hi += old + lo < old ? 1u : 0u;
        if (hi != 0) atomicAdd(&sh.hist_hi[bin], hi);
      };
      for (int it = 0; it < iters; ++it) {
        float v[8];
        row.load(chunk(it), v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t k = key_of(v[j]);
          const uint64_t span = static_cast<uint64_t>(k - base) >> bits;       // bits may be 32
          const bool in = k > cut.key && k >= base && span == 0;
          if (!__any_sync(kFull, in)) continue;
          const uint64_t a = kWeights ? fixed(weight(v[j])) : 1;
          if (in) add((k - base) >> s, a);
        }
      }
      const double wt = weight(cut.key != 0 ? value_of(cut.key) : -INFINITY);
      if (rank == 0 && threadIdx.x == 0 && cut.ties > 0 && cut.key >= base &&
          (static_cast<uint64_t>(cut.key - base) >> bits) == 0)
        add((cut.key - base) >> s, kWeights ? cut.ties * fixed(wt) : cut.ties);
      sync();
      // thread t adds up four bins, from the top; sums over the CTAs, the same in each
      constexpr int kPer = (1 << kBinBits) / kThreads;
      uint64_t h[kPer], mine = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int bin = bins - 1 - (static_cast<int>(threadIdx.x) * kPer + j);
        h[j] = 0;
        if (bin >= 0)
          for (int r = 0; r < ctas; ++r)
            h[j] += static_cast<uint64_t>(of(r).hist_hi[bin]) << 32 | of(r).hist_lo[bin];
        mine += h[j];
      }
      const uint64_t inc = block_scan(mine, sh.scan);
      if (threadIdx.x == 0) sh.found[0] = ~0ull;
      __syncthreads();
      // the first thread whose sum reaches the target; the last with any amount if rounding hides it
      const bool reach = mine > 0 && static_cast<double>(above + inc) >= target &&
                         !(static_cast<double>(above + inc - mine) >= target);
      if (reach || (mine > 0 && static_cast<double>(above + inc) < target)) {
        const uint64_t order = (reach ? 0ull : 1ull << 32) | (reach ? threadIdx.x : kThreads - threadIdx.x);
        atomicMin(reinterpret_cast<unsigned long long*>(&sh.found[0]), static_cast<unsigned long long>(order));
      }
      __syncthreads();
      const uint64_t order = sh.found[0];
      const uint32_t winner = (order >> 32) == 0 ? static_cast<uint32_t>(order)
                                                 : kThreads - static_cast<uint32_t>(order & 0xffffffffu);
      if (threadIdx.x == winner) {
        uint64_t run = above + inc - mine, here = 0, before = run;
        int bin = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int b = bins - 1 - (static_cast<int>(threadIdx.x) * kPer + j);
          if (h[j] > 0 && (here == 0 || static_cast<double>(run) < target)) {
            bin = b;
            here = h[j];
            before = run;
          }
          run += h[j];
        }
        sh.found[1] = before;
        sh.found[2] = here;
        sh.scan[0] = static_cast<uint64_t>(bin);
      }
      __syncthreads();
      base += static_cast<uint32_t>(sh.scan[0]) << s;
      above = sh.found[1];
      at = sh.found[2];
      bits = s;
      sync();
    } while (bits > 0);
    return base;
  }

  __device__ __forceinline__ void run(int64_t n) {
    if (threadIdx.x == 0) sh.listed = 0;
    uint32_t thread_key = largest();
    uint32_t kmax = row_max(thread_key, &Shared::best);
    const float t = p.temperature != nullptr ? p.temperature[n] : p.temperature_all;
    const float mp = p.min_p != nullptr ? p.min_p[n] : p.min_p_all;
    if (kmax == 0 || !(t > 0.f) || !(mp <= 1.f)) {         // min_p above 1 leaves the largest alone
      const uint32_t at = kmax != 0 ? first_of(kmax, thread_key) : 0u;
      if (rank == 0 && threadIdx.x == 0) {
        p.token[n] = kmax == 0 ? -1 : static_cast<int64_t>(at);
        if (p.logprob != nullptr) p.logprob[n] = kmax == 0 ? -INFINITY : 0.f;
      }
      return;
    }
    if (value_of(kmax) == INFINITY) {
      row.only_inf = true;
      thread_key = thread_key == kmax ? key_of(0.f) : 0u;
      kmax = key_of(0.f);
    }
    weight.init(kmax, t);
    int64_t k64 = p.top_k_all;
    if (p.top_k != nullptr)
      k64 = p.top_k_64 ? reinterpret_cast<const int64_t*>(p.top_k)[n] : reinterpret_cast<const int*>(p.top_k)[n];
    const int k = k64 > 0 && k64 < p.V ? static_cast<int>(k64) : 0;
    const float tp = p.top_p != nullptr ? p.top_p[n] : p.top_p_all;
    const bool by_p = !(tp >= 1.f);
    const double share = by_p ? fmax(static_cast<double>(tp), 0.0) : 1.0;
    const double min_w = mp > 0.f ? static_cast<double>(mp) : 0.0;

    // images from `low` up hold everything that is kept; 1 is below all candidates
    uint32_t low = 1, guess = 1;
    double z = 0.0;
    const Kept all{Cut{0, 0}, 0.0};
    if (k > 0) {
      // a CTA's own: what is among the first k of the row is among the first k of its slice
      if (k <= kThreads) low = bound_of_k(thread_key, k);
    } else if (by_p) {
      z = sums<kAll>(all, 0);
      low = bound_of_weight((1.0 - share) * z / p.V);
      // that bound is far too low for a steep distribution: try what about kGuess elements reach, and see whether they
      // weigh enough
      guess = shared_bound(bound_of_k(thread_key, kGuess / ctas));
    }
    if (min_w > 0.0 && !(k > 0 && by_p)) low = max(low, bound_of_weight(min_w));
    // (decided alike by the CTAs of a row, which wait for one another in there)
    if ((k > 0 ? k <= kThreads : low > 1 || guess > 1) || p.V <= kList) {
      const bool sure = guess <= low;
      const uint32_t c = gather(max(low, guess), thread_key);
      if (c <= kList) {
        if (sure) {
          if (rank == 0)
            draw_list(n, static_cast<int>(c), k, by_p ? static_cast<float>(share) : 1.f, min_w, z, true);
          return;
        }
        if (rank == 0) {
          const bool done = draw_list(n, static_cast<int>(c), 0, static_cast<float>(share), min_w, z, false);
          if (threadIdx.x == 0) sh.done = done;
        }
        sync();
        if (of(0).done) return;
      }
    }
    Cut cut{0, 0};
    uint64_t above, at;
    if (k > 0) {
      const uint32_t key = radix_find<false>(cut, 1, static_cast<double>(k), above, at);
      const uint64_t left = static_cast<uint64_t>(k) - min(above, static_cast<uint64_t>(k));
      cut = Cut{key, static_cast<uint32_t>(min(left, at))};
    }
    if (by_p) {
      if (k > 0) {
        double sum = 0.0;
        for (int it = 0; it < iters; ++it) {
          float v[8];
          row.load(chunk(it), v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const double w = weight(v[j]);
            sum += key_of(v[j]) > cut.key ? w : 0.0;
          }
        }
        const double wt = weight(value_of(cut.key));
        sum = block_scan(sum, sh.part_sum);
        __syncthreads();
        if (threadIdx.x == kThreads - 1) sh.sum = sum;
        sync();
        z = cut.ties * wt;
        for (int r = 0; r < ctas; ++r) z += of(r).sum;
        low = cut.key;
      }
      set_unit(z);
      const double target = fmax(share * (z * unit), 1.0);       // the largest is always kept
      const uint32_t key = radix_find<true>(cut, low, target, above, at);
      const uint64_t w = fixed(weight(value_of(key)));
      uint64_t ties = 1;
      if (w > 0 && target > static_cast<double>(above)) {
        // smallest count with above + count w >= target, from a quotient that may be off by one
        const uint64_t have = at / w;
        ties = static_cast<uint64_t>((target - static_cast<double>(above)) / static_cast<double>(w));
        ties = ties > 1 ? ties - 1 : 1;
        while (ties < have && static_cast<double>(above + ties * w) < target) ++ties;
      }
      if (key == cut.key && cut.ties < ties) ties = cut.ties;
      cut = Cut{key, static_cast<uint32_t>(min(ties, static_cast<uint64_t>(0xffffffffu)))};
    }
    const Kept kept{cut, min_w};
    if (cut.key != 0) {
      const uint32_t ties0 = ties_before(cut);
      draw<kByCut>(n, kept, ties0, sums<kByCut>(kept, ties0));
    } else if (min_w > 0.0) {
      draw<kByWeight>(n, kept, 0, sums<kByWeight>(kept, 0));
    } else {
      draw<kAll>(n, kept, 0, sums<kAll>(kept, 0));
    }
  }

  // an image that every weight >= w reaches (rounded down by more than its own and the weights' rounding)
  __device__ __forceinline__ uint32_t bound_of_weight(double w) {
    const double x = weight.top + log2(w) * 32.0 / weight.scale;           // w = 0: -inf
    const float f = __double2float_rd(x - 1e-9 * (1.0 + fabs(x)));
    return max(key_of(f), 1u);                                             // NaN, -inf: all candidates
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  __shared__ Shared sh;
  Sampler<T> s(p, sh, blockIdx.x / cg::this_cluster().num_blocks());
  s.run(blockIdx.x / cg::this_cluster().num_blocks());
  s.sync();                            // a CTA's shared memory outlives the readers in its cluster
}

const void* row_param(const c10::optional<at::Tensor>& t, const at::Tensor& logits, at::ScalarType type,
                      const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  FYB_SUITS(t->device() == logits.device() && t->scalar_type() == type && t->dim() == 1 &&
                t->is_contiguous() && t->size(0) == logits.size(0),
            std::string("sample: ") + name);
  return t->data_ptr();
}

template <typename T>
void launch(const SampleParams& p, int64_t rows, int ctas) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = cur_stream();
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = ctas;
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  FYB_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, p));
  check_launch("sample");
}

}  // namespace

std::vector<at::Tensor> sample(const at::Tensor& logits, const at::Tensor& u,
                               const c10::optional<at::Tensor>& temperature, double temperature_all,
                               const c10::optional<at::Tensor>& top_k, int64_t top_k_all,
                               const c10::optional<at::Tensor>& top_p, double top_p_all,
                               const c10::optional<at::Tensor>& min_p, double min_p_all, bool want_logprob) {
  FYB_RANGE("fyb::sample");
  FYB_SUITS(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1),
            "sample: logits [N, V] with a contiguous last dim expected");
  const int64_t N = logits.size(0), V = logits.size(1);
  FYB_SUITS(V >= 1 && V < (1ll << 30) && N < (1ll << 27), "sample: sizes");
  FYB_SUITS(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf ||
                logits.scalar_type() == at::kFloat,
            "sample: bf16, fp16 or fp32 logits expected");
  c10::cuda::CUDAGuard guard(logits.device());
  SampleParams p{};
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  p.V = static_cast<int>(V);
  FYB_SUITS(u.device() == logits.device() && u.scalar_type() == at::kFloat && u.dim() == 1 && u.is_contiguous() &&
                u.size(0) == N,
            "sample: u");
  p.u = u.data_ptr<float>();
  p.temperature = static_cast<const float*>(row_param(temperature, logits, at::kFloat, "temperature"));
  p.top_p = static_cast<const float*>(row_param(top_p, logits, at::kFloat, "top_p"));
  p.min_p = static_cast<const float*>(row_param(min_p, logits, at::kFloat, "min_p"));
  p.top_k_64 = top_k.has_value() && top_k->defined() && top_k->scalar_type() == at::kLong;
  p.top_k = row_param(top_k, logits, p.top_k_64 ? at::kLong : at::kInt, "top_k");
  p.temperature_all = static_cast<float>(temperature_all);
  p.top_p_all = static_cast<float>(top_p_all);
  p.min_p_all = static_cast<float>(min_p_all);
  p.top_k_all = top_k_all;
  auto token = at::empty({N}, logits.options().dtype(at::kLong));
  at::Tensor logprob;
  if (want_logprob) logprob = at::empty({N}, logits.options().dtype(at::kFloat));
  p.token = token.data_ptr<int64_t>();
  p.logprob = want_logprob ? logprob.data_ptr<float>() : nullptr;
  if (N > 0) {
    // CTAs a row: as many as two an SM allow, up to 8, while a thread still has a chunk of its own
    const int64_t chunks = (V + 7 + 7) / 8;      // a row may start anywhere in its first chunk
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    int ctas = 1;
    while (ctas < kMaxCluster && N * ctas * 2 <= 2 * sms && chunks >= ctas * 2 * kThreads) ctas *= 2;
    p.chunks = static_cast<int>((chunks + ctas - 1) / ctas);
    if (logits.scalar_type() == at::kBFloat16)
      launch<__nv_bfloat16>(p, N, ctas);
    else if (logits.scalar_type() == at::kHalf)
      launch<__half>(p, N, ctas);
    else
      launch<float>(p, N, ctas);
  }
  return {token, logprob};
}

}  // namespace fyb
