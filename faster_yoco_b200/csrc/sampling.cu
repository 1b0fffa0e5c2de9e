// Sampling of one token for each row of logits from one uniform number a row: temperature, top-k, top-p, min-p.
//
// With w_i = exp((x_i - max) / T) the candidates, in descending order of x (ties: lowest index), are cut to the first k, to
// the shortest prefix with at least p of the weight left and to w_i >= min_p; the token is the first kept index whose
// running weight in index order passes u times the kept weight.
//
// No sort: every cut is a threshold (a value and how many of its ties, by index, are kept), found by a radix search
// over the order-preserving 32-bit image of the logits, most significant digit first, with a histogram of counts
// (top-k) or of weights (top-p) for each digit.
//
// Tokens are decided by comparing sums over the whole vocabulary, so weights are evaluated in 64 bits and summed as
// 64-bit integers (a fixed point that leaves room for V weights of at most 1): integer sums do not depend on the order
// of the additions, so neither the token nor its log-probability depends on how the row is divided.
#include <ATen/ATen.h>
#include <c10/util/Optional.h>
#include <cuda_fp16.h>

#include "common/host.h"
#include "common/ptx.cuh"

namespace fyb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kFull = 0xffffffffu;
constexpr double kLog2e64 = 1.4426950408889634074;
constexpr int64_t kNone = -1;

struct SampleParams {
  const void* logits;
  int64_t ld;                // row stride (elements)
  int64_t V;
  const float* u;
  const float* temperature;  // per row, or null: temperature_all
  const void* top_k;         // per row (int32 or int64), or null
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int64_t top_k_all;
  int top_k_64;
  double unit;               // fixed-point units of a weight of 1
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

template <typename T>
struct Row {
  const T* x;
  int64_t V;
  uint32_t kmax;
  double top, inv_t;   // largest logit, log2(e) / T

  __device__ __forceinline__ uint32_t key(int64_t i) const { return key_of(to_float(x[i])); }
  // weight of a candidate's image (> 0); exactly 1 for the largest
  __device__ __forceinline__ double weight(uint32_t k) const {
    if (k == kmax) return 1.0;
    const double t = (static_cast<double>(value_of(k)) - top) * inv_t;
    return t > -1000.0 ? exp2(t) : 0.0;    // NaN (0 * inf) also gives 0
  }
};

__device__ __forceinline__ uint64_t fixed(double w, double unit) {
  return static_cast<uint64_t>(__double2ll_rn(w * unit));
}

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// sum over the block, returned to every thread
template <typename V>
__device__ __forceinline__ V block_sum(V v, V* scratch) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  V s = 0;
  for (int i = 0; i < kWarps; ++i) s += scratch[i];
  return s;
}

struct Cut {
  uint32_t key;         // images above are kept, those below are not
  uint64_t ties;        // how many images equal to `key` are kept (the first ones by index)
};

// Digit by digit search for the image where the running amount, from the largest image down, first reaches `target`:
// amount = 1 for each candidate (kWeights false) or its fixed-point weight, over the candidates that `cut` keeps.
// Returns the image; above: the amount of larger images; at: the number of candidates with it.
template <typename T, bool kWeights>
__device__ uint32_t radix_find(const Row<T>& row, const Cut& cut, double unit, double target, uint64_t* hist,
                               uint64_t* scratch, uint64_t& above, uint64_t& at) {
  uint32_t prefix = 0;
  above = 0;
  at = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < row.V; i += kThreads) {
      const uint32_t k = row.key(i);
      if (k == 0 || k <= cut.key) continue;
      if (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
      const uint64_t a = kWeights ? fixed(row.weight(k), unit) : 1;
      atomicAdd(reinterpret_cast<unsigned long long*>(&hist[(k >> shift) & 255u]), static_cast<unsigned long long>(a));
    }
    __syncthreads();
    if (threadIdx.x == 0 && cut.ties > 0 && (shift == 24 || (cut.key >> (shift + 8)) == (prefix >> (shift + 8))))
      hist[(cut.key >> shift) & 255u] += kWeights ? cut.ties * fixed(row.weight(cut.key), unit) : cut.ties;
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t run = above;
      int d = 255, last = -1;
      for (; d >= 0; --d) {
        if (hist[d] == 0) continue;
        last = d;
        if (static_cast<double>(run + hist[d]) >= target) break;
        run += hist[d];
      }
      if (d < 0) {               // rounding only: the smallest digit that occurs
        d = last < 0 ? 0 : last;
        run -= last < 0 ? 0 : hist[d];
      }
      scratch[0] = static_cast<uint64_t>(d);
      scratch[1] = run;
      scratch[2] = hist[d];
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(scratch[0]) << shift;
    above = scratch[1];
    at = scratch[2];
    __syncthreads();
  }
  return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleParams p) {
  __shared__ uint64_t hist[256];
  __shared__ uint64_t scratch[2 * kWarps];
  __shared__ uint64_t seg_w[kWarps], seg_t[kWarps];
  const int64_t n = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Row<T> row;
  row.x = reinterpret_cast<const T*>(p.logits) + n * p.ld;
  row.V = p.V;

  // largest image, lowest index
  uint64_t best = 0;
  for (int64_t i = threadIdx.x; i < p.V; i += kThreads) {
    const uint64_t c = (static_cast<uint64_t>(row.key(i)) << 32) | static_cast<uint32_t>(~static_cast<uint32_t>(i));
    best = c > best ? c : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t c = __shfl_xor_sync(kFull, best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) scratch[warp] = best;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) best = scratch[i] > best ? scratch[i] : best;
  row.kmax = static_cast<uint32_t>(best >> 32);
  const float t = p.temperature != nullptr ? p.temperature[n] : p.temperature_all;
  if (row.kmax == 0 || !(t > 0.f)) {
    if (threadIdx.x == 0) {
      p.token[n] = row.kmax == 0 ? kNone : static_cast<int64_t>(~static_cast<uint32_t>(best));
      if (p.logprob != nullptr) p.logprob[n] = row.kmax == 0 ? -INFINITY : 0.f;
    }
    return;
  }
  row.top = static_cast<double>(value_of(row.kmax));
  row.inv_t = kLog2e64 / static_cast<double>(t);

  int64_t k = p.top_k_all;
  if (p.top_k != nullptr)
    k = p.top_k_64 ? reinterpret_cast<const int64_t*>(p.top_k)[n] : reinterpret_cast<const int*>(p.top_k)[n];
  const float tp = p.top_p != nullptr ? p.top_p[n] : p.top_p_all;
  const float mp = p.min_p != nullptr ? p.min_p[n] : p.min_p_all;

  Cut cut{0u, 0};
  uint64_t above, at;
  if (k > 0 && k < p.V) {
    const uint32_t key = radix_find<T, false>(row, cut, p.unit, static_cast<double>(k), hist, scratch, above, at);
    if (key != 0) {
      const uint64_t left = static_cast<uint64_t>(k) - min(above, static_cast<uint64_t>(k));
      cut = Cut{key, left < at ? left : at};
    }
  }
  if (!(tp >= 1.f)) {
    uint64_t part = 0;
    for (int64_t i = threadIdx.x; i < p.V; i += kThreads) {
      const uint32_t key = row.key(i);
      if (key > cut.key) part += fixed(row.weight(key), p.unit);
    }
    uint64_t all = block_sum(part, scratch);
    if (cut.ties > 0) all += cut.ties * fixed(row.weight(cut.key), p.unit);
    const double target = fmax(static_cast<double>(tp), 0.0) * static_cast<double>(all);
    const uint32_t key = radix_find<T, true>(row, cut, p.unit, target, hist, scratch, above, at);
    const uint64_t w = fixed(row.weight(key), p.unit);
    uint64_t ties = ~0ull;
    if (w > 0) {
      const uint64_t have = at / w;
      ties = 1;
      if (target > static_cast<double>(above)) {
        // smallest count with above + count * w >= target, from a quotient that may be off by one
        ties = static_cast<uint64_t>((target - static_cast<double>(above)) / static_cast<double>(w));
        ties = ties > 1 ? ties - 1 : 1;
        while (ties < have && static_cast<double>(above + ties * w) < target) ++ties;
      }
    }
    if (key == cut.key && cut.ties < ties) ties = cut.ties;
    cut = Cut{key, ties};
  }

  // kept weight by segment: each warp owns a contiguous piece of the row
  const int64_t seg = (p.V + kThreads - 1) / kThreads * 32;
  const int64_t s0 = min(seg * warp, p.V), s1 = min(s0 + seg, p.V);
  uint64_t ties = 0;
  for (int64_t i = s0 + lane; i < s1; i += 32) ties += row.key(i) == cut.key ? 1 : 0;
  ties = warp_sum(ties);
  __syncthreads();
  if (lane == 0) seg_t[warp] = ties;
  __syncthreads();
  uint64_t tie0 = 0;
  for (int i = 0; i < warp; ++i) tie0 += seg_t[i];
  const double floor_w = static_cast<double>(mp);
  auto kept = [&](int64_t i, uint64_t& tie_run, double& w) -> bool {   // all lanes of the warp call it
    const uint32_t key = i < s1 ? row.key(i) : 0u;
    const bool tie = key != 0 && key == cut.key;
    const uint32_t m = __ballot_sync(kFull, tie);
    const uint64_t rank = tie_run + __popc(m & ((1u << lane) - 1u));
    tie_run += __popc(m);
    bool keep = key > cut.key || (tie && rank < cut.ties);
    w = keep ? row.weight(key) : 0.0;
    return keep && (w >= floor_w || key == row.kmax);
  };
  // u = 0 asks for the first index with any weight at all: there a weight counts at least one unit
  const double u01 = fmin(fmax(static_cast<double>(p.u[n]), 0.0), 1.0 - 0x1p-24);
  auto units = [&](double w) -> uint64_t {
    const uint64_t f = fixed(w, p.unit);
    return (u01 == 0.0 && f == 0 && w > 0.0) ? 1 : f;
  };
  uint64_t mine = 0, run_t = tie0;
  for (int64_t i = s0 + lane; i - lane < s1; i += 32) {
    double w;
    if (kept(i, run_t, w)) mine += units(w);
  }
  mine = warp_sum(mine);
  if (lane == 0) seg_w[warp] = mine;
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += seg_w[i];
    total += seg_w[i];
  }
  const double r = u01 * static_cast<double>(total);
  if (static_cast<double>(before) > r || !(static_cast<double>(before + mine) > r)) return;
  // this warp's segment holds the token
  run_t = tie0;
  for (int64_t i = s0 + lane; i - lane < s1; i += 32) {
    double w;
    const bool keep = kept(i, run_t, w);
    uint64_t run = keep ? units(w) : 0;
    const uint64_t own_w = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t c = __shfl_up_sync(kFull, run, o);
      if (lane >= o) run += c;
    }
    const bool hit = own_w > 0 && static_cast<double>(before + run) > r;
    const uint32_t m = __ballot_sync(kFull, hit);
    if (m != 0) {
      if (lane == __ffs(m) - 1) {
        p.token[n] = i;
        if (p.logprob != nullptr)
          p.logprob[n] = static_cast<float>(log(w) - log(static_cast<double>(total) / p.unit));
      }
      return;
    }
    before += __shfl_sync(kFull, run, 31);
  }
}

const void* row_param(const c10::optional<at::Tensor>& t, const at::Tensor& logits, at::ScalarType type,
                      const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  FYB_CHECK(t->device() == logits.device() && t->scalar_type() == type && t->is_contiguous() &&
                t->numel() == logits.size(0),
            std::string("sample: ") + name);
  return t->data_ptr();
}

}  // namespace

std::vector<at::Tensor> sample(const at::Tensor& logits, const at::Tensor& u,
                               const c10::optional<at::Tensor>& temperature, double temperature_all,
                               const c10::optional<at::Tensor>& top_k, int64_t top_k_all,
                               const c10::optional<at::Tensor>& top_p, double top_p_all,
                               const c10::optional<at::Tensor>& min_p, double min_p_all, bool want_logprob) {
  FYB_RANGE("fyb::sample");
  FYB_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1),
            "sample: logits [N, V] with a contiguous last dim expected");
  const int64_t N = logits.size(0), V = logits.size(1);
  FYB_CHECK(V >= 1 && V < (1ll << 31) && N < (1ll << 31), "sample: sizes");
  c10::cuda::CUDAGuard guard(logits.device());
  SampleParams p{};
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  p.V = V;
  FYB_CHECK(u.device() == logits.device() && u.scalar_type() == at::kFloat && u.is_contiguous() && u.numel() == N,
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
  int bits = 0;
  while ((1ll << bits) < V) ++bits;
  p.unit = std::ldexp(1.0, 62 - bits);
  auto token = at::empty({N}, logits.options().dtype(at::kLong));
  at::Tensor logprob;
  if (want_logprob) logprob = at::empty({N}, logits.options().dtype(at::kFloat));
  p.token = token.data_ptr<int64_t>();
  p.logprob = want_logprob ? logprob.data_ptr<float>() : nullptr;
  if (N > 0) {
    if (logits.scalar_type() == at::kBFloat16)
      sample_kernel<__nv_bfloat16><<<N, kThreads, 0, cur_stream()>>>(p);
    else if (logits.scalar_type() == at::kHalf)
      sample_kernel<__half><<<N, kThreads, 0, cur_stream()>>>(p);
    else if (logits.scalar_type() == at::kFloat)
      sample_kernel<float><<<N, kThreads, 0, cur_stream()>>>(p);
    else
      FYB_CHECK(false, "sample: bf16, fp16 or fp32 logits expected");
    check_launch("sample");
  }
  return {token, logprob};
}

}  // namespace fyb
