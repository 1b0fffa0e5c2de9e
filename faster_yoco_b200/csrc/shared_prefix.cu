// Decode attention of a batch whose rows share long prefixes: query i of row b sees the prefix keys of its group and its
// row's own keys up to its position.
#include <ATen/ATen.h>
#include <c10/util/Optional.h>
#include <cuda_fp16.h>

#include "common/host.h"
#include "common/ptx.cuh"

namespace fyb {
namespace {

struct View {               // [rows, keys, heads, D], last dim contiguous
  const void* p;
  int64_t s0, s1, s2;
};

struct PrefixParams {
  View q, pk, pv, k, v;
  int B, Lq, Hq, Hk, G, P, S;
  const void* lengths;      // per row (int32 or int64), or null: S
  const void* prefix_lengths;
  int lengths_64, prefix_lengths_64;
  float scale;
  void* o;                  // [B, Lq, Hq, D] contiguous
};

__device__ __forceinline__ int length_of(const void* p, int wide, int i, int most) {
  if (p == nullptr) return most;
  const int64_t n = wide ? reinterpret_cast<const int64_t*>(p)[i] : reinterpret_cast<const int*>(p)[i];
  return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
}

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// one warp for each (row, query, head), one key at a time with the running maximum and sum
template <typename T, int D>
__global__ void shared_prefix_kernel(PrefixParams p) {
  constexpr int E = D / 32;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= static_cast<int64_t>(p.B) * p.Lq * p.Hq) return;
  const int h = static_cast<int>(w % p.Hq);
  const int i = static_cast<int>(w / p.Hq % p.Lq);
  const int b = static_cast<int>(w / p.Hq / p.Lq);
  const int hk = h / (p.Hq / p.Hk), g = b / (p.B / p.G);
  float q[E], o[E];
  const T* qp = reinterpret_cast<const T*>(p.q.p) + b * p.q.s0 + i * p.q.s1 + h * p.q.s2 + lane * E;
  for (int e = 0; e < E; ++e) {
    q[e] = to_float(qp[e]) * p.scale;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto walk = [&](const View& kk, const View& vv, int row, int n) {
    for (int j = 0; j < n; ++j) {
      const T* kp = reinterpret_cast<const T*>(kk.p) + row * kk.s0 + j * kk.s1 + hk * kk.s2 + lane * E;
      float s = 0.f;
      for (int e = 0; e < E; ++e) s += q[e] * to_float(kp[e]);
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float mn = fmaxf(m, s);
      const float f = m == -INFINITY ? 0.f : __expf(m - mn), a = __expf(s - mn);
      m = mn;
      l = l * f + a;
      const T* vp = reinterpret_cast<const T*>(vv.p) + row * vv.s0 + j * vv.s1 + hk * vv.s2 + lane * E;
      for (int e = 0; e < E; ++e) o[e] = o[e] * f + a * to_float(vp[e]);
    }
  };
  walk(p.pk, p.pv, g, length_of(p.prefix_lengths, p.prefix_lengths_64, g, p.P));
  const int own = length_of(p.lengths, p.lengths_64, b, p.S);
  walk(p.k, p.v, b, max(0, own - p.Lq + i + 1));
  T* op = reinterpret_cast<T*>(p.o) + w * D + lane * E;
  for (int e = 0; e < E; ++e) op[e] = from_float<T>(l > 0.f ? o[e] / l : 0.f);
}

View view_of(const at::Tensor& t, const at::Tensor& q, const char* name) {
  FYB_CHECK(t.device() == q.device() && t.scalar_type() == q.scalar_type() && t.dim() == 4 &&
                t.size(3) == q.size(3) && t.stride(3) == 1,
            std::string("shared_prefix_attention: ") + name);
  FYB_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
            std::string("shared_prefix_attention: 16-byte aligned ") + name);
  for (int d = 0; d < 3; ++d)
    FYB_CHECK(t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0),
              std::string("shared_prefix_attention: strides of ") + name + " must be positive multiples of 8 elements");
  return View{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

const void* length_ptr(const c10::optional<at::Tensor>& t, const at::Tensor& q, int64_t n, int& wide) {
  wide = 0;
  if (!t.has_value() || !t->defined()) return nullptr;
  wide = t->scalar_type() == at::kLong;
  FYB_CHECK(t->device() == q.device() && (wide || t->scalar_type() == at::kInt) && t->dim() == 1 && t->size(0) == n &&
                (n <= 1 || t->stride(0) == 1),
            "shared_prefix_attention: lengths");
  return t->data_ptr();
}

}  // namespace

at::Tensor shared_prefix_attention(const at::Tensor& q, const at::Tensor& pk, const at::Tensor& pv,
                                   const at::Tensor& k, const at::Tensor& v,
                                   const c10::optional<at::Tensor>& lengths,
                                   const c10::optional<at::Tensor>& prefix_lengths, double scale) {
  FYB_RANGE("fyb::shared_prefix_attention");
  FYB_CHECK(q.is_cuda() && q.dim() == 4 && (q.size(3) == 64 || q.size(3) == 128) &&
                (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf),
            "shared_prefix_attention: bf16 or fp16 q [B, Lq, Hq, 64 or 128] expected");
  const int64_t B = q.size(0), Lq = q.size(1), Hq = q.size(2), D = q.size(3);
  PrefixParams p{};
  p.q = view_of(q, q, "q");
  p.pk = view_of(pk, q, "prefix_k");
  p.pv = view_of(pv, q, "prefix_v");
  p.k = view_of(k, q, "k");
  p.v = view_of(v, q, "v");
  const int64_t G = pk.size(0), P = pk.size(1), Hk = pk.size(2), S = k.size(1);
  FYB_CHECK(pv.sizes() == pk.sizes() && v.sizes() == k.sizes() && k.size(0) == B && k.size(2) == Hk && Hk > 0 && G > 0 &&
                Hq % Hk == 0 && Hq / Hk <= 128 && B % G == 0,
            "shared_prefix_attention: shape mismatch");
  FYB_CHECK(B * Lq * Hq < (1ll << 31) && P < (1ll << 30) && S < (1ll << 30), "shared_prefix_attention: sizes");
  c10::cuda::CUDAGuard guard(q.device());
  auto o = at::empty({B, Lq, Hq, D}, q.options());
  if (o.numel() == 0) return o;
  p.B = (int)B, p.Lq = (int)Lq, p.Hq = (int)Hq, p.Hk = (int)Hk, p.G = (int)G, p.P = (int)P, p.S = (int)S;
  p.lengths = length_ptr(lengths, q, B, p.lengths_64);
  p.prefix_lengths = length_ptr(prefix_lengths, q, G, p.prefix_lengths_64);
  p.scale = (float)scale;
  p.o = o.data_ptr();
  const int64_t grid = (B * Lq * Hq + 3) / 4;
  if (q.scalar_type() == at::kBFloat16)
    (D == 64 ? shared_prefix_kernel<__nv_bfloat16, 64> : shared_prefix_kernel<__nv_bfloat16, 128>)
        <<<grid, 128, 0, cur_stream()>>>(p);
  else
    (D == 64 ? shared_prefix_kernel<__half, 64> : shared_prefix_kernel<__half, 128>)<<<grid, 128, 0, cur_stream()>>>(p);
  check_launch("shared_prefix_attention");
  return o;
}

}  // namespace fyb
