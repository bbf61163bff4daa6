// One AdamW step (Adam with decoupled weight decay) over a list of tensors in one launch.
//
//   g = grad * grad_scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All in float32, the master copy where there is one.  The states are float32, or 8 bits:
// m as e4m3, v as e5m2, both times a power-of-two scale for each 256 elements of a tensor.
//   * The power of two keeps a block's grid where it is when its maximum moves: a value that
//     has not changed keeps its code.
//   * The rounding is stochastic (up with the probability that keeps the mean): with b2 = 0.999
//     one step moves v by a thousandth, which rounding to nearest with two mantissa bits would
//     never let through.
//   * The maximum goes one binade below the type's top, so that rounding up never saturates.
// The noise is Philox4x32 with 7 rounds, counter (element / 4, tensor, step), key the seed: the
// upper half of an element's word rounds m, the lower half v.
#include <cmath>

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace mcl4 {
namespace {

constexpr int kAdamBlock = 256;                 // elements that share a scale; one warp's share at a time
constexpr int kAdamThreads = 256;
constexpr int64_t kAdamChunk = 32 * kAdamBlock;  // elements of a CTA

struct AdamHyper {
  float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, lr, weight_decay;
  float step_size;  // lr / (1 - beta1^t)
  float decay;      // 1 - lr * weight_decay
  float inv_root;   // 1 / sqrt(1 - beta2^t)
  double beta1_d, beta2_d;
  const int64_t* step_dev;  // or nullptr: the values above hold
  const float* lr_dev;
  const float* grad_scale;
  uint32_t step;
  uint32_t seed_lo, seed_hi;
};

template <int N>
struct AdamTable {
  void* p[N];
  const void* g[N];
  void* m[N];
  void* v[N];
  float* ms[N];
  float* vs[N];
  float* master[N];
  int64_t numel[N];
  int32_t first[N + 1];  // first chunk of each tensor
  int32_t index[N];      // the tensor's number in the noise counter
  int32_t n;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f(uint16_t v) {
  return bf16_to_f32(v);
}
template <>
__device__ __forceinline__ float to_f(__half v) {
  return __half2float(v);
}
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(uint16_t& d, float v) { d = f32_to_bf16(v); }
__device__ __forceinline__ void from_f(__half& d, float v) { d = __float2half_rn(v); }

// Four consecutive elements: one vector access where all four exist and the address allows it.
template <typename T>
struct __align__(4 * sizeof(T)) Four {
  T v[4];
};
template <typename T>
__device__ __forceinline__ Four<T> load4(const T* p, int count, bool wide) {
  Four<T> r;
  if (wide && count == 4) return *reinterpret_cast<const Four<T>*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = i < count ? p[i] : T(0);
  return r;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const Four<T>& r, int count, bool wide) {
  if (wide && count == 4) {
    *reinterpret_cast<Four<T>*>(p) = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) p[i] = r.v[i];
}

// Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11),
// 7 rounds, the fewest that the paper found to pass BigCrush.
__device__ __forceinline__ uint4 philox7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = uint64_t(0xD2511F53u) * c0, b = uint64_t(0xCD9E8D57u) * c2;
    c0 = uint32_t(b >> 32) ^ c1 ^ k0;
    c1 = uint32_t(b);
    c2 = uint32_t(a >> 32) ^ c3 ^ k1;
    c3 = uint32_t(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// 8-bit float with MANT mantissa bits and exponent bias BIAS of x * inv, rounded up where the
// dropped part plus noise / 2^16 reaches a step; NaN where x is not finite.
template <int MANT, int BIAS>
__device__ __forceinline__ uint32_t round8(float x, float inv, uint32_t noise) {
  const uint32_t sign = (__float_as_uint(x) >> 31) << 7;
  if (!finite(x)) return 0x7Fu | sign;
  const float a = __fmul_rn(fabsf(x), inv);
  int e = int(__float_as_uint(a) >> 23) - 127;  // binade; denormals and 0 end up below the smallest
  e = e < 1 - BIAS ? 1 - BIAS : e;
  const float steps = floorf(__fadd_rn(__fmul_rn(a, pow2f(MANT - e)), __fmul_rn(float(noise), 1.52587890625e-05f)));
  return ((uint32_t(e + BIAS) << MANT) + uint32_t(steps) - (1u << MANT)) | sign;
}
__device__ __forceinline__ float e4m3_value(uint32_t c) {
  const float v = (c & 0x7Fu) == 0x7Fu ? __uint_as_float(0x7FC00000u) : e4m3_to_f32(c & 0x7Fu);
  return c & 0x80u ? -v : v;
}
__device__ __forceinline__ float e5m2_value(uint32_t c) {  // the upper byte of a half
  return __half2float(__ushort_as_half(static_cast<unsigned short>(c << 8)));
}

// The power of two that puts the block's largest finite magnitude into binade TOP, and its inverse.
template <int TOP>
__device__ __forceinline__ void block_scale(uint32_t largest_bits, float& scale, float& inv) {
  int e = 31 - __clz(int(largest_bits));  // of a denormal: its binade is e - 149
  e = largest_bits >> 23 ? int(largest_bits >> 23) - 127 : e - 149;
  e = e < -112 ? -112 : e;
  scale = largest_bits ? pow2f(e - TOP) : 1.f;
  inv = pow2f(TOP - e);
}

template <typename P, typename G, bool EIGHT, int N>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamTable<N> tab,
                                                             const AdamHyper h0) {
  AdamHyper h = h0;
  if (h.step_dev != nullptr || h.lr_dev != nullptr) {
    __shared__ float dev[4];
    if (threadIdx.x == 0) {
      const int64_t step = h.step_dev != nullptr ? *h.step_dev : int64_t(h.step);
      const double lr = h.lr_dev != nullptr ? double(*h.lr_dev) : double(h.lr);
      dev[0] = float(lr / (1.0 - pow(h.beta1_d, double(step))));
      dev[1] = float(1.0 - lr * double(h.weight_decay));
      dev[2] = float(1.0 / sqrt(1.0 - pow(h.beta2_d, double(step))));
      dev[3] = __uint_as_float(uint32_t(step));
    }
    __syncthreads();
    h.step_size = dev[0];
    h.decay = dev[1];
    h.inv_root = dev[2];
    h.step = __float_as_uint(dev[3]);
  }
  int lo = 0, hi = tab.n - 1;  // the last tensor whose first chunk is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= int(blockIdx.x)) lo = mid;
    else hi = mid - 1;
  }
  const int t = lo;
  const int64_t numel = tab.numel[t];
  const int64_t begin = int64_t(int(blockIdx.x) - tab.first[t]) * kAdamChunk;
  const int64_t end = begin + kAdamChunk < numel ? begin + kAdamChunk : numel;
  P* p = static_cast<P*>(tab.p[t]);
  const G* g = static_cast<const G*>(tab.g[t]);
  float* master = tab.master[t];
  const bool wide_p = (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(P) - 1)) == 0;
  const bool wide_g = (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(G) - 1)) == 0;
  const bool wide_w = (reinterpret_cast<uintptr_t>(master) & 15) == 0;
  const int state = EIGHT ? 1 : 4;
  const bool wide_s =
      ((reinterpret_cast<uintptr_t>(tab.m[t]) | reinterpret_cast<uintptr_t>(tab.v[t])) & (4 * state - 1)) == 0;
  const float grad_scale = h.grad_scale != nullptr ? *h.grad_scale : 1.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t base = begin + warp * kAdamBlock; base < end; base += kAdamThreads / 32 * kAdamBlock) {
    float m[2][4], v[2][4];
    uint32_t m_top = 0, v_top = 0;
    float ms = 1.f, vs = 1.f;
    if (EIGHT) {
      ms = tab.ms[t][base / kAdamBlock];
      vs = tab.vs[t][base / kAdamBlock];
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t at = base + q * 128 + lane * 4;
      const int count = at >= end ? 0 : end - at >= 4 ? 4 : int(end - at);
      if (count == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m[q][i] = v[q][i] = 0.f;
        continue;
      }
      const Four<G> g4 = load4(g + at, count, wide_g);
      Four<P> p4 = load4(p + at, count, wide_p);
      Four<float> w4;
      if (master != nullptr) w4 = load4(master + at, count, wide_w);
      if (EIGHT) {
        const Four<uint8_t> mc = load4(static_cast<const uint8_t*>(tab.m[t]) + at, count, wide_s);
        const Four<uint8_t> vc = load4(static_cast<const uint8_t*>(tab.v[t]) + at, count, wide_s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[q][i] = __fmul_rn(e4m3_value(mc.v[i]), ms);
          v[q][i] = __fmul_rn(e5m2_value(vc.v[i]), vs);
        }
      } else {
        const Four<float> m4 = load4(static_cast<const float*>(tab.m[t]) + at, count, wide_s);
        const Four<float> v4 = load4(static_cast<const float*>(tab.v[t]) + at, count, wide_s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[q][i] = m4.v[i];
          v[q][i] = v4.v[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gr = __fmul_rn(to_f(g4.v[i]), grad_scale);
        m[q][i] = __fadd_rn(__fmul_rn(m[q][i], h.beta1), __fmul_rn(gr, h.one_minus_beta1));
        v[q][i] = __fadd_rn(__fmul_rn(v[q][i], h.beta2), __fmul_rn(__fmul_rn(gr, gr), h.one_minus_beta2));
        const float denom = sqrtf(v[q][i]) * h.inv_root + h.eps;
        const float w = master != nullptr ? w4.v[i] : to_f(p4.v[i]);
        const float now = w * h.decay - (m[q][i] / denom) * h.step_size;
        w4.v[i] = now;
        from_f(p4.v[i], now);
        if (i < count) {
          const uint32_t mb = __float_as_uint(m[q][i]) & 0x7FFFFFFFu, vb = __float_as_uint(v[q][i]) & 0x7FFFFFFFu;
          if (mb < 0x7F800000u) m_top = max(m_top, mb);
          if (vb < 0x7F800000u) v_top = max(v_top, vb);
        }
      }
      store4(p + at, p4, count, wide_p);
      if (master != nullptr) store4(master + at, w4, count, wide_w);
      if (!EIGHT) {
        Four<float> m4, v4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m4.v[i] = m[q][i];
          v4.v[i] = v[q][i];
        }
        store4(static_cast<float*>(tab.m[t]) + at, m4, count, wide_s);
        store4(static_cast<float*>(tab.v[t]) + at, v4, count, wide_s);
      }
    }
    if (!EIGHT) continue;
    float m_inv, v_inv;
    block_scale<7>(__reduce_max_sync(0xffffffffu, m_top), ms, m_inv);
    block_scale<14>(__reduce_max_sync(0xffffffffu, v_top), vs, v_inv);
    if (lane == 0) {
      tab.ms[t][base / kAdamBlock] = ms;
      tab.vs[t][base / kAdamBlock] = vs;
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t at = base + q * 128 + lane * 4;
      const int count = at >= end ? 0 : end - at >= 4 ? 4 : int(end - at);
      if (count == 0) continue;
      const uint4 word = philox7(uint32_t(at >> 2), uint32_t(at >> 34), uint32_t(tab.index[t]), h.step, h.seed_lo,
                                 h.seed_hi);
      const uint32_t w[4] = {word.x, word.y, word.z, word.w};
      Four<uint8_t> mc, vc;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mc.v[i] = uint8_t(round8<3, 7>(m[q][i], m_inv, w[i] >> 16));
        vc.v[i] = uint8_t(round8<2, 15>(v[q][i], v_inv, w[i] & 0xFFFFu));
      }
      store4(static_cast<uint8_t*>(tab.m[t]) + at, mc, count, wide_s);
      store4(static_cast<uint8_t*>(tab.v[t]) + at, vc, count, wide_s);
    }
  }
}

template <typename P, typename G, bool EIGHT, int N>
int launch_table(const mcl4moe_adamw_args* a, int first, int count, const AdamHyper& h, cudaStream_t stream) {
  AdamTable<N> tab;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const int t = first + i;
    tab.p[i] = a->params[t];
    tab.g[i] = a->grads[t];
    tab.m[i] = a->exp_avgs[t];
    tab.v[i] = a->exp_avg_sqs[t];
    tab.ms[i] = EIGHT ? a->exp_avg_scales[t] : nullptr;
    tab.vs[i] = EIGHT ? a->exp_avg_sq_scales[t] : nullptr;
    tab.master[i] = a->masters ? a->masters[t] : nullptr;
    tab.numel[i] = a->numels[t];
    tab.index[i] = a->indices ? a->indices[t] : t;
    tab.first[i] = int32_t(chunks);
    chunks += (a->numels[t] + kAdamChunk - 1) / kAdamChunk;
    if (chunks > (int64_t(1) << 30)) return MCL4MOE_ERR_UNSUPPORTED;
  }
  tab.first[count] = int32_t(chunks);
  tab.n = count;
  if (chunks == 0) return MCL4MOE_OK;
  adamw_kernel<P, G, EIGHT, N><<<unsigned(chunks), kAdamThreads, 0, stream>>>(tab, h);
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

// The tensors' pointers travel as kernel arguments (32764 bytes at most): a small table for few
// tensors, full ones for the rest.
template <typename P, typename G, bool EIGHT>
int launch_adamw(const mcl4moe_adamw_args* a, const AdamHyper& h, cudaStream_t stream) {
  for (int first = 0; first < a->n;) {
    const int left = a->n - first;
    const int count = left < 440 ? left : 440;
    const int st = count <= 32 ? launch_table<P, G, EIGHT, 32>(a, first, count, h, stream)
                               : launch_table<P, G, EIGHT, 440>(a, first, count, h, stream);
    if (st != MCL4MOE_OK) return st;
    first += count;
  }
  return MCL4MOE_OK;
}

template <typename P>
int launch_adamw_grad(const mcl4moe_adamw_args* a, const AdamHyper& h, cudaStream_t stream) {
  if (a->grad_dtype == 0)
    return a->bits == 8 ? launch_adamw<P, uint16_t, true>(a, h, stream) : launch_adamw<P, uint16_t, false>(a, h, stream);
  if (a->grad_dtype == 1)
    return a->bits == 8 ? launch_adamw<P, float, true>(a, h, stream) : launch_adamw<P, float, false>(a, h, stream);
  return a->bits == 8 ? launch_adamw<P, __half, true>(a, h, stream) : launch_adamw<P, __half, false>(a, h, stream);
}

}  // namespace
}  // namespace mcl4

using namespace mcl4;

extern "C" int mcl4moe_adamw_step(const mcl4moe_adamw_args* a, mcl4moe_stream_t stream) {
  if (!a || a->n < 0 || a->param_dtype < 0 || a->param_dtype > 2 || a->grad_dtype < 0 || a->grad_dtype > 2 ||
      (a->bits != 8 && a->bits != 32))
    return MCL4MOE_ERR_INVALID;
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 && a->eps >= 0.0))
    return MCL4MOE_ERR_INVALID;
  if (!a->step_dev && a->step < 1) return MCL4MOE_ERR_INVALID;
  if (a->n > 0 && (!a->params || !a->grads || !a->exp_avgs || !a->exp_avg_sqs || !a->numels ||
                   (a->bits == 8 && (!a->exp_avg_scales || !a->exp_avg_sq_scales))))
    return MCL4MOE_ERR_INVALID;
  for (int i = 0; i < a->n; ++i) {
    if (a->numels[i] < 0) return MCL4MOE_ERR_INVALID;
    if (a->numels[i] > 0 && (!a->params[i] || !a->grads[i] || !a->exp_avgs[i] || !a->exp_avg_sqs[i] ||
                             (a->bits == 8 && (!a->exp_avg_scales[i] || !a->exp_avg_sq_scales[i])) ||
                             (a->masters && !a->masters[i])))
      return MCL4MOE_ERR_INVALID;
  }
  AdamHyper h{};
  h.beta1 = float(a->beta1);
  h.beta2 = float(a->beta2);
  h.one_minus_beta1 = float(1.0 - a->beta1);
  h.one_minus_beta2 = float(1.0 - a->beta2);
  h.eps = float(a->eps);
  h.lr = float(a->lr);
  h.weight_decay = float(a->weight_decay);
  h.decay = float(1.0 - a->lr * a->weight_decay);
  if (!a->step_dev) {
    h.step_size = float(a->lr / (1.0 - std::pow(a->beta1, double(a->step))));
    h.inv_root = float(1.0 / std::sqrt(1.0 - std::pow(a->beta2, double(a->step))));
  }
  h.beta1_d = a->beta1;
  h.beta2_d = a->beta2;
  h.step_dev = a->step_dev;
  h.lr_dev = a->lr_dev;
  h.grad_scale = a->grad_scale;
  h.step = uint32_t(a->step);
  h.seed_lo = uint32_t(a->seed);
  h.seed_hi = uint32_t(a->seed >> 32);
  if (a->param_dtype == 0) return launch_adamw_grad<uint16_t>(a, h, stream);
  if (a->param_dtype == 1) return launch_adamw_grad<float>(a, h, stream);
  return launch_adamw_grad<__half>(a, h, stream);
}
