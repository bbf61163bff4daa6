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
#include <type_traits>

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace mcl4 {
namespace {

constexpr int kAdamBlock = 256;    // elements that share a scale; one warp's share at a time
constexpr int kAdamThreads = 256;
constexpr int kAdamPass = kAdamThreads / 32 * kAdamBlock;  // elements of a CTA's pass: a block for each warp
constexpr int kAdamCtas = 3;                    // resident on an SM

struct AdamHyper {
  float beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
  float step_size;  // lr / (1 - beta1^t)
  float decay;      // 1 - lr * weight_decay
  float inv_root;   // 1 / sqrt(1 - beta2^t)
  double beta1_d, beta2_d, lr, weight_decay;
  const int64_t* step_dev;  // or nullptr: the values above hold
  const float* lr_dev;
  const float* grad_scale;
  uint32_t step;
  uint32_t keys[14];  // Philox's key of each round
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
  uint8_t wide[N];       // its arrays allow accesses of four elements
  int32_t n;
  int32_t passes;        // of a CTA's turn
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

// Four consecutive elements, by one access or (`count` of them) singly.
template <typename T>
struct __align__(4 * sizeof(T)) Four {
  T v[4];
};
template <bool WHOLE, typename T>
__device__ __forceinline__ Four<T> load4(const T* p, int count) {
  if constexpr (WHOLE) {
    return *reinterpret_cast<const Four<T>*>(p);
  } else {
    Four<T> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = i < count ? p[i] : T(0);
    return r;
  }
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store4(T* p, const Four<T>& r, int count) {
  if constexpr (WHOLE) {
    *reinterpret_cast<Four<T>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) p[i] = r.v[i];
  }
}

template <int BYTES>
__device__ __forceinline__ void copy_ahead(void* to, const void* from) {
  const uint32_t at = uint32_t(__cvta_generic_to_shared(to));
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES == 16 ? 4 : BYTES) : "memory");
}

__device__ __forceinline__ uint32_t word4(const Four<uint8_t>& b) { return *reinterpret_cast<const uint32_t*>(&b); }
__device__ __forceinline__ Four<uint8_t> bytes4(uint32_t w) { return *reinterpret_cast<const Four<uint8_t>*>(&w); }

// Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11),
// 7 rounds, the fewest that the paper found to pass BigCrush.
__device__ __forceinline__ uint4 philox7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, const uint32_t (&keys)[14]) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = uint64_t(0xD2511F53u) * c0, b = uint64_t(0xCD9E8D57u) * c2;
    c0 = uint32_t(b >> 32) ^ c1 ^ keys[2 * r];
    c1 = uint32_t(b);
    c2 = uint32_t(a >> 32) ^ c3 ^ keys[2 * r + 1];
    c3 = uint32_t(a);
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

// 8-bit float with MANT mantissa bits and exponent bias BIAS of x * inv, rounded up where the
// dropped part plus noise / 2^16 reaches a step; NaN where x is not finite.  A block's values lie
// below 2^(TOP + 1).
//   * In the type's normal range the bits themselves are the sum's fixed point: the noise goes onto
//     the dropped bits and carries into the kept ones.  round8_normal returns that code less
//     1 << MANT, and tells of values outside the range.
//   * Below it (2^-13 of the block's largest for e4m3, 2^-28 for e5m2) the step is fixed and the
//     sum is taken in float32: round8, for all.
template <int MANT, int BIAS, int TOP>
__device__ __forceinline__ uint32_t round8_normal(float x, float inv, uint32_t noise, bool& outside) {
  constexpr uint32_t kLow = uint32_t(128 - BIAS) << 23, kRange = uint32_t(TOP + BIAS) << 23;
  const uint32_t over = __float_as_uint(__fmul_rn(fabsf(x), inv)) - kLow;
  outside |= over >= kRange;
  return (over + (noise << (7 - MANT))) >> (23 - MANT);
}
template <int MANT, int BIAS, int TOP>
__device__ __forceinline__ uint32_t round8(float x, float inv, uint32_t noise) {
  bool outside = false;
  const uint32_t code = round8_normal<MANT, BIAS, TOP>(x, inv, noise, outside) + (1u << MANT);
  if (!outside) return code;
  if ((__float_as_uint(x) & 0x7F800000u) == 0x7F800000u) return 0x7Fu;
  const float a = __fmul_rn(fabsf(x), inv);
  return uint32_t(__fadd_rn(__fmul_rn(a, float(1 << (MANT + BIAS - 1))), __fmul_rn(float(noise), 1.52587890625e-05f)));
}

__device__ __forceinline__ uint32_t pack4(const uint32_t (&b)[4]) {
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// The codes of four moments of either kind where one of them is outside its type's normal range: rare,
// so its registers stay out of the caller.
__device__ __noinline__ uint2 round_any(float4 m, float4 v, float m_inv, float v_inv, uint4 word) {
  const float mf[4] = {m.x, m.y, m.z, m.w}, vf[4] = {v.x, v.y, v.z, v.w};
  const uint32_t w[4] = {word.x, word.y, word.z, word.w};
  uint32_t mc[4], vc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mc[i] = round8<3, 7, 7>(mf[i], m_inv, w[i] >> 16);
    vc[i] = round8<2, 15, 14>(vf[i], v_inv, w[i] & 0xFFFFu);
  }
  return make_uint2(pack4(mc), pack4(vc));
}

// Four e4m3 / e5m2 codes of one word, by the hardware's conversion to halves.
__device__ __forceinline__ void e4m3x4(uint32_t w, float (&v)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t r;
    asm("{ .reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t; }" : "=r"(r) : "r"(w >> (16 * h)));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
    v[2 * h] = f.x;
    v[2 * h + 1] = f.y;
  }
}
__device__ __forceinline__ void e5m2x4(uint32_t w, float (&v)[4]) {  // a code is the upper byte of its half
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t r = __byte_perm(w, 0u, h ? 0x3424 : 0x1404);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
    v[2 * h] = f.x;
    v[2 * h + 1] = f.y;
  }
}

// The update's square root and reciprocal, within 2^-22 each: their rounding ends up far below the
// parameter's own.
__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float inverse_of(float d) {
  float r;  // the flush to zero of a denormal denominator meets eps = 0 and v = 0 alone
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
__device__ __forceinline__ uint64_t both(float v) { return f2pack(v, v); }
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
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

// What a warp needs of a tensor: its arrays from the CTA's first element of this turn on.
template <typename P, typename G, bool EIGHT, bool MASTER>
struct AdamTensor {
  using S = typename std::conditional<EIGHT, uint8_t, float>::type;
  P* p;
  const G* g;
  S* m;
  S* v;
  float* master;
};

// A lane's elements of a block, 2 x 4, as they were.
template <typename P, typename G, bool EIGHT, bool MASTER>
struct AdamRaw {
  using S = typename AdamTensor<P, G, EIGHT, MASTER>::S;
  Four<G> g[2];
  Four<P> p[2];
  Four<float> w[2];
  Four<S> m[2], v[2];
  float ms, vs;
};

template <bool WHOLE, typename P, typename G, bool EIGHT, bool MASTER>
__device__ __forceinline__ AdamRaw<P, G, EIGHT, MASTER> adam_load(const AdamTensor<P, G, EIGHT, MASTER>& t, int off, int left,
                                                                  const float* scale_m, const float* scale_v) {
  const int lane = threadIdx.x & 31;
  AdamRaw<P, G, EIGHT, MASTER> r;
  r.ms = EIGHT ? *scale_m : 1.f;
  r.vs = EIGHT ? *scale_v : 1.f;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int at = off + q * 128 + lane * 4;
    const int count = WHOLE ? 4 : max(0, min(4, left - q * 128 - lane * 4));
    r.g[q] = load4<WHOLE>(t.g + at, count);
    if (MASTER) r.w[q] = load4<WHOLE>(t.master + at, count);
    else r.p[q] = load4<WHOLE>(t.p + at, count);
    r.m[q] = load4<WHOLE>(t.m + at, count);
    r.v[q] = load4<WHOLE>(t.v + at, count);
  }
  return r;
}

// The step's factors: those of the launch, or taken from the device's step count and rate.
struct AdamFactors {
  float step_size, decay, inv_root, grad_scale;
  uint32_t step;
  __device__ __forceinline__ explicit AdamFactors(const AdamHyper& h) {
    step_size = h.step_size;
    decay = h.decay;
    inv_root = h.inv_root;
    step = h.step;
    if (h.step_dev != nullptr || h.lr_dev != nullptr) {
      __shared__ float dev[4];
      if (threadIdx.x == 0) {
        const int64_t now = h.step_dev != nullptr ? *h.step_dev : int64_t(h.step);
        const double lr = h.lr_dev != nullptr ? double(*h.lr_dev) : h.lr;
        dev[0] = float(lr / (1.0 - pow(h.beta1_d, double(now))));
        dev[1] = float(1.0 - lr * h.weight_decay);
        dev[2] = float(1.0 / sqrt(1.0 - pow(h.beta2_d, double(now))));
        dev[3] = __uint_as_float(uint32_t(now));
      }
      __syncthreads();
      step_size = dev[0];
      decay = dev[1];
      inv_root = dev[2];
      step = __float_as_uint(dev[3]);
    }
    grad_scale = h.grad_scale != nullptr ? *h.grad_scale : 1.f;
  }
};

// One block of 256 elements.  WHOLE: all 256 are there and lie on vector addresses.
template <bool WHOLE, typename P, typename G, bool EIGHT, bool MASTER>
__device__ __forceinline__ void adam_block(const AdamTensor<P, G, EIGHT, MASTER>& t, AdamRaw<P, G, EIGHT, MASTER>& r, int off,
                                           int left, float* scale_m, float* scale_v, int64_t element, int32_t index,
                                           const AdamHyper& h, const AdamFactors& f) {
  const int lane = threadIdx.x & 31;
  int count[2] = {4, 4};
  if (!WHOLE)
#pragma unroll
    for (int q = 0; q < 2; ++q) count[q] = max(0, min(4, left - q * 128 - lane * 4));
  float m[2][4], v[2][4];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int at = off + q * 128 + lane * 4;
    if constexpr (EIGHT) {
      e4m3x4(word4(r.m[q]), m[q]);
      e5m2x4(word4(r.v[q]), v[q]);
    }
// Two elements an instruction where a product stands alone.  The moments' sums are single: each
    // product and sum is rounded by itself, which the 8-bit codes' definition goes by, and a packed
    // product and a packed sum (mul and add.rn.f32x2) came out fused.
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint64_t gr = fmul2(f2pack(to_f(r.g[q].v[i]), to_f(r.g[q].v[i + 1])), both(f.grad_scale));
      uint64_t mm, vv;
      if constexpr (EIGHT) {
        mm = fmul2(f2pack(m[q][i], m[q][i + 1]), both(r.ms));
        vv = fmul2(f2pack(v[q][i], v[q][i + 1]), both(r.vs));
      } else {
        mm = f2pack(r.m[q].v[i], r.m[q].v[i + 1]);
        vv = f2pack(r.v[q].v[i], r.v[q].v[i + 1]);
      }
      float m0, m1, v0, v1, g0, g1, h0, h1;
      f2unpack(fmul2(mm, both(h.beta1)), m0, m1);
      f2unpack(fmul2(gr, both(h.one_minus_beta1)), g0, g1);
      f2unpack(fmul2(vv, both(h.beta2)), v0, v1);
      f2unpack(fmul2(fmul2(gr, gr), both(h.one_minus_beta2)), h0, h1);
      m[q][i] = __fadd_rn(m0, g0);
      m[q][i + 1] = __fadd_rn(m1, g1);
      v[q][i] = __fadd_rn(v0, h0);
      v[q][i + 1] = __fadd_rn(v1, h1);
      const uint64_t w = MASTER ? f2pack(r.w[q].v[i], r.w[q].v[i + 1]) : f2pack(to_f(r.p[q].v[i]), to_f(r.p[q].v[i + 1]));
      const uint64_t denom = ffma2(f2pack(root_of(v[q][i]), root_of(v[q][i + 1])), both(f.inv_root), both(h.eps));
      float d0, d1, now0, now1;
      f2unpack(denom, d0, d1);
      const uint64_t ratio = fmul2(f2pack(m[q][i], m[q][i + 1]), f2pack(inverse_of(d0), inverse_of(d1)));
      f2unpack(ffma2(ratio, both(-f.step_size), fmul2(w, both(f.decay))), now0, now1);
      r.w[q].v[i] = now0;
      r.w[q].v[i + 1] = now1;
      from_f(r.p[q].v[i], now0);
      from_f(r.p[q].v[i + 1], now1);
    }
    store4<WHOLE>(t.p + at, r.p[q], count[q]);
    if (MASTER) store4<WHOLE>(t.master + at, r.w[q], count[q]);
    if constexpr (!EIGHT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.m[q].v[i] = m[q][i];
        r.v[q].v[i] = v[q][i];
      }
      store4<WHOLE>(t.m + at, r.m[q], count[q]);
      store4<WHOLE>(t.v + at, r.v[q], count[q]);
    }
  }
  if constexpr (EIGHT) {
    // The largest magnitudes; elements behind the end were loaded as zeros and stay 0, NaN is passed over.
    float m_max = 0.f, v_max = 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m_max = fmaxf(m_max, fabsf(m[q][i]));
        v_max = fmaxf(v_max, fabsf(v[q][i]));
      }
    uint32_t m_top = __reduce_max_sync(0xffffffffu, __float_as_uint(m_max));
    uint32_t v_top = __reduce_max_sync(0xffffffffu, __float_as_uint(v_max));
    if (m_top == 0x7F800000u || v_top == 0x7F800000u) {  // rare: the largest of the finite ones
      m_top = v_top = 0;
      for (int q = 0; q < 2; ++q)
        for (int i = 0; i < 4; ++i) {
          const uint32_t mb = __float_as_uint(m[q][i]) & 0x7FFFFFFFu, vb = __float_as_uint(v[q][i]) & 0x7FFFFFFFu;
          if (mb < 0x7F800000u) m_top = max(m_top, mb);
          if (vb < 0x7F800000u) v_top = max(v_top, vb);
        }
      m_top = __reduce_max_sync(0xffffffffu, m_top);
      v_top = __reduce_max_sync(0xffffffffu, v_top);
    }
    float ms, vs, m_inv, v_inv;
    block_scale<7>(m_top, ms, m_inv);
    block_scale<14>(v_top, vs, v_inv);
    if (lane == 0) {
      *scale_m = ms;
      *scale_v = vs;
    }
    const int64_t quad = (element >> 2) + lane;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (!WHOLE && count[q] == 0) continue;
      const uint4 word = philox7(uint32_t(quad + 32 * q), uint32_t(quad >> 32), uint32_t(index), f.step, h.keys);
      const uint32_t w[4] = {word.x, word.y, word.z, word.w};
      uint32_t mc[4], vc[4];
      bool outside = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mc[i] = round8_normal<3, 7, 7>(m[q][i], m_inv, w[i] >> 16, outside);
        vc[i] = round8_normal<2, 15, 14>(v[q][i], v_inv, w[i] & 0xFFFFu, outside);
      }
      uint32_t m_word = pack4(mc) + 0x08080808u, v_word = pack4(vc) + 0x04040404u;
      if (outside) {
        const uint2 both = round_any(make_float4(m[q][0], m[q][1], m[q][2], m[q][3]),
                                     make_float4(v[q][0], v[q][1], v[q][2], v[q][3]), m_inv, v_inv, word);
        m_word = both.x;
        v_word = both.y;
      }
      uint32_t sign[4];  // of m; v is a sum of squares
#pragma unroll
      for (int i = 0; i < 4; ++i) sign[i] = __float_as_uint(m[q][i]);
      const uint32_t top = __byte_perm(__byte_perm(sign[0], sign[1], 0x0073), __byte_perm(sign[2], sign[3], 0x0073), 0x5410);
      const int at = off + q * 128 + lane * 4;
      store4<WHOLE>(t.m + at, bytes4(m_word | (top & 0x80808080u)), count[q]);
      store4<WHOLE>(t.v + at, bytes4(v_word), count[q]);
    }
  }
}

// The tensor of a turn: the last one whose first turn is not behind it.
template <int N>
__device__ __forceinline__ int adam_find(const AdamTable<N>& tab, int turn) {
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= turn) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
template <typename P, typename G, bool EIGHT, bool MASTER, int N>
__device__ __forceinline__ AdamTensor<P, G, EIGHT, MASTER> adam_tensor(const AdamTable<N>& tab, int t, int64_t element) {
  using S = typename AdamTensor<P, G, EIGHT, MASTER>::S;
  return {static_cast<P*>(tab.p[t]) + element, static_cast<const G*>(tab.g[t]) + element, static_cast<S*>(tab.m[t]) + element,
          static_cast<S*>(tab.v[t]) + element, MASTER ? tab.master[t] + element : nullptr};
}

// 32-bit moments: bound by HBM with one block after the other, one CTA a turn (403 M elements 1.65 ms,
// 6.8 TB/s; persistent CTAs 1.80 ms).
template <typename P, typename G, bool MASTER, int N>
__global__ void __launch_bounds__(kAdamThreads, 4) adamw_kernel(const __grid_constant__ AdamTable<N> tab,
                                                                const __grid_constant__ AdamHyper h) {
  const AdamFactors f(h);
  const int t = adam_find(tab, blockIdx.x);
  const int chunk = tab.passes * kAdamPass;
  const int64_t begin = int64_t(int(blockIdx.x) - tab.first[t]) * chunk;
  const AdamTensor<P, G, false, MASTER> a = adam_tensor<P, G, false, MASTER>(tab, t, begin);
  const int here = int(min(int64_t(chunk), tab.numel[t] - begin));
  const bool wide = tab.wide[t] != 0;
  for (int off = (threadIdx.x >> 5) * kAdamBlock; off < here; off += kAdamPass) {
    if (here - off >= kAdamBlock && wide) {
      auto raw = adam_load<true>(a, off, kAdamBlock, nullptr, nullptr);
      adam_block<true>(a, raw, off, kAdamBlock, nullptr, nullptr, begin + off, 0, h, f);
    } else {
      const int left = min(kAdamBlock, here - off);
      auto raw = adam_load<false>(a, off, left, nullptr, nullptr);
      adam_block<false>(a, raw, off, left, nullptr, nullptr, begin + off, 0, h, f);
    }
  }
}

// 8-bit moments: half the bytes and more arithmetic (about 75 instructions an element, bound by their
// issue and HBM together), so the loads have to run ahead of it.  Persistent CTAs take turns; each
// lane copies its own elements of the blocks to come into shared memory (cp.async), kAdamAhead turns
// ahead, and reads them back itself.  94 M elements: 281 us, 5.4 TB/s (loads into registers, no
// turns ahead: 448 us).
constexpr int kAdamAhead = 3;

template <typename P, typename G, bool MASTER, int N>
__global__ void __launch_bounds__(kAdamThreads, kAdamCtas) adamw8_kernel(const __grid_constant__ AdamTable<N> tab,
                                                                         const __grid_constant__ AdamHyper h) {
  using W = typename std::conditional<MASTER, float, P>::type;
  struct Ahead {
    Four<G> g[2][kAdamThreads];
    Four<W> w[2][kAdamThreads];
    uint32_t m[2][kAdamThreads], v[2][kAdamThreads];
    float scales[kAdamThreads / 32][2];
    int64_t element[kAdamThreads / 32];
    int tensor[kAdamThreads / 32], left[kAdamThreads / 32];  // left < 256: the block is loaded when its time comes
  };
  extern __shared__ __align__(16) char smem[];
  Ahead* ahead = reinterpret_cast<Ahead*>(smem);
  const AdamFactors f(h);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the block to fetch next; where it lies goes into its slot with it
  int t = adam_find(tab, blockIdx.x), turn = blockIdx.x;
  const int turns = tab.first[tab.n];
  auto fetch = [&](Ahead& s) {
    if (turn < turns) {
      while (turn >= tab.first[t + 1]) ++t;
      const int64_t element = int64_t(turn - tab.first[t]) * kAdamPass + warp * kAdamBlock;
      const int64_t rest = tab.numel[t] - element;
      const bool whole = rest >= kAdamBlock && tab.wide[t] != 0;
      if (lane == 0) {
        s.element[warp] = element;
        s.tensor[warp] = t;
        s.left[warp] = whole ? kAdamBlock : rest <= 0 ? 0 : rest < kAdamBlock ? int(rest) : -kAdamBlock;
      }
      if (whole) {
        const AdamTensor<P, G, true, MASTER> a = adam_tensor<P, G, true, MASTER>(tab, t, element);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int e = q * 128 + lane * 4;
          copy_ahead<sizeof(Four<G>)>(&s.g[q][threadIdx.x], a.g + e);
          if constexpr (MASTER) copy_ahead<16>(&s.w[q][threadIdx.x], a.master + e);
          else copy_ahead<sizeof(Four<W>)>(&s.w[q][threadIdx.x], a.p + e);
          copy_ahead<4>(&s.m[q][threadIdx.x], a.m + e);
          copy_ahead<4>(&s.v[q][threadIdx.x], a.v + e);
        }
        if (lane < 2) copy_ahead<4>(&s.scales[warp][lane], (lane == 0 ? tab.ms : tab.vs)[t] + element / kAdamBlock);
      }
      turn += gridDim.x;
    } else if (lane == 0) {
      s.tensor[warp] = -1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < kAdamAhead; ++s) fetch(ahead[s]);
  for (int stage = 0;; stage = stage + 1 == kAdamAhead ? 0 : stage + 1) {
    Ahead& s = ahead[stage];
    asm volatile("cp.async.wait_group %0;" ::"n"(kAdamAhead - 1) : "memory");
    __syncwarp();  // place and scales come from other lanes
    const int at = s.tensor[warp];
    if (at < 0) break;
    const int64_t element = s.element[warp];
    const int left = s.left[warp];
    AdamRaw<P, G, true, MASTER> raw;
    if (left == kAdamBlock) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        raw.g[q] = s.g[q][threadIdx.x];
        if constexpr (MASTER) raw.w[q] = s.w[q][threadIdx.x];
        else raw.p[q] = s.w[q][threadIdx.x];
        raw.m[q] = bytes4(s.m[q][threadIdx.x]);
        raw.v[q] = bytes4(s.v[q][threadIdx.x]);
      }
      raw.ms = s.scales[warp][0];
      raw.vs = s.scales[warp][1];
    }
    __syncwarp();  // the slot is read: the next copies may go over it
    fetch(s);
    const AdamTensor<P, G, true, MASTER> a = adam_tensor<P, G, true, MASTER>(tab, at, element);
    float* ms = tab.ms[at] + element / kAdamBlock;
    float* vs = tab.vs[at] + element / kAdamBlock;
    if (left == kAdamBlock) {
      adam_block<true>(a, raw, 0, kAdamBlock, ms, vs, element, tab.index[at], h, f);
    } else if (left > 0 || left == -kAdamBlock) {
      const int count = left > 0 ? left : kAdamBlock;
      raw = adam_load<false>(a, 0, count, ms, vs);
      adam_block<false>(a, raw, 0, count, ms, vs, element, tab.index[at], h, f);
    }
  }
}

template <typename P, typename G, bool EIGHT, bool MASTER, int N>
int launch_table(const mcl4moe_adamw_args* a, int first, int count, const AdamHyper& h, cudaStream_t stream) {
  AdamTable<N> tab;
  int64_t passes = 0;
  for (int i = 0; i < count; ++i) {
    const int t = first + i;
    tab.p[i] = a->params[t];
    tab.g[i] = a->grads[t];
    tab.m[i] = a->exp_avgs[t];
    tab.v[i] = a->exp_avg_sqs[t];
    tab.ms[i] = EIGHT ? a->exp_avg_scales[t] : nullptr;
    tab.vs[i] = EIGHT ? a->exp_avg_sq_scales[t] : nullptr;
    tab.master[i] = MASTER ? a->masters[t] : nullptr;
    tab.numel[i] = a->numels[t];
    tab.index[i] = a->indices ? a->indices[t] : t;
    const uintptr_t state = EIGHT ? 3 : 15;
    tab.wide[i] = (reinterpret_cast<uintptr_t>(tab.p[i]) & (4 * sizeof(P) - 1)) == 0 &&
                  (reinterpret_cast<uintptr_t>(tab.g[i]) & (4 * sizeof(G) - 1)) == 0 &&
                  ((reinterpret_cast<uintptr_t>(tab.m[i]) | reinterpret_cast<uintptr_t>(tab.v[i])) & state) == 0 &&
                  (reinterpret_cast<uintptr_t>(tab.master[i]) & 15) == 0;
    passes += (a->numels[t] + kAdamPass - 1) / kAdamPass;
  }
  // Turns of one pass (8-bit moments: all CTAs sweep one region; turns of four passes 320 us for 291
  // at 94 M elements), with 32-bit moments of four once every SM has a few: 32 KB in a row of each array.
  const int64_t most = int64_t(kAdamCtas) * num_sms();
  tab.passes = EIGHT || passes <= 8 * most ? 1 : 4;
  const int64_t chunk = int64_t(tab.passes) * kAdamPass;
  int64_t turns = 0;
  for (int i = 0; i < count; ++i) {
    tab.first[i] = int32_t(turns);
    turns += (tab.numel[i] + chunk - 1) / chunk;
    if (turns > (int64_t(1) << 30)) return MCL4MOE_ERR_UNSUPPORTED;
  }
  tab.first[count] = int32_t(turns);
  tab.n = count;
  if (turns == 0) return MCL4MOE_OK;
  if constexpr (EIGHT) {
    constexpr int kBytes = kAdamAhead * (kAdamThreads * 2 * (4 * (sizeof(G) + (MASTER ? 4 : sizeof(P))) + 8) + kAdamThreads / 32 * 24);
    static std::atomic<uint64_t> raised{0};
    if (!raise_smem_limit(adamw8_kernel<P, G, MASTER, N>, kBytes, raised)) return MCL4MOE_ERR_CUDA;
    adamw8_kernel<P, G, MASTER, N><<<unsigned(turns < most ? turns : most), kAdamThreads, kBytes, stream>>>(tab, h);
  } else {
    adamw_kernel<P, G, MASTER, N><<<unsigned(turns), kAdamThreads, 0, stream>>>(tab, h);
  }
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

// The tensors' pointers travel as kernel arguments (32764 bytes at most): a small table for few
// tensors, full ones for the rest.
template <typename P, typename G, bool EIGHT, bool MASTER>
int launch_adamw(const mcl4moe_adamw_args* a, const AdamHyper& h, cudaStream_t stream) {
  for (int first = 0; first < a->n;) {
    const int left = a->n - first;
    const int count = left < 440 ? left : 440;
    const int st = count <= 32 ? launch_table<P, G, EIGHT, MASTER, 32>(a, first, count, h, stream)
                               : launch_table<P, G, EIGHT, MASTER, 440>(a, first, count, h, stream);
    if (st != MCL4MOE_OK) return st;
    first += count;
  }
  return MCL4MOE_OK;
}
template <typename P, typename G>
int launch_adamw(const mcl4moe_adamw_args* a, const AdamHyper& h, cudaStream_t stream) {
  if (a->masters) return a->bits == 8 ? launch_adamw<P, G, true, true>(a, h, stream) : launch_adamw<P, G, false, true>(a, h, stream);
  return a->bits == 8 ? launch_adamw<P, G, true, false>(a, h, stream) : launch_adamw<P, G, false, false>(a, h, stream);
}
template <typename P>
int launch_adamw(const mcl4moe_adamw_args* a, const AdamHyper& h, cudaStream_t stream) {
  if (a->grad_dtype == 0) return launch_adamw<P, uint16_t>(a, h, stream);
  if (a->grad_dtype == 1) return launch_adamw<P, float>(a, h, stream);
  return launch_adamw<P, __half>(a, h, stream);
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
    if (a->numels[i] > (int64_t(1) << 42)) return MCL4MOE_ERR_UNSUPPORTED;  // more turns than a grid has, at any size
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
  h.lr = a->lr;
  h.weight_decay = a->weight_decay;
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
  for (uint32_t r = 0; r < 7; ++r) {
    h.keys[2 * r] = uint32_t(a->seed) + r * 0x9E3779B9u;
    h.keys[2 * r + 1] = uint32_t(a->seed >> 32) + r * 0xBB67AE85u;
  }
  if (a->param_dtype == 0) return launch_adamw<uint16_t>(a, h, stream);
  if (a->param_dtype == 1) return launch_adamw<float>(a, h, stream);
  return launch_adamw<__half>(a, h, stream);
}
