// Routing from scores: softmax or sigmoid of the router logits, a selection-only
// bias, group-limited top-k, renormalised and scaled weights, and the gradient.
//
//   s = sigmoid(l) or softmax(l);  key = s + b  (without a bias: l, which orders alike)
//   group value = sum of a group's two best keys, or its best; the top_groups best
//   groups stay open;  ids = the k best keys of the open groups, ties to the lower id
//   w = scale * s / (sum of the chosen s if renormalised)
//
// A masked expert (l or b = -inf) is never chosen; a slot without an expert is id -1,
// weight 0.  NaN keys rank first, as torch.topk has them, and make the row's weights NaN.
//
// The ids are those of exact arithmetic: the float32 keys carry an error bound, and a
// row whose order hangs on less than that bound (neighbouring picks, or the border
// between open and closed groups) is selected again in float64.
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace mcl4 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kScoreWarps = 4;        // rows in flight per CTA, one warp each
constexpr int kMaxScoreExperts = 512;

enum { kSoftmax = 0, kSigmoid = 1 };
enum { kGroupTop2 = 0, kGroupMax = 1 };

struct ScoreArgs {
  const void* logits;
  int64_t ld;
  const float* bias;
  const uint8_t* valid;
  int T, E, k;
  int score, groups, top_groups, group_score, renorm;
  float scale;
  int32_t* idx;
  float* w;
  int32_t* counts;
};

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const uint16_t* p) { return bf16_to_f32(__ldg(p)); }
__device__ __forceinline__ float load_logit(const __half* p) { return __half2float(__ldg(p)); }
__device__ __forceinline__ void store_grad(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_grad(uint16_t* p, float v) { *p = f32_to_bf16(v); }
__device__ __forceinline__ void store_grad(__half* p, float v) { *p = __float2half_rn(v); }

// Unsigned integers in the keys' order; 0 is "not there", NaN is above +inf, -0 equals 0.
__device__ __forceinline__ uint32_t ordered(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
  if (v != v) return ~uint64_t(0);
  const uint64_t b = uint64_t(__double_as_longlong(__dadd_rn(v, 0.0)));
  return b >> 63 ? ~b : b | (uint64_t(1) << 63);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(kFull, v); }
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(kFull, uint32_t(v >> 32));
  const uint32_t lo = __reduce_max_sync(kFull, uint32_t(v >> 32) == hi ? uint32_t(v) : 0u);
  return uint64_t(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t warp_min(uint64_t v) { return ~warp_max(~v); }
__device__ __forceinline__ uint32_t warp_min(uint32_t v) { return __reduce_min_sync(kFull, v); }

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float warp_fmax(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

template <typename F>
struct Order;
template <>
struct Order<float> {
  using U = uint32_t;
};
template <>
struct Order<double> {
  using U = uint64_t;
};

template <typename F>
__device__ __forceinline__ F minus_inf() {
  return F(__int_as_float(0xFF800000));
}
__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// Selects the row's experts: lane j < k returns its pick (-1: none).  F = float: `close`
// tells that the order is within the error bound of the keys.
template <typename F, int NPL>
__device__ __forceinline__ int select_row(const ScoreArgs& a, const float (&l)[NPL], float row_max, float bias_max,
                                          char* smem, bool& close) {
  using U = typename Order<F>::U;
  const int lane = threadIdx.x & 31;
  const int gsize = a.E / a.groups;
  const bool sums = a.groups > 1 && a.group_score == kGroupTop2 && gsize > 1;
  const bool values = a.bias != nullptr || sums;  // else the logits alone give the order, exactly
  // |key - exact key| <= rel * (|key| + bias) with rel = 2^-21.5 for the sigmoid (exp 2 ulp, sum and
  // quotient half an ulp each) and 2^-17.2 for the softmax (l - max rounds to half an ulp of up to
  // 104); twice that for a comparison, with room to spare; 1e-36 covers denormal scores.
  const float rel = a.score == kSigmoid ? 9.5367431640625e-07f : 1.52587890625e-05f;
  auto near = [&](U hi, U lo) {
    if (sizeof(F) == 8 || !values || lo == 0) return false;
    const float x = value_of(uint32_t(hi)), y = value_of(uint32_t(lo));
    return x - y <= rel * (fabsf(x) + fabsf(y) + 8.f * bias_max) + 1e-36f;
  };
  F key[NPL];
  F val[NPL];
  F z = F(1);
  if (values && a.score == kSoftmax) {
    F part = F(0);
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (lane * NPL + i < a.E) part += exp_of(F(l[i]) - F(row_max));
    z = warp_sum(part);
  }
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int e = lane * NPL + i;
    key[i] = val[i] = minus_inf<F>();
    if (e >= a.E) continue;
    key[i] = F(l[i]);
    if (!values) continue;
    const F s = a.score == kSigmoid ? F(1) / (F(1) + exp_of(-F(l[i]))) : exp_of(F(l[i]) - F(row_max)) / z;
    const F b = a.bias != nullptr ? F(__ldg(a.bias + e)) : F(0);
    if (l[i] != minus_inf<float>()) val[i] = a.bias != nullptr ? s + b : s;
    if (a.bias != nullptr) key[i] = val[i];
  }
  close = false;
  U ord[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) ord[i] = key[i] == minus_inf<F>() ? U(0) : ordered(key[i]);
  if (a.groups > 1) {
    F* sv = reinterpret_cast<F*>(smem);
    U* so = reinterpret_cast<U*>(smem + 8 * a.E);
    uint8_t* open = reinterpret_cast<uint8_t*>(smem + 16 * a.E);
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (lane * NPL + i < a.E) sv[lane * NPL + i] = sums ? val[i] : key[i];
    __syncwarp();
    for (int g = lane; g < a.groups; g += 32) {
      F first = minus_inf<F>(), second = minus_inf<F>();
      bool nan = false;
      for (int i = 0; i < gsize; ++i) {
        const F v = sv[g * gsize + i];
        nan |= v != v;
        second = v > first ? first : (v > second ? v : second);
        first = v > first ? v : first;
      }
      if (sums && second != minus_inf<F>()) first += second;
      so[g] = nan ? ~U(0) : first == minus_inf<F>() ? U(0) : ordered(first);
    }
    __syncwarp();
    U lowest_open = ~U(0), highest_closed = 0;
    for (int g = lane; g < a.groups; g += 32) {
      const U mine = so[g];
      int rank = 0;
      for (int h = 0; h < a.groups; ++h) rank += so[h] > mine || (so[h] == mine && h < g);
      open[g] = rank < a.top_groups;
      if (rank < a.top_groups) lowest_open = mine < lowest_open ? mine : lowest_open;
      else highest_closed = mine > highest_closed ? mine : highest_closed;
    }
    lowest_open = warp_min(lowest_open);
    highest_closed = warp_max(highest_closed);
    close = near(lowest_open, highest_closed);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int e = lane * NPL + i;
      if (e < a.E && !open[e / gsize]) ord[i] = 0;
    }
    __syncwarp();
  }
  int pick = -1;
  U before = 0;
  const int rounds = values && sizeof(F) == 4 ? a.k + 1 : a.k;  // one more: the best key left behind
  for (int j = 0; j < rounds; ++j) {
    U best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (ord[i] > best) {
        best = ord[i];
        at = i;
      }
    const U top = warp_max(best);
    if (j > 0 && near(before, top)) close = true;
    if (top == 0) break;
    const int owner = __ffs(__ballot_sync(kFull, best == top)) - 1;
    const int e = __shfl_sync(kFull, lane * NPL + at, owner);
    if (j < a.k && lane == j) pick = e;
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (i == at) ord[i] = 0;
    }
    before = top;
  }
  return pick;
}

// exp(min(l, 0)) / (1 + e^-|l|): denormal, not zero, where 1 + e^-l would overflow.
__device__ __forceinline__ float sigmoid_of(float l) { return expf(fminf(l, 0.f)) / (1.f + expf(-fabsf(l))); }

// exp(min(l, 0) - min(m, 0)) (1 + e^-|m|) / (1 + e^-|l|) = sigmoid(l) / sigmoid(m): no underflow
// of the ratio where both scores underflow.
__device__ __forceinline__ float sigmoid_ratio(float l, float m) {
  return expf(fminf(l, 0.f) - fminf(m, 0.f)) * (1.f + expf(-fabsf(m))) / (1.f + expf(-fabsf(l)));
}

// The chosen score relative to the chosen ones' sum (renorm) or as it is; lanes without a pick: 0.
// `z`, `row_max`: the softmax's, where it is not renormalised.
__device__ __forceinline__ float chosen_share(bool has, float l, int score, int renorm, float row_max, float z) {
  if (!renorm) {
    if (!has) return 0.f;
    return score == kSigmoid ? sigmoid_of(l) : expf(l - row_max) / z;
  }
  // the largest chosen logit (fmaxf passes over NaN, which the ratios carry)
  const float top = warp_fmax(has ? l : minus_inf<float>());
  const float r = !has ? 0.f : score == kSigmoid ? sigmoid_ratio(l, top) : expf(l - top);
  const float sum = warp_sum(r);
  return has ? r / sum : 0.f;
}

template <typename L, int NPL>
__global__ void __launch_bounds__(kScoreWarps * 32) route_scores_kernel(ScoreArgs a) {
  extern __shared__ __align__(16) char smem[];
  int32_t* hist = reinterpret_cast<int32_t*>(smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t hist_bytes = (size_t(a.E) * 4 + 15) / 16 * 16;
  const size_t warp_bytes = (size_t(a.E) * 17 + 15) / 16 * 16;
  char* mine = smem + hist_bytes + warp * warp_bytes;
  if (a.counts != nullptr)
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
  float bias_max = 0.f;
  if (a.bias != nullptr) {
    for (int e = lane; e < a.E; e += 32) {
      const float b = fabsf(__ldg(a.bias + e));
      if (b <= kFltMax) bias_max = fmaxf(bias_max, b);
    }
    bias_max = warp_fmax(bias_max);
  }
  __syncthreads();
  for (int64_t t = int64_t(blockIdx.x) * kScoreWarps + warp; t < a.T; t += int64_t(gridDim.x) * kScoreWarps) {
    const L* row = static_cast<const L*>(a.logits) + t * a.ld;
    int pick = -1;
    float share = 0.f;
    if (a.valid == nullptr || a.valid[t] != 0) {
      float l[NPL];
      float row_max = minus_inf<float>();
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int e = lane * NPL + i;
        l[i] = e < a.E ? load_logit(row + e) : minus_inf<float>();
        row_max = fmaxf(row_max, l[i]);
      }
      row_max = warp_fmax(row_max);
      bool close;
      pick = select_row<float, NPL>(a, l, row_max, bias_max, mine, close);
      if (close) {
        bool ignored;
        pick = select_row<double, NPL>(a, l, row_max, bias_max, mine, ignored);
      }
      float z = 1.f;
      if (a.score == kSoftmax && !a.renorm) {
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (lane * NPL + i < a.E) part += expf(l[i] - row_max);
        z = warp_sum(part);
      }
      const float mine_l = pick >= 0 ? load_logit(row + pick) : 0.f;
      share = chosen_share(pick >= 0, mine_l, a.score, a.renorm, row_max, z);
    }
    if (lane < a.k) {
      a.idx[t * a.k + lane] = pick;
      a.w[t * a.k + lane] = pick >= 0 ? share * a.scale : 0.f;
      if (a.counts != nullptr && pick >= 0) atomicAdd(hist + pick, 1);
    }
  }
  if (a.counts == nullptr) return;
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x)
    if (hist[e] != 0) atomicAdd(a.counts + e, hist[e]);  // whole numbers: the order does not matter
}

struct ScoreBwdArgs {
  const void* logits;
  int64_t ld;
  const int32_t* idx;
  const float* d_w;
  int T, E, k;
  int score, renorm;
  float scale;
  void* d_logits;
};

// One warp per row.  With r the weights before the scale, d = scale * d_w and c = sum r d:
//   renormalised:  dl = r (d - c) [* (1 - s) for the sigmoid] at the chosen, 0 elsewhere
//   sigmoid:       dl = d s (1 - s) at the chosen
//   softmax:       dl = p (d at the chosen - c) everywhere
template <typename L>
__global__ void __launch_bounds__(kScoreWarps * 32) route_scores_bwd_kernel(ScoreBwdArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t t = int64_t(blockIdx.x) * kScoreWarps + warp; t < a.T; t += int64_t(gridDim.x) * kScoreWarps) {
    const L* row = static_cast<const L*>(a.logits) + t * a.ld;
    L* out = static_cast<L*>(a.d_logits) + t * a.E;
    const int pick = lane < a.k ? a.idx[t * a.k + lane] : -1;
    const bool has = pick >= 0 && pick < a.E;
    const bool any = __any_sync(kFull, has);
    const bool dense = a.score == kSoftmax && !a.renorm && any;
    float row_max = minus_inf<float>(), z = 1.f;
    if (dense) {
      for (int e = lane; e < a.E; e += 32) row_max = fmaxf(row_max, load_logit(row + e));
      row_max = warp_fmax(row_max);
      float part = 0.f;
      for (int e = lane; e < a.E; e += 32) part += expf(load_logit(row + e) - row_max);
      z = warp_sum(part);
    }
    const float l = has ? load_logit(row + pick) : 0.f;
    const float d = has ? a.d_w[t * a.k + lane] * a.scale : 0.f;
    const float r = any ? chosen_share(has, l, a.score, a.renorm, row_max, z) : 0.f;
    const float c = warp_sum(has ? r * d : 0.f);
    for (int e = lane; e < a.E; e += 32)
      store_grad(out + e, dense ? -c * (expf(load_logit(row + e) - row_max) / z) : 0.f);
    __syncwarp();  // the chosen entries go over the row written above
    if (has) {
      float g;
      if (a.score == kSoftmax) g = r * (d - c);
      else g = (a.renorm ? r * (d - c) : r * d) * sigmoid_of(-l);  // 1 - sigmoid(l) = sigmoid(-l)
      store_grad(out + pick, g);
    }
  }
}

int check_scores(int64_t T, int E, int k, int dtype, int score) {
  if (T < 0 || E <= 0 || k <= 0 || k > E || dtype < 0 || dtype > 2 || score < 0 || score > 1) return MCL4MOE_ERR_INVALID;
  if (E > kMaxScoreExperts || k > kMaxTopK || T * k > kMaxRoutedSlots) return MCL4MOE_ERR_UNSUPPORTED;
  return MCL4MOE_OK;
}

template <typename L>
cudaError_t launch_scores(const ScoreArgs& a, int grid, size_t smem, cudaStream_t s) {
  const dim3 block(kScoreWarps * 32);
  if (a.E <= 32) route_scores_kernel<L, 1><<<grid, block, smem, s>>>(a);
  else if (a.E <= 64) route_scores_kernel<L, 2><<<grid, block, smem, s>>>(a);
  else if (a.E <= 128) route_scores_kernel<L, 4><<<grid, block, smem, s>>>(a);
  else if (a.E <= 256) route_scores_kernel<L, 8><<<grid, block, smem, s>>>(a);
  else route_scores_kernel<L, 16><<<grid, block, smem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace mcl4

using namespace mcl4;

extern "C" {

int mcl4moe_route_scores(const void* logits, int dtype, int64_t ld, const float* bias, const uint8_t* valid, int64_t T,
                         int E, int k, int score, int groups, int top_groups, int group_score, int renorm, float scale,
                         int32_t* topk_idx, float* topk_w, int32_t* counts, mcl4moe_stream_t stream) {
  int st = check_scores(T, E, k, dtype, score);
  if (st == MCL4MOE_ERR_INVALID) return st;
  if (groups <= 0 || E % groups != 0 || top_groups <= 0 || top_groups > groups || group_score < 0 || group_score > 1 ||
      int64_t(top_groups) * (E / groups) < k || (T > 0 && (!logits || !topk_idx || !topk_w)) || ld < E)
    return MCL4MOE_ERR_INVALID;
  if (st != MCL4MOE_OK) return st;
  if (counts != nullptr && cudaMemsetAsync(counts, 0, sizeof(int32_t) * E, stream) != cudaSuccess)
    return MCL4MOE_ERR_CUDA;
  if (T == 0) return MCL4MOE_OK;
  ScoreArgs a{logits, ld, bias, valid, int(T), E, k, score, groups, top_groups, group_score, renorm != 0, scale,
              topk_idx, topk_w, counts};
  const int64_t blocks = (T + kScoreWarps - 1) / kScoreWarps;
  const int grid = int(blocks < int64_t(16) * num_sms() ? blocks : int64_t(16) * num_sms());
  const size_t smem = (size_t(E) * 4 + 15) / 16 * 16 + kScoreWarps * ((size_t(E) * 17 + 15) / 16 * 16);
  cudaError_t e = dtype == 0   ? launch_scores<uint16_t>(a, grid, smem, stream)
                  : dtype == 1 ? launch_scores<float>(a, grid, smem, stream)
                               : launch_scores<__half>(a, grid, smem, stream);
  return e == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

int mcl4moe_route_scores_backward(const void* logits, int dtype, int64_t ld, const int32_t* topk_idx, const float* d_w,
                                  int64_t T, int E, int k, int score, int renorm, float scale, void* d_logits,
                                  mcl4moe_stream_t stream) {
  int st = check_scores(T, E, k, dtype, score);
  if (st == MCL4MOE_ERR_INVALID) return st;
  if (ld < E || (T > 0 && (!logits || !topk_idx || !d_w || !d_logits))) return MCL4MOE_ERR_INVALID;
  if (st != MCL4MOE_OK) return st;
  if (T == 0) return MCL4MOE_OK;
  ScoreBwdArgs a{logits, ld, topk_idx, d_w, int(T), E, k, score, renorm != 0, scale, d_logits};
  const int64_t blocks = (T + kScoreWarps - 1) / kScoreWarps;
  const int grid = int(blocks < int64_t(16) * num_sms() ? blocks : int64_t(16) * num_sms());
  const dim3 block(kScoreWarps * 32);
  if (dtype == 0) route_scores_bwd_kernel<uint16_t><<<grid, block, 0, stream>>>(a);
  else if (dtype == 1) route_scores_bwd_kernel<float><<<grid, block, 0, stream>>>(a);
  else route_scores_bwd_kernel<__half><<<grid, block, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

}  // extern "C"
