// Routing from scores: softmax or sigmoid of the router logits, a selection-only
// bias, group-limited top-k, renormalised and scaled weights, and the gradient.
//
//   s = sigmoid(l) or softmax(l);  key = s + b  (without a bias: l, which orders alike)
//   group value = sum of a group's two best keys, or its best; the top_groups best
//   groups stay open;  ids = the k best keys of the open groups, ties to the lower id
//   w = scale * s / (sum of the chosen s if renormalised)
//
// A masked expert (l or b = -inf) is never chosen; a slot without an expert is id -1,
// weight 0.  A group with one unmasked expert has that one's key for its value.  NaN keys rank
// first, as torch.topk has them, and make the row's weights NaN.
//
// The ids are those of exact arithmetic: the float32 keys carry an error bound, and a
// row whose order hangs on less than that bound (neighbouring picks, or the border
// between open and closed groups) is selected again in float64, by a whole warp.  The
// bound takes keys for unsettled that are equal because logit and bias are, and it is
// that of a softmax over any span of logits, so the share of such rows is 0.1% for
// float32 logits under a sigmoid, but 22% for bf16 logits under a zero bias (64 experts,
// top 8) and 7 to 22% for a softmax of 256 experts with a bias (top 8 and 16).
//
// A row is a few hundred bytes and a few hundred instructions, so latency bounds it, not HBM: the
// k + 1 rounds of butterfly, ballot and shift follow each other, with 17 warps an SM (96 registers)
// and 58% of the issue slots busy.  A row gets 8, 16 or 32 lanes with up to 8 experts in each one's
// registers (16 above 256 experts), so that the rounds serve up to four rows at once, on lists that
// each lane has sorted.  32768 x 64, sigmoid, bias, 4 of 8 groups, top 8: 31 us (a warp a row: 51 us);
// softmax without groups 20 us; 16383 x 256 with groups 45 us; 32768 x 64 bf16 with a zero bias 49 us
// (float32: 29 us), the difference in float64.  Gradients: 10 us for 32768 x 64, 18 us for 32768 x 256,
// 16 us for the dense one of 65536 x 40 bf16.
//
// The scores of the weights and gradients are float32 throughout, with approximate quotients (2 ulp
// each): a mean error of 1.1e-7 with 256 experts, two float32 roundings, on weights that the experts'
// combine rounds to bf16.
#include <type_traits>

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace mcl4 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kScoreWarps = 4;        // of a CTA
constexpr int kScoreWarpsOne = 16;    // of the one CTA that a small batch fits into
constexpr int kMaxScoreExperts = 512;

constexpr int32_t kUnsure = -2;

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
  int one;   // a single CTA: it writes the counts itself
  int wide;  // rows allow 16-byte loads
};

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const uint16_t* p) { return bf16_to_f32(__ldg(p)); }
__device__ __forceinline__ float load_logit(const __half* p) { return __half2float(__ldg(p)); }
__device__ __forceinline__ float logit_value(float v) { return v; }
__device__ __forceinline__ float logit_value(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float logit_value(__half v) { return __half2float(v); }
__device__ __forceinline__ void store_grad(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_grad(uint16_t* p, float v) { *p = f32_to_bf16(v); }
__device__ __forceinline__ void store_grad(__half* p, float v) { *p = __float2half_rn(v); }

// Unsigned integers in the keys' order; 0 is "not there", NaN is above +inf, -0 equals 0.
__device__ __forceinline__ uint64_t ordered(double v) {
  if (v != v) return ~uint64_t(0);
  const uint64_t b = uint64_t(__double_as_longlong(__dadd_rn(v, 0.0)));
  return b >> 63 ? ~b : b | (uint64_t(1) << 63);
}

// Butterflies over the LPT lanes of a row.
template <int LPT, typename F, typename Op>
__device__ __forceinline__ F lanes(F v, Op op) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <int LPT, typename F>
__device__ __forceinline__ F lanes_sum(F v) {
  return lanes<LPT>(v, [](F a, F b) { return a + b; });
}
template <int LPT>
__device__ __forceinline__ float lanes_fmax(float v) {
  return lanes<LPT>(v, [](float a, float b) { return fmaxf(a, b); });
}
// The largest of a row's lanes (no NaN).
template <int LPT>
__device__ __forceinline__ float lanes_top(float v) {
  if constexpr (LPT == 32) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
  } else {
    return lanes_fmax<LPT>(v);
  }
}

// Batcher's odd-even merge sort as a list of compare-exchange pairs.
template <int N>
struct SortPairs {
  int n = 0;
  int lo[64] = {}, hi[64] = {};
  constexpr SortPairs() {
    for (int p = 1; p < N; p *= 2)
      for (int k = p; k >= 1; k /= 2)
        for (int j = k % p; j + k < N; j += 2 * k)
          for (int i = 0; i < k && i + j + k < N; ++i)
            if ((i + j) / (2 * p) == (i + j + k) / (2 * p)) {
              lo[n] = i + j;
              hi[n] = i + j + k;
              ++n;
            }
  }
};
// Sorts a lane's keys, falling, ties by place; returns the places, four bits each, best lowest.
template <int N>
using Places = typename std::conditional<(N > 8), uint64_t, uint32_t>::type;
template <int N>
__device__ __forceinline__ Places<N> sort_lane(float (&key)[N]) {
  constexpr SortPairs<N> pairs;
  int at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = i;
#pragma unroll
  for (int c = 0; c < pairs.n; ++c) {
    const int i = pairs.lo[c], j = pairs.hi[c];
    const float a = key[i], b = key[j];
    const int x = at[i], y = at[j];
    const bool swap = b > a || (b == a && y < x);
    key[i] = swap ? b : a;
    key[j] = swap ? a : b;
    at[i] = swap ? y : x;
    at[j] = swap ? x : y;
  }
  Places<N> places = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) places |= Places<N>(at[i]) << (4 * i);
  return places;
}

__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(kFull, uint32_t(v >> 32));
  const uint32_t lo = __reduce_max_sync(kFull, uint32_t(v >> 32) == hi ? uint32_t(v) : 0u);
  return uint64_t(hi) << 32 | lo;
}

__device__ __forceinline__ float minus_inf() { return __uint_as_float(0xFF800000u); }

// What a warp keeps in shared memory for its rows (32 / LPT of them): values and group values of
// rows whose groups do not fall on lanes, and the picks (one more: the best key left behind).
struct ScoreScratch {
  double* val;     // [slots] (float32 values of the rows side by side, or one row's float64 values)
  uint64_t* ord;   // [slots]
  uint8_t* open;   // [slots]
  int32_t* pick;   // [rows][33]
};
__host__ __device__ inline int score_slots(int E, int lpt) { return (32 / lpt * E + 15) / 16 * 16; }
__host__ __device__ inline size_t score_scratch_bytes(int E, int lpt) {
  return size_t(score_slots(E, lpt)) * 17 + size_t(32 / lpt) * 33 * 4 + 12;
}

// exp(min(l, 0)) / (1 + e^-|l|): denormal, not zero, where 1 + e^-l would overflow.
__device__ __forceinline__ float sigmoid_of(float l) { return __fdividef(expf(fminf(l, 0.f)), 1.f + expf(-fabsf(l))); }

// exp(min(l, 0) - min(m, 0)) (1 + e^-|m|) / (1 + e^-|l|) = sigmoid(l) / sigmoid(m): no underflow
// of the ratio where both scores underflow.
__device__ __forceinline__ float sigmoid_ratio(float l, float m) {
  return __fdividef(expf(fminf(l, 0.f) - fminf(m, 0.f)) * (1.f + expf(-fabsf(m))), 1.f + expf(-fabsf(l)));
}

// Vector loads and stores of a lane's experts: NPL consecutive elements from e0 on.
template <int NPL, typename L>
__device__ __forceinline__ void load_lane(const L* row, int e0, int E, bool wide, float (&l)[NPL]) {
  constexpr int kPer = 16 / int(sizeof(L));
  if constexpr (NPL % kPer == 0) {
    if (wide && e0 < E) {  // wide: E is a multiple of NPL, so a lane's experts are all there or none
#pragma unroll
      for (int q = 0; q < NPL / kPer; ++q) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + e0) + q);
        const L* v = reinterpret_cast<const L*>(&w);
#pragma unroll
        for (int i = 0; i < kPer; ++i) l[q * kPer + i] = logit_value(v[i]);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NPL; ++i) l[i] = e0 + i < E ? load_logit(row + e0 + i) : minus_inf();
}
template <int NPL, typename L>
__device__ __forceinline__ void store_lane(L* row, int e0, int E, bool wide, const float (&v)[NPL]) {
  constexpr int kPer = 16 / int(sizeof(L));
  if constexpr (NPL % kPer == 0) {
    if (wide && e0 < E) {
#pragma unroll
      for (int q = 0; q < NPL / kPer; ++q) {
        uint4 w;
        L* o = reinterpret_cast<L*>(&w);
#pragma unroll
        for (int i = 0; i < kPer; ++i) store_grad(o + i, v[q * kPer + i]);
        reinterpret_cast<uint4*>(row + e0)[q] = w;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NPL; ++i)
    if (e0 + i < E) store_grad(row + e0 + i, v[i]);
}

// The chosen scores of a row's lanes, lane j % LPT holding pick j in slot j / LPT: relative to their
// sum (renorm), or as they are.  Slots without a pick get 0.
template <int LPT>
__device__ __forceinline__ void chosen_shares(const bool (&has)[32 / LPT], const float (&l)[32 / LPT], int slots, int score,
                                              int renorm, float row_max, float z, float (&share)[32 / LPT]) {
  if (!renorm) {
#pragma unroll
    for (int q = 0; q < 32 / LPT; ++q) {
      share[q] = 0.f;
      if (q < slots && has[q]) share[q] = score == kSigmoid ? sigmoid_of(l[q]) : expf(l[q] - row_max) / z;
    }
    return;
  }
  float top = minus_inf();  // the largest chosen logit (fmaxf passes over NaN, which the ratios carry)
#pragma unroll
  for (int q = 0; q < 32 / LPT; ++q)
    if (q < slots && has[q]) top = fmaxf(top, l[q]);
  top = lanes_fmax<LPT>(top);
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < 32 / LPT; ++q) {
    share[q] = 0.f;
    if (q < slots && has[q]) share[q] = score == kSigmoid ? sigmoid_ratio(l[q], top) : expf(l[q] - top);
    sum += share[q];
  }
  sum = lanes_sum<LPT>(sum);
#pragma unroll
  for (int q = 0; q < 32 / LPT; ++q)
    if (q < slots && has[q]) share[q] = __fdividef(share[q], sum);
}

// A row whose order float32 does not settle, by a whole warp in float64: N experts a lane.  It is
// called behind the main loop: a call inside would cost every row its register spills (270 of 790
// instructions a pass).  What it takes is one row's
// latency, most of that the fetch of code that no other warp runs: hence the short loops.
template <typename L, int N>
__device__ __noinline__ void select_exact(const ScoreArgs& a, int64_t t, ScoreScratch s, int32_t* hist) {
  const L* row = static_cast<const L*>(a.logits) + t * a.ld;
  int32_t* pick = s.pick;
  const int lane = threadIdx.x & 31, e0 = lane * N;
  const int gsize = a.E / a.groups;
  const bool sums = a.groups > 1 && a.group_score == kGroupTop2 && gsize > 1;
  const double none = double(minus_inf());
  double top = none, z = 1.0;
  if (a.score == kSoftmax) {
    for (int e = lane; e < a.E; e += 32) top = fmax(top, double(load_logit(row + e)));
    top = lanes<32>(top, [](double x, double y) { return fmax(x, y); });
    double part = 0.0;
#pragma unroll 1
    for (int e = lane; e < a.E; e += 32) part += exp(double(load_logit(row + e)) - top);
    z = lanes_sum<32>(part);
  }
  __syncwarp();
#pragma unroll 1
  for (int e = lane; e < a.E; e += 32) {
    const float lf = load_logit(row + e);
    const double l = double(lf), x = exp(a.score == kSigmoid ? -l : l - top);
    const double score = (a.score == kSigmoid ? 1.0 : x) / (a.score == kSigmoid ? 1.0 + x : z);
    const float b = a.bias != nullptr ? __ldg(a.bias + e) : 0.f;
    // masked by its logit or by its bias, which a NaN score would swallow
    const double v = lf == minus_inf() || b == minus_inf() ? none : score + double(b);
    const double key = a.bias != nullptr ? v : l;
    s.val[e] = sums ? v : key;
    s.ord[e] = key == none ? 0 : ordered(key);
  }
  __syncwarp();
  uint64_t ord[N];
#pragma unroll
  for (int i = 0; i < N; ++i) ord[i] = e0 + i < a.E ? s.ord[e0 + i] : 0;
  __syncwarp();
  if (a.groups > 1) {
    for (int g = lane; g < a.groups; g += 32) {
      double first = none, second = none;
      bool nan = false;
#pragma unroll 1
      for (int i = 0; i < gsize; ++i) {
        const double v = s.val[g * gsize + i];
        nan |= v != v;
        second = v > first ? first : (v > second ? v : second);
        first = v > first ? v : first;
      }
      if (sums && second != none) first += second;
      s.ord[g] = nan ? ~uint64_t(0) : first == none ? 0 : ordered(first);
    }
    __syncwarp();
    for (int g = lane; g < a.groups; g += 32) {
      const uint64_t mine = s.ord[g];
      int rank = 0;
#pragma unroll 1
      for (int h = 0; h < a.groups; ++h) rank += s.ord[h] > mine || (s.ord[h] == mine && h < g);
      s.open[g] = rank < a.top_groups;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (e0 + i < a.E && !s.open[(e0 + i) / gsize]) ord[i] = 0;
  }
  __syncwarp();
#pragma unroll 1
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = ord[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (ord[i] > best) {
        best = ord[i];
        at = i;
      }
    const uint64_t top_key = warp_max64(best);
    const unsigned held = __ballot_sync(kFull, best == top_key);
    if (lane == __ffs(held) - 1) {  // the lowest lane that has it, and its first
      pick[j] = top_key == 0 ? -1 : e0 + at;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i == at) ord[i] = 0;
    }
  }
  __syncwarp();
  float row_max = 0.f, sum = 1.f;
  if (a.score == kSoftmax && !a.renorm) {
    row_max = float(top);
    float part = 0.f;
    for (int e = lane; e < a.E; e += 32) part += expf(load_logit(row + e) - row_max);
    sum = lanes_sum<32>(part);
  }
  const int32_t id = lane < a.k ? pick[lane] : -1;
  const bool has[1] = {id >= 0};
  const float l[1] = {has[0] ? load_logit(row + id) : 0.f};
  float share[1];
  chosen_shares<32>(has, l, 1, a.score, a.renorm, row_max, sum, share);
  // a NaN or +inf logit makes every score of a softmax NaN, that of experts chosen by other keys too
  if (a.score == kSoftmax && z != z) share[0] = __uint_as_float(0x7FFFFFFFu);
  if (lane < a.k) {
    a.idx[t * a.k + lane] = id;
    a.w[t * a.k + lane] = has[0] ? share[0] * a.scale : 0.f;
    if (a.counts != nullptr && has[0]) atomicAdd(hist + id, 1);
  }
  __syncwarp();
}

// WARPS of a CTA at most: the one CTA of a small batch has many, the others stay at few and more registers.
template <typename L, int LPT, int NPL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) route_scores_kernel(ScoreArgs a) {
  extern __shared__ __align__(16) char smem[];
  constexpr int kRows = 32 / LPT;  // of a warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int seg = lane / LPT, sl = lane % LPT;
  const unsigned seg_mask = LPT == 32 ? kFull : ((1u << LPT) - 1u);
  int32_t* hist = reinterpret_cast<int32_t*>(smem);
  ScoreScratch s;
  {
    const int slots = score_slots(a.E, LPT);
    char* at = smem + (size_t(a.E) * 4 + 15) / 16 * 16 + warp * ((score_scratch_bytes(a.E, LPT) + 15) / 16 * 16);
    s.val = reinterpret_cast<double*>(at);
    s.ord = reinterpret_cast<uint64_t*>(at + size_t(slots) * 8);
    s.pick = reinterpret_cast<int32_t*>(at + size_t(slots) * 16);
    s.open = reinterpret_cast<uint8_t*>(s.pick + kRows * 33);
  }
  if (a.counts != nullptr)
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
  float bias_max = 0.f;
  if (a.bias != nullptr) {
    for (int e = lane; e < a.E; e += 32) {
      const float b = fabsf(__ldg(a.bias + e));
      if (b <= kFltMax) bias_max = fmaxf(bias_max, b);
    }
    bias_max = lanes_fmax<32>(bias_max);
  }
  __syncthreads();
  const int gsize = a.E / a.groups;
  const bool sums = a.groups > 1 && a.group_score == kGroupTop2 && gsize > 1;
  const bool values = a.bias != nullptr || sums;  // else the logits alone give the order, exactly
  // groups of 1, 2, 4 .. whole lanes are valued by butterflies
  const int glanes = gsize / NPL;
  const bool on_lanes = a.groups > 1 && gsize % NPL == 0 && (glanes & (glanes - 1)) == 0;
  const bool soft = a.score == kSoftmax && (values || !a.renorm);
  const bool wide = a.wide && a.E % NPL == 0;
  // |key - exact key| <= u * (|key| + |bias|): sigmoid u = 2^-21.1 (exp 2 ulp, sum half an ulp, reciprocal
  // 1 ulp, the key's own rounding), softmax 2^-17.2 (l - max rounds to half an ulp of up to 104).  Two keys
  // are told apart if they differ by more than rel * (2 |larger| + 8 max|bias|), rel = 1.5 u and 2.3 u;
  // 1e-36 covers denormal scores.
  const float rel = a.score == kSigmoid ? 6.7e-07f : 1.52587890625e-05f;
  // (y <= x, and where |y| > |x| it is at most |x| + (x - y); false for an infinite x or y)
  const float near_abs = values ? rel * 8.f * bias_max + 1e-36f : -1.f, near_rel = values ? 2.f * rel : 0.f;
  auto near = [&](float x, float y) { return x - y <= near_rel * fminf(fabsf(x), kFltMax) + near_abs; };
  const int e0 = sl * NPL;
  float bias[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) bias[i] = a.bias != nullptr && e0 + i < a.E ? __ldg(a.bias + e0 + i) : 0.f;
  const int slots = (a.k + LPT - 1) / LPT;
  int32_t* pick = s.pick + seg * 33;
  const unsigned lower = (1u << sl) - 1u;  // the row's lanes below this one
  bool any_unsure = false;  // rows of this warp marked for float64

  for (int64_t base = (int64_t(blockIdx.x) * warps + warp) * kRows; base < a.T; base += int64_t(gridDim.x) * warps * kRows) {
    const int64_t t = base + seg;
    const bool live = t < a.T && (a.valid == nullptr || a.valid[t] != 0);
    const L* row = static_cast<const L*>(a.logits) + (live ? t : 0) * a.ld;
    float l[NPL];
    if (live) {
      load_lane(row, e0, a.E, wide, l);
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (!live) l[i] = minus_inf();
    float row_max = 0.f, z = 1.f;
    if (soft) {
      row_max = l[0];
#pragma unroll
      for (int i = 1; i < NPL; ++i) row_max = fmaxf(row_max, l[i]);
      row_max = lanes_fmax<LPT>(row_max);
    }
    float val[NPL];  // the scores, with the bias: what keys and group values are made of
    if (values || soft) {
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (a.score == kSigmoid) {
          asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(val[i]) : "f"(1.f + expf(-l[i])));
        } else {
          val[i] = e0 + i < a.E ? expf(l[i] - row_max) : 0.f;
          part += val[i];
        }
      }
      if (soft) z = lanes_sum<LPT>(part);
      const float scale = soft ? 1.f / z : 1.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) val[i] = l[i] == minus_inf() ? minus_inf() : val[i] * scale + bias[i];
    }
    float key[NPL];  // -inf: not there
    bool close = false;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      key[i] = e0 + i < a.E ? (a.bias != nullptr ? val[i] : l[i]) : minus_inf();
      close |= key[i] != key[i];  // NaN ranks first: the float64 selection knows how
    }
    if (a.groups > 1) {
      if (on_lanes) {
        float first = minus_inf(), second = minus_inf();
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
          const float v = sums && e0 + i < a.E ? val[i] : key[i];
          close |= v != v;
          second = fmaxf(second, fminf(first, v));
          first = fmaxf(first, v);
        }
        for (int o = 1; o < glanes; o <<= 1) {
          const float f2 = __shfl_xor_sync(kFull, first, o), s2 = __shfl_xor_sync(kFull, second, o);
          second = fmaxf(fmaxf(second, s2), fminf(first, f2));
          first = fmaxf(first, f2);
        }
        const float mine = sums && second != minus_inf() ? first + second : first;
        const int g = sl / glanes;
        float below = minus_inf();  // the best group behind this one
        int rank = 0;
        for (int h = 0; h < a.groups; ++h) {
          const float o = __shfl_sync(kFull, mine, h * glanes, LPT);
          const bool ahead = o > mine || (o == mine && h < g);
          rank += ahead;
          if (!ahead && h != g) below = fmaxf(below, o);
        }
        close |= rank == a.top_groups - 1 && near(mine, below);
        if (rank >= a.top_groups) {
#pragma unroll
          for (int i = 0; i < NPL; ++i) key[i] = minus_inf();
        }
      } else {
        float* sv = reinterpret_cast<float*>(s.val) + seg * a.E;
        float* so = reinterpret_cast<float*>(s.ord) + seg * a.E;
        uint8_t* open = s.open + seg * a.E;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (e0 + i < a.E) sv[e0 + i] = sums ? val[i] : key[i];
        __syncwarp();
        for (int g = sl; g < a.groups; g += LPT) {
          float first = minus_inf(), second = minus_inf();
          for (int i = 0; i < gsize; ++i) {
            const float v = sv[g * gsize + i];
            close |= v != v;
            second = fmaxf(second, fminf(first, v));
            first = fmaxf(first, v);
          }
          so[g] = sums && second != minus_inf() ? first + second : first;
        }
        __syncwarp();
        for (int g = sl; g < a.groups; g += LPT) {
          const float mine = so[g];
          float below = minus_inf();
          int rank = 0;
          for (int h = 0; h < a.groups; ++h) {
            const float o = so[h];
            const bool ahead = o > mine || (o == mine && h < g);
            rank += ahead;
            if (!ahead && h != g) below = fmaxf(below, o);
          }
          open[g] = rank < a.top_groups;
          close |= rank == a.top_groups - 1 && near(mine, below);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (e0 + i < a.E && !open[(e0 + i) / gsize]) key[i] = minus_inf();
      }
    }
    Places<NPL> places = sort_lane(key);
    __syncwarp();  // the last rows' picks are read
    const int rounds = values ? a.k + 1 : a.k;  // one more: the best key left behind
    float before = __uint_as_float(0x7F800000u);
    for (int j = 0; j < rounds; ++j) {
      const float top = lanes_top<LPT>(key[0]);
      const bool mine = key[0] == top;
      const unsigned held = __ballot_sync(kFull, mine) >> (seg * LPT) & seg_mask;
      close |= near(before, top);
      before = top;
      const bool goes = mine && (held & lower) == 0;  // the lowest lane that has it: its best goes
      if (goes) pick[j] = top == minus_inf() ? -1 : e0 + int(places & 15);
      places = goes ? places >> 4 : places;
#pragma unroll
      for (int i = 0; i + 1 < NPL; ++i) key[i] = goes ? key[i + 1] : key[i];
      key[NPL - 1] = goes ? minus_inf() : key[NPL - 1];
    }
    __syncwarp();
    const unsigned unsure = __ballot_sync(kFull, close) >> (seg * LPT) & seg_mask;
    any_unsure |= __any_sync(kFull, close);
    // An unsure row's picks are not read: where every lane's best is NaN, no lane equals the largest
    // and a round writes none.  A NaN key makes its row unsure, so a settled row has all its picks.
    int id[kRows];
    bool has[kRows];
    float lc[kRows], share[kRows];
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int j = q * LPT + sl;
      id[q] = unsure == 0 && q < slots && j < a.k ? pick[j] : -1;
      has[q] = id[q] >= 0;
      lc[q] = has[q] ? load_logit(row + id[q]) : 0.f;
    }
    chosen_shares<LPT>(has, lc, slots, a.score, a.renorm, row_max, z, share);
    if (t < a.T && unsure != 0) {
      if (sl == 0) a.idx[t * a.k] = kUnsure;
    } else if (t < a.T) {
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        const int j = q * LPT + sl;
        if (q >= slots || j >= a.k) continue;
        a.idx[t * a.k + j] = id[q];
        a.w[t * a.k + j] = has[q] ? share[q] * a.scale : 0.f;
        if (a.counts != nullptr && has[q]) atomicAdd(hist + id[q], 1);
      }
    }
  }
  __syncwarp();
  if (any_unsure)
    for (int64_t base = (int64_t(blockIdx.x) * warps + warp) * kRows; base < a.T; base += int64_t(gridDim.x) * warps * kRows)
      for (int r = 0; r < kRows && base + r < a.T; ++r) {
        const int32_t mark = __shfl_sync(kFull, lane == 0 ? *const_cast<volatile int32_t*>(a.idx + (base + r) * a.k) : 0, 0);
        if (mark == kUnsure) select_exact<L, (LPT * NPL + 31) / 32>(a, base + r, s, hist);
      }
  if (a.counts == nullptr) return;
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    if (a.one) a.counts[e] = hist[e];
    else if (hist[e] != 0) atomicAdd(a.counts + e, hist[e]);  // whole numbers: the order does not matter
  }
}

struct ScoreBwdArgs {
  const void* logits;
  int64_t ld;
  const int32_t* idx;
  const float* d_w;
  int T, E, k;
  int score, renorm, wide;
  float scale;
  void* d_logits;
};

// With r the weights before the scale, d = scale * d_w and c = sum r d:
//   renormalised:  dl = r (d - c) [* (1 - s) for the sigmoid] at the chosen, 0 elsewhere
//   sigmoid:       dl = d s (1 - s) at the chosen
//   softmax:       dl = p (d at the chosen - c) everywhere
template <typename L, int LPT, int NPL>
__global__ void __launch_bounds__(kScoreWarps * 32) route_scores_bwd_kernel(ScoreBwdArgs a) {
  constexpr int kRows = 32 / LPT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = lane / LPT, sl = lane % LPT, e0 = sl * NPL;
  const int slots = (a.k + LPT - 1) / LPT;
  const bool wide = a.wide && a.E % NPL == 0;
  for (int64_t base = (int64_t(blockIdx.x) * kScoreWarps + warp) * kRows; base < a.T;
       base += int64_t(gridDim.x) * kScoreWarps * kRows) {
    const int64_t t = base + seg;
    const bool live = t < a.T;
    const L* row = static_cast<const L*>(a.logits) + (live ? t : 0) * a.ld;
    L* out = static_cast<L*>(a.d_logits) + (live ? t : 0) * a.E;
    int id[kRows];
    bool has[kRows];
    float lc[kRows], d[kRows], share[kRows];
    bool any = false;
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int j = q * LPT + sl;
      id[q] = live && q < slots && j < a.k ? a.idx[t * a.k + j] : -1;
      has[q] = id[q] >= 0 && id[q] < a.E;
      any |= has[q];
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      lc[q] = has[q] ? load_logit(row + id[q]) : 0.f;
      d[q] = has[q] ? a.d_w[t * a.k + q * LPT + sl] * a.scale : 0.f;
    }
    // the dense gradient reads the whole row; a row without picks keeps zeros whatever it holds
    any = lanes<LPT>(int(any), [](int x, int y) { return x | y; }) != 0;
    float g[NPL];
    float row_max = 0.f, z = 1.f;
    const bool dense = a.score == kSoftmax && !a.renorm;
    if (dense) {
      load_lane(row, e0, a.E, wide, g);
      row_max = g[0];
#pragma unroll
      for (int i = 1; i < NPL; ++i) row_max = fmaxf(row_max, g[i]);
      row_max = lanes_fmax<LPT>(row_max);
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        g[i] = e0 + i < a.E ? expf(g[i] - row_max) : 0.f;
        part += g[i];
      }
      z = lanes_sum<LPT>(part);
    }
    chosen_shares<LPT>(has, lc, slots, a.score, a.renorm, row_max, z, share);
    float c = 0.f;
#pragma unroll
    for (int q = 0; q < kRows; ++q)
      if (has[q]) c += share[q] * d[q];
    c = lanes_sum<LPT>(c);
    const float factor = -c / z;
#pragma unroll
    for (int i = 0; i < NPL; ++i) g[i] = dense && any ? factor * g[i] : 0.f;
    if (live) store_lane(out, e0, a.E, wide, g);
    __syncwarp();  // the chosen entries go over the row written above
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      if (!has[q]) continue;
      float v = a.score == kSoftmax || a.renorm ? share[q] * (d[q] - c) : share[q] * d[q];
      if (a.score == kSigmoid) v *= sigmoid_of(-lc[q]);  // 1 - sigmoid(l) = sigmoid(-l)
      store_grad(out + id[q], v);
    }
  }
}

int check_scores(int64_t T, int E, int k, int dtype, int score) {
  if (T < 0 || E <= 0 || k <= 0 || k > E || dtype < 0 || dtype > 2 || score < 0 || score > 1) return MCL4MOE_ERR_INVALID;
  if (E > kMaxScoreExperts || k > kMaxTopK || T > kMaxRoutedSlots / k) return MCL4MOE_ERR_UNSUPPORTED;
  return MCL4MOE_OK;
}

// Lanes of a row and experts of a lane: 8 lanes up to 64 experts, 16 up to 128, else 32.
template <typename F>
void score_shape(int E, F&& f) {
  using std::integral_constant;
  const auto pick = [&](auto lpt, auto npl) { f(lpt, npl); };
  if (E <= 8) pick(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  else if (E <= 16) pick(integral_constant<int, 8>{}, integral_constant<int, 2>{});
  else if (E <= 32) pick(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  else if (E <= 64) pick(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  else if (E <= 128) pick(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  else if (E <= 256) pick(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  else pick(integral_constant<int, 32>{}, integral_constant<int, 16>{});
}

template <typename L>
bool rows_wide(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * int64_t(sizeof(L)) % 16 == 0;
}

template <typename L>
int launch_scores(ScoreArgs a, cudaStream_t stream) {
  int st = MCL4MOE_OK;
  score_shape(a.E, [&](auto lpt, auto npl) {
    constexpr int kLpt = decltype(lpt)::value, kNpl = decltype(npl)::value;
    a.wide = rows_wide<L>(a.logits, a.ld);
    // a batch that one CTA's warps hold in one pass: no counts to clear beforehand
    a.one = a.T <= kScoreWarpsOne * (32 / kLpt);
    const int warps = a.one ? (a.T + 32 / kLpt - 1) / (32 / kLpt) : kScoreWarps;
    const int64_t blocks = (a.T + int64_t(warps) * (32 / kLpt) - 1) / (int64_t(warps) * (32 / kLpt));
    // as many CTAs as are resident (32768 x 256 softmax 102 -> 90 us from 8 an SM), but the widest rows
    // leave more of their latency to others (16384 x 512: 86 us, 96 with 5)
    const int64_t most = int64_t(kLpt * kNpl > 256 ? 8 : 5) * num_sms();
    const size_t smem = (size_t(a.E) * 4 + 15) / 16 * 16 + warps * ((score_scratch_bytes(a.E, kLpt) + 15) / 16 * 16);
    static std::atomic<uint64_t> raised{0};
    if (!raise_smem_limit(route_scores_kernel<L, kLpt, kNpl, kScoreWarpsOne>, 200 * 1024, raised) ||
        (!a.one && a.counts != nullptr && cudaMemsetAsync(a.counts, 0, sizeof(int32_t) * a.E, stream) != cudaSuccess)) {
      st = MCL4MOE_ERR_CUDA;
      return;
    }
    const unsigned grid = unsigned(blocks < most ? blocks : most);
    if (a.one) route_scores_kernel<L, kLpt, kNpl, kScoreWarpsOne><<<grid, warps * 32, smem, stream>>>(a);
    else route_scores_kernel<L, kLpt, kNpl, kScoreWarps><<<grid, warps * 32, smem, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) st = MCL4MOE_ERR_CUDA;
  });
  return st;
}

template <typename L>
int launch_scores_bwd(ScoreBwdArgs a, cudaStream_t stream) {
  a.wide = rows_wide<L>(a.logits, a.ld) && rows_wide<L>(a.d_logits, a.E);
  score_shape(a.E, [&](auto lpt, auto npl) {
    constexpr int kLpt = decltype(lpt)::value, kNpl = decltype(npl)::value;
    const int64_t blocks = (a.T + int64_t(kScoreWarps) * (32 / kLpt) - 1) / (int64_t(kScoreWarps) * (32 / kLpt));
    const int64_t most = int64_t(16) * num_sms();
    route_scores_bwd_kernel<L, kLpt, kNpl><<<unsigned(blocks < most ? blocks : most), kScoreWarps * 32, 0, stream>>>(a);
  });
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
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
  if (T == 0) {
    if (counts != nullptr && cudaMemsetAsync(counts, 0, sizeof(int32_t) * E, stream) != cudaSuccess)
      return MCL4MOE_ERR_CUDA;
    return MCL4MOE_OK;
  }
  const ScoreArgs a{logits, ld, bias, valid, int(T), E, k, score, groups, top_groups, group_score, renorm != 0, scale,
                    topk_idx, topk_w, counts, 0, 0};
  return dtype == 0 ? launch_scores<uint16_t>(a, stream)
                    : dtype == 1 ? launch_scores<float>(a, stream) : launch_scores<__half>(a, stream);
}

int mcl4moe_route_scores_backward(const void* logits, int dtype, int64_t ld, const int32_t* topk_idx, const float* d_w,
                                  int64_t T, int E, int k, int score, int renorm, float scale, void* d_logits,
                                  mcl4moe_stream_t stream) {
  int st = check_scores(T, E, k, dtype, score);
  if (st == MCL4MOE_ERR_INVALID) return st;
  if (ld < E || (T > 0 && (!logits || !topk_idx || !d_w || !d_logits))) return MCL4MOE_ERR_INVALID;
  if (st != MCL4MOE_OK) return st;
  if (T == 0) return MCL4MOE_OK;
  const ScoreBwdArgs a{logits, ld, topk_idx, d_w, int(T), E, k, score, renorm != 0, 0, scale, d_logits};
  return dtype == 0 ? launch_scores_bwd<uint16_t>(a, stream)
                    : dtype == 1 ? launch_scores_bwd<float>(a, stream) : launch_scores_bwd<__half>(a, stream);
}

}  // extern "C"
