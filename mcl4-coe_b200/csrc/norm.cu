// The norms around a block with its gate and residual sum, in one pass each way:
//
//   n = u rsqrt(mean(u^2) + eps) w_post      (n = u without w_post)
//   y = rs x + bs act(g) n                   (act(g) = 1 without a gate; y = x without a branch)
//   h = y rsqrt(mean(y^2) + eps) w_pre       (only with w_pre)
//
// Backward, with dz = dy + r_y (w_pre dh - yh mean(w_pre dh yh)), yh = y r_y:
//   dx = rs dz;  dn = bs act(g) dz;  dg = bs act'(g) n dz;  dw_pre = sum over rows of dh yh
//   du = r_u (w_post dn - uh mean(w_post dn uh)), uh = u r_u;  dw_post = sum of dn uh
// y is computed again from x and u, in float32: the rounded output would put its rounding into
// the float32 weight gradients.  All arithmetic is float32; each output is rounded once.
//
// Both directions are bound by HBM (forward 2 reads and 2 writes of a row, backward 4 and 2), so a
// row is read once: it stays in the registers of its team (a warp for up to 256 columns, else a
// CTA, 8 or 16 columns a thread) between the reductions, and the next row's loads are issued
// before them.  Teams are persistent, which keeps the columns' factors in registers and, in the
// backward, the column sums: a row of partial sums per team, added afterwards in their order.
// With one gate row per part of the rows, dw_post and dg both come from one column sum
//   S = sum over rows of dz uh:  dw_post = bs act(g) S,  dg = bs act'(g) w_post S.
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace mcl4 {
namespace {

constexpr int kMaxNormCols = 16384;
constexpr int kNormThreads = 256;   // of the generic kernels
constexpr int kTeamCols = 8192;     // the widest row that a team keeps in registers

enum { kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateFull = 3 };
enum { kActNone = 0, kActSigmoid = 1, kActTanh = 2 };

using NormArgs = mcl4moe_norm_args;

__device__ __forceinline__ float load_f(const void* p, int dtype, int64_t i) {
  if (dtype == 0) return bf16_to_f32(__ldg(static_cast<const uint16_t*>(p) + i));
  if (dtype == 1) return __ldg(static_cast<const float*>(p) + i);
  return __half2float(__ldg(static_cast<const __half*>(p) + i));
}
__device__ __forceinline__ void store_f(void* p, int dtype, int64_t i, float v) {
  if (dtype == 0) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else if (dtype == 1) static_cast<float*>(p)[i] = v;
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ float act_of(float g, int act) {
  return act == kActSigmoid ? 1.f / (1.f + expf(-g)) : act == kActTanh ? tanhf(g) : g;
}
// act'(g) from a = act(g)
__device__ __forceinline__ float act_slope(float a, int act) {
  return act == kActSigmoid ? a * (1.f - a) : act == kActTanh ? 1.f - a * a : 1.f;
}

// ---------------------------------------------------------------- rows in registers

// Eight elements of a row per chunk: VEC consecutive ones by 16-byte accesses, else (odd widths,
// strides or addresses) every team-th one, so that a warp's accesses still lie side by side.
__device__ __forceinline__ float elem_f(float v) { return v; }
__device__ __forceinline__ float elem_f(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float elem_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void elem_set(float& d, float v) { d = v; }
__device__ __forceinline__ void elem_set(uint16_t& d, float v) { d = f32_to_bf16(v); }
__device__ __forceinline__ void elem_set(__half& d, float v) { d = __float2half_rn(v); }

template <typename T>
struct __align__(16) Pack8 {
  T v[8];
};

template <bool VEC>
__device__ __forceinline__ int col_of(int chunk, int i, int tid, int team) {
  return VEC ? (chunk * team + tid) * 8 + i : (chunk * 8 + i) * team + tid;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(Pack8<T>& d, const T* row, int chunk, int tid, int team, int cols) {
  if (VEC) {
    const int c = (chunk * team + tid) * 8;
    uint4* w = reinterpret_cast<uint4*>(&d);
    if (c < cols) {
      const uint4* src = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
      for (int i = 0; i < int(sizeof(T)) / 2; ++i) w[i] = __ldg(src + i);
    } else {
#pragma unroll
      for (int i = 0; i < int(sizeof(T)) / 2; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<false>(chunk, i, tid, team);
      d.v[i] = c < cols ? __ldg(row + c) : T(0.f);
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, const float (&v)[8], int chunk, int tid, int team, int cols) {
  if (VEC) {
    const int c = (chunk * team + tid) * 8;
    if (c >= cols) return;
    Pack8<T> p;
#pragma unroll
    for (int i = 0; i < 8; ++i) elem_set(p.v[i], v[i]);
    uint4* dst = reinterpret_cast<uint4*>(row + c);
    const uint4* w = reinterpret_cast<const uint4*>(&p);
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) dst[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<false>(chunk, i, tid, team);
      if (c < cols) elem_set(row[c], v[i]);
    }
  }
}

// Sums over the team, the same order every time; every thread gets them.  One barrier per call:
// three buffers in turn, so that a buffer is written again only behind the barrier after its reads.
struct TeamSum {
  float2* buf;  // [3][32] shared, or unused by a one-warp team
  int turn;
  __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (buf == nullptr) return make_float2(a, b);
    float2* t = buf + turn * 32;
    turn = turn == 2 ? 0 : turn + 1;
    if ((threadIdx.x & 31) == 0) t[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
    for (int w = 0; w < int(blockDim.x >> 5); ++w) {
      s.x += t[w].x;
      s.y += t[w].y;
    }
    return s;
  }
};

// The gate of a row where it is not one of the columns' factors.
template <typename TU, int NCH, bool VEC>
__device__ __forceinline__ void load_gate(Pack8<TU> (&raw)[NCH], float& one, const NormArgs& a, int64_t r, int tid, int team) {
  if (a.gate_mode == kGateRow) one = load_f(a.gate, a.gate_dtype, r);
  if (a.gate_mode == kGateFull)
#pragma unroll
    for (int j = 0; j < NCH; ++j)
      load8<TU, VEC>(raw[j], static_cast<const TU*>(a.gate) + r * a.ld_gate, j, tid, team, a.cols);
}

// Column factors of the team: k = bs act(g) w_post (the gate only where it is the columns'), w = w_pre.
template <int NCH, bool VEC>
__device__ __forceinline__ void load_factors(const NormArgs& a, int64_t group, int tid, int team, float (&k)[NCH][8],
                                             float (&w)[NCH][8]) {
#pragma unroll
  for (int j = 0; j < NCH; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<VEC>(j, i, tid, team);
      const bool in = c < a.cols;
      float f = in ? a.branch_scale : 0.f;
      if (in && a.post_weight != nullptr) f *= __ldg(a.post_weight + c);
      if (in && a.gate_mode == kGateChannel)
        f *= act_of(load_f(a.gate, a.gate_dtype, group * a.cols + c), a.gate_act);
      k[j][i] = f;
      w[j][i] = in && a.pre_weight != nullptr ? __ldg(a.pre_weight + c) : 0.f;
    }
}

struct TeamPlan {
  int64_t parts;       // teams of a group of rows
  int64_t group_rows;
  int64_t teams;       // in all
};

template <typename TX, typename TU, int NCH, bool VEC>
__global__ void __launch_bounds__(NCH == 1 ? 256 : 512, NCH == 1 ? 3 : 1)
    residual_norm_team_kernel(const NormArgs a, const TeamPlan plan) {
  __shared__ float2 buf[3 * 32];
  const bool warp_team = a.cols <= 256;
  const int team = warp_team ? 32 : int(blockDim.x);
  const int tid = warp_team ? int(threadIdx.x & 31) : int(threadIdx.x);
  const int64_t id = warp_team ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : int64_t(blockIdx.x);
  if (id >= plan.teams) return;  // a whole team: no barrier is left behind
  TeamSum sum{warp_team ? nullptr : buf, 0};
  const int64_t group = id / plan.parts;
  const int64_t end = (group + 1) * plan.group_rows;
  float k[NCH][8], w[NCH][8];
  load_factors<NCH, VEC>(a, group, tid, team, k, w);
  const float inv = 1.f / float(a.cols);
  Pack8<TX> x[NCH];
  Pack8<TU> u[NCH], g[NCH];
  float g1 = 1.f;
  auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      load8<TX, VEC>(x[j], static_cast<const TX*>(a.x) + r * a.ld_x, j, tid, team, a.cols);
      if (a.branch != nullptr) load8<TU, VEC>(u[j], static_cast<const TU*>(a.branch) + r * a.ld_branch, j, tid, team, a.cols);
    }
    load_gate<TU, NCH, VEC>(g, g1, a, r, tid, team);
  };
  int64_t r = group * plan.group_rows + id % plan.parts;
  if (r < end) load(r);
  for (; r < end; r += plan.parts) {
    float y[NCH][8];
    float ru = 1.f;
    if (a.branch != nullptr) {
      float f[NCH][8];
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f[j][i] = k[j][i] * elem_f(u[j].v[i]);
          y[j][i] = a.residual_scale * elem_f(x[j].v[i]);
        }
      if (a.post_weight != nullptr) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) s += elem_f(u[j].v[i]) * elem_f(u[j].v[i]);
        ru = rsqrtf(sum(s, 0.f).x * inv + a.eps);
      }
      if (a.gate_mode == kGateFull) {
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[j][i] *= act_of(elem_f(g[j].v[i]), a.gate_act);
      }
      const float scale = a.gate_mode == kGateRow ? ru * act_of(g1, a.gate_act) : ru;
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[j][i] += scale * f[j][i];
    } else {
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[j][i] = elem_f(x[j].v[i]);
    }
    const int64_t next = r + plan.parts;
    if (next < end) load(next);
    if (a.stream_out != nullptr)
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        store8<TX, VEC>(static_cast<TX*>(a.stream_out) + r * a.cols, y[j], j, tid, team, a.cols);
    float ry = 1.f;
    if (a.pre_weight != nullptr) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += y[j][i] * y[j][i];
      ry = rsqrtf(sum(s, 0.f).x * inv + a.eps);
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[j][i] *= ry * w[j][i];
        store8<TU, VEC>(static_cast<TU*>(a.norm_out) + r * a.cols, y[j], j, tid, team, a.cols);
      }
    }
    if (a.stats != nullptr && tid == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(ru, ry);
  }
}

template <typename TX, typename TU, int NCH, bool VEC>
__global__ void __launch_bounds__(NCH == 1 ? 256 : 512, NCH == 1 ? 2 : 1)
    residual_norm_team_bwd_kernel(const NormArgs a, const TeamPlan plan, float* partial) {
  __shared__ float2 buf[3 * 32];
  const bool warp_team = a.cols <= 256;
  const int team = warp_team ? 32 : int(blockDim.x);
  const int tid = warp_team ? int(threadIdx.x & 31) : int(threadIdx.x);
  const int64_t id = warp_team ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : int64_t(blockIdx.x);
  if (id >= plan.teams) return;
  TeamSum sum{warp_team ? nullptr : buf, 0};
  const int64_t group = id / plan.parts;
  const int64_t end = (group + 1) * plan.group_rows;
  float k[NCH][8], w[NCH][8], acc_pre[NCH][8], acc_s[NCH][8];
  load_factors<NCH, VEC>(a, group, tid, team, k, w);
#pragma unroll
  for (int j = 0; j < NCH; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc_pre[j][i] = acc_s[j][i] = 0.f;
  const float inv = 1.f / float(a.cols);
  const bool normed = a.d_normed != nullptr, post = a.post_weight != nullptr, branch = a.branch != nullptr;
  const float rs = branch ? a.residual_scale : 1.f;
  Pack8<TX> x[NCH], dy[NCH];
  Pack8<TU> u[NCH], dh[NCH], g[NCH];
  float g1 = 0.f;
  float2 st = make_float2(1.f, 1.f);
  auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      load8<TX, VEC>(x[j], static_cast<const TX*>(a.x) + r * a.ld_x, j, tid, team, a.cols);
      if (branch) load8<TU, VEC>(u[j], static_cast<const TU*>(a.branch) + r * a.ld_branch, j, tid, team, a.cols);
      if (a.d_stream != nullptr)
        load8<TX, VEC>(dy[j], static_cast<const TX*>(a.d_stream) + r * a.ld_d_stream, j, tid, team, a.cols);
      if (normed) load8<TU, VEC>(dh[j], static_cast<const TU*>(a.d_normed) + r * a.ld_d_normed, j, tid, team, a.cols);
    }
    load_gate<TU, NCH, VEC>(g, g1, a, r, tid, team);
    if (a.stats != nullptr) st = *reinterpret_cast<const float2*>(a.stats + 2 * r);
  };
  int64_t r = group * plan.group_rows + id % plan.parts;
  if (r < end) load(r);
  for (; r < end; r += plan.parts) {
    const float ru = st.x, ry = st.y;
    const float a1 = a.gate_mode == kGateRow ? act_of(g1, a.gate_act) : 1.f;
    // z: dz; uh: u r_u; f: the element's k, its gate applied
    float z[NCH][8], uh[NCH][8], f[NCH][8];
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        z[j][i] = a.d_stream != nullptr ? elem_f(dy[j].v[i]) : 0.f;
        uh[j][i] = branch ? elem_f(u[j].v[i]) * ru : 0.f;
        f[j][i] = a.gate_mode == kGateFull ? k[j][i] * act_of(elem_f(g[j].v[i]), a.gate_act) : k[j][i] * a1;
      }
    if (normed) {
      float yh[NCH][8];
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = elem_f(dh[j].v[i]);
          yh[j][i] = (rs * elem_f(x[j].v[i]) + f[j][i] * uh[j][i]) * ry;
          acc_pre[j][i] += d * yh[j][i];
          dot += d * w[j][i] * yh[j][i];
        }
      const float mean = sum(dot, 0.f).x * inv;
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) z[j][i] += ry * (elem_f(dh[j].v[i]) * w[j][i] - yh[j][i] * mean);
    }
    float dot_u = 0.f, dot_g = 0.f;
    float slope[NCH][8];  // of the full gate: bs act'(g) w_post uh dz
    const float s1 = act_slope(a1, a.gate_act);
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float zu = z[j][i] * uh[j][i];
        dot_u += f[j][i] * zu;
        dot_g += k[j][i] * zu;
        if (a.gate_mode == kGateFull) {
          const float ga = act_of(elem_f(g[j].v[i]), a.gate_act);
          slope[j][i] = act_slope(ga, a.gate_act) * (k[j][i] * zu);
          acc_s[j][i] += ga * zu;
        } else {
          acc_s[j][i] += a1 * zu;
        }
      }
    const float row_slope = s1;
    const int64_t here = r;
    const int64_t next = r + plan.parts;
    if (next < end) load(next);
    if (a.d_x != nullptr)
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = rs * z[j][i];
        store8<TX, VEC>(static_cast<TX*>(a.d_x) + here * a.cols, o, j, tid, team, a.cols);
      }
    if (!branch) continue;
    if (a.gate_mode == kGateFull && a.d_gate != nullptr)
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        store8<TU, VEC>(static_cast<TU*>(a.d_gate) + here * a.cols, slope[j], j, tid, team, a.cols);
    float mean_u = 0.f;
    if (post || a.gate_mode == kGateRow) {
      const float2 s = sum(dot_u, dot_g);
      if (post) mean_u = s.x * inv;
      if (a.gate_mode == kGateRow && tid == 0 && a.d_gate != nullptr) static_cast<float*>(a.d_gate)[here] = row_slope * s.y;
    }
    if (a.d_branch != nullptr)
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = ru * (f[j][i] * z[j][i] - uh[j][i] * mean_u);
        store8<TU, VEC>(static_cast<TU*>(a.d_branch) + here * a.cols, o, j, tid, team, a.cols);
      }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < NCH; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<VEC>(j, i, tid, team);
      if (c >= a.cols) continue;
      partial[id * a.cols + c] = acc_pre[j][i];
      partial[(plan.teams + id) * a.cols + c] = acc_s[j][i];
    }
}

// ---------------------------------------------------------------- any width and types: rows from memory

// Sum over the CTA, the same order every time; every thread gets it.
__device__ __forceinline__ float cta_sum(float v, float* tmp) { return block_sum(v, tmp); }

struct Row {
  const NormArgs& a;
  int64_t r;
  float ru, ry;
  __device__ float x(int c) const { return load_f(a.x, a.x_dtype, r * a.ld_x + c); }
  __device__ float u(int c) const { return load_f(a.branch, a.branch_dtype, r * a.ld_branch + c); }
  __device__ float gate(int c) const {
    if (a.gate_mode == kGateNone) return 1.f;
    const int64_t i = a.gate_mode == kGateChannel ? r / a.gate_rows * a.cols + c
                      : a.gate_mode == kGateRow   ? r
                                                  : r * a.ld_gate + c;
    return act_of(load_f(a.gate, a.gate_dtype, i), a.gate_act);
  }
  __device__ float post(int c) const { return a.post_weight ? __ldg(a.post_weight + c) : 1.f; }
  __device__ float y(int c) const {
    if (a.branch == nullptr) return x(c);
    return a.residual_scale * x(c) + a.branch_scale * (gate(c) * (u(c) * ru * post(c)));
  }
};

__global__ void __launch_bounds__(kNormThreads) residual_norm_kernel(const NormArgs a) {
  __shared__ float tmp[32];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    Row row{a, r, 1.f, 1.f};
    if (a.branch != nullptr && a.post_weight != nullptr) {
      float sum = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += kNormThreads) sum += row.u(c) * row.u(c);
      row.ru = rsqrtf(cta_sum(sum, tmp) / float(a.cols) + a.eps);
    }
    float sum = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
      const float y = row.y(c);
      sum += y * y;
      if (a.stream_out != nullptr) store_f(a.stream_out, a.x_dtype, r * a.cols + c, y);
    }
    if (a.pre_weight != nullptr) {
      row.ry = rsqrtf(cta_sum(sum, tmp) / float(a.cols) + a.eps);
      for (int c = threadIdx.x; c < a.cols; c += kNormThreads)
        store_f(a.norm_out, a.norm_dtype, r * a.cols + c, row.y(c) * row.ry * __ldg(a.pre_weight + c));
    }
    if (a.stats != nullptr && threadIdx.x == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(row.ru, row.ry);
  }
}

// One CTA per part of a gate group's rows; its column sums stay in shared memory (each column
// belongs to one thread) and leave as rows of `partial`.
__global__ void __launch_bounds__(kNormThreads) residual_norm_bwd_kernel(const NormArgs a, const TeamPlan plan,
                                                                         float* partial) {
  extern __shared__ float acc[];  // [2][cols]: pre, S
  __shared__ float tmp[32];
  const int64_t group = blockIdx.x / plan.parts, part = blockIdx.x % plan.parts;
  const int64_t end = (group + 1) * plan.group_rows;
  for (int c = threadIdx.x; c < 2 * a.cols; c += kNormThreads) acc[c] = 0.f;
  __syncthreads();
  const float inv = 1.f / float(a.cols);
  const bool normed = a.d_normed != nullptr;
  for (int64_t r = group * plan.group_rows + part; r < end; r += plan.parts) {
    Row row{a, r, 1.f, 1.f};
    if (a.stats != nullptr) {
      row.ru = a.stats[2 * r];
      row.ry = a.stats[2 * r + 1];
    }
    float mean_t = 0.f;
    if (normed) {
      float dot = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += kNormThreads)
        dot += load_f(a.d_normed, a.norm_dtype, r * a.ld_d_normed + c) * __ldg(a.pre_weight + c) * row.y(c);
      mean_t = cta_sum(dot, tmp) * inv * row.ry;
    }
    auto dz = [&](int c) {
      float v = a.d_stream != nullptr ? load_f(a.d_stream, a.x_dtype, r * a.ld_d_stream + c) : 0.f;
      if (normed) {
        const float t = load_f(a.d_normed, a.norm_dtype, r * a.ld_d_normed + c) * __ldg(a.pre_weight + c);
        v += row.ry * (t - row.y(c) * row.ry * mean_t);
      }
      return v;
    };
    float dot_u = 0.f, dot_g = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
      const float z = dz(c);
      if (a.d_x != nullptr) store_f(a.d_x, a.x_dtype, r * a.cols + c, (a.branch ? a.residual_scale : 1.f) * z);
      if (normed) acc[c] += load_f(a.d_normed, a.norm_dtype, r * a.ld_d_normed + c) * row.y(c) * row.ry;
      if (a.branch == nullptr) continue;
      const float g = row.gate(c), zu = z * row.u(c) * row.ru, kzu = a.branch_scale * row.post(c) * zu;
      acc[a.cols + c] += a.gate_mode == kGateChannel ? zu : g * zu;
      dot_u += g * kzu;
      dot_g += kzu * act_slope(g, a.gate_act);
      if (a.gate_mode == kGateFull && a.d_gate != nullptr)
        store_f(a.d_gate, a.gate_dtype, r * a.cols + c, kzu * act_slope(g, a.gate_act));
    }
    if (a.branch == nullptr) continue;
    if (a.gate_mode == kGateRow) {
      const float sum = cta_sum(dot_g, tmp);
      if (threadIdx.x == 0 && a.d_gate != nullptr) static_cast<float*>(a.d_gate)[r] = sum;
    }
    const float mean_u = a.post_weight != nullptr ? cta_sum(dot_u, tmp) * inv : 0.f;
    if (a.d_branch != nullptr)
      for (int c = threadIdx.x; c < a.cols; c += kNormThreads)
        store_f(a.d_branch, a.branch_dtype, r * a.cols + c,
                row.ru * (a.branch_scale * dz(c) * row.gate(c) * row.post(c) - row.u(c) * row.ru * mean_u));
  }
  if (partial == nullptr) return;
  __syncthreads();
  for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
    partial[int64_t(blockIdx.x) * a.cols + c] = acc[c];
    partial[(plan.teams + blockIdx.x) * a.cols + c] = acc[a.cols + c];
  }
}

// ---------------------------------------------------------------- column sums

constexpr int kSumRows = 32;

// Adds `count` rows of `src`, the same order every time (32 interleaved sums, then those).
__device__ __forceinline__ float column_sum(const float* src, int64_t count, int cols, int c, float (*tmp)[33]) {
  float s = 0.f;
  if (c < cols)
    for (int64_t b = threadIdx.y; b < count; b += kSumRows) s += src[b * cols + c];
  tmp[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  for (int o = kSumRows / 2; o > 0; o >>= 1) {
    if (int(threadIdx.y) < o) tmp[threadIdx.y][threadIdx.x] += tmp[threadIdx.y + o][threadIdx.x];
    __syncthreads();
  }
  return tmp[0][threadIdx.x];
}

// blockIdx.y < groups: S of that group -> d_gate and, for one group, d_post (for more, its part
// of it into `parts_post`); blockIdx.y == groups: d_pre.
__global__ void __launch_bounds__(32 * kSumRows) norm_columns_kernel(const NormArgs a, const TeamPlan plan,
                                                                     const float* partial, int groups,
                                                                     float* parts_post) {
  __shared__ float tmp[kSumRows][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int group = blockIdx.y;
  if (group == groups) {
    if (a.d_pre == nullptr) return;
    const float s = column_sum(partial, plan.teams, a.cols, c, tmp);
    if (threadIdx.y == 0 && c < a.cols) a.d_pre[c] = s;
    return;
  }
  const float s = column_sum(partial + (plan.teams + group * plan.parts) * a.cols, plan.parts, a.cols, c, tmp);
  if (threadIdx.y != 0 || c >= a.cols) return;
  float gate = 1.f;
  if (a.gate_mode == kGateChannel) {
    gate = act_of(load_f(a.gate, a.gate_dtype, int64_t(group) * a.cols + c), a.gate_act);
    const float post = a.post_weight != nullptr ? __ldg(a.post_weight + c) : 1.f;
    if (a.d_gate != nullptr)
      static_cast<float*>(a.d_gate)[int64_t(group) * a.cols + c] = a.branch_scale * act_slope(gate, a.gate_act) * post * s;
  }
  if (a.d_post == nullptr) return;
  const float d = a.branch_scale * gate * s;
  if (groups == 1) a.d_post[c] = d;
  else parts_post[int64_t(group) * a.cols + c] = d;
}

__global__ void __launch_bounds__(32 * kSumRows) norm_groups_kernel(const float* parts_post, int groups, int cols,
                                                                    float* d_post) {
  __shared__ float tmp[kSumRows][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float s = column_sum(parts_post, groups, cols, c, tmp);
  if (threadIdx.y == 0 && c < cols) d_post[c] = s;
}

// ---------------------------------------------------------------- host

bool dtype_ok(int t) { return t >= 0 && t <= 2; }

int check_norm(const NormArgs* a, bool backward) {
  if (!a || a->rows < 0 || a->cols <= 0 || !dtype_ok(a->x_dtype) || !dtype_ok(a->norm_dtype)) return MCL4MOE_ERR_INVALID;
  const bool some = a->rows > 0;
  if ((some && !a->x) || a->ld_x < a->cols) return MCL4MOE_ERR_INVALID;
  if (a->branch) {
    if (!dtype_ok(a->branch_dtype) || a->ld_branch < a->cols) return MCL4MOE_ERR_INVALID;
  } else if (a->post_weight || a->gate_mode != kGateNone) {
    return MCL4MOE_ERR_INVALID;
  }
  if (a->gate_mode < 0 || a->gate_mode > 3 || a->gate_act < 0 || a->gate_act > 2) return MCL4MOE_ERR_INVALID;
  if (a->gate_mode != kGateNone) {
    if ((some && !a->gate) || !dtype_ok(a->gate_dtype)) return MCL4MOE_ERR_INVALID;
    if (a->gate_mode == kGateChannel && (a->gate_rows <= 0 || a->rows % a->gate_rows != 0)) return MCL4MOE_ERR_INVALID;
    if (a->gate_mode == kGateFull && a->ld_gate < a->cols) return MCL4MOE_ERR_INVALID;
  }
  if ((reinterpret_cast<uintptr_t>(a->stats) & 7) != 0) return MCL4MOE_ERR_INVALID;
  if (!backward && some &&
      ((a->pre_weight && !a->norm_out) || (a->branch && !a->stream_out) || (!a->branch && !a->pre_weight)))
    return MCL4MOE_ERR_INVALID;
  if (backward && some &&
      ((a->d_stream && a->ld_d_stream < a->cols) || (a->d_normed && (!a->pre_weight || a->ld_d_normed < a->cols)) ||
       (!a->stats && (a->post_weight || a->d_normed))))
    return MCL4MOE_ERR_INVALID;
  if (a->cols > kMaxNormCols) return MCL4MOE_ERR_UNSUPPORTED;
  return MCL4MOE_OK;
}

// Threads of a team's CTA and the teams of a call: as many as are resident at once (`per_sm` threads
// an SM: what the registers of the kernels leave room for), shared out over the gate's groups.
struct NormShape {
  bool wide;         // 16 columns a thread instead of 8
  int threads;       // of a CTA
  int rows_per_cta;  // teams of a CTA
  TeamPlan plan;
  int64_t groups;
};

NormShape norm_shape(int64_t rows, int cols, int gate_mode, int64_t gate_rows, bool backward) {
  NormShape s{};
  s.wide = cols > 2048;
  const int per = s.wide ? 16 : 8;
  const int need = (cols + per - 1) / per;
  s.threads = cols <= 256 ? 128 : (need + 31) / 32 * 32;
  s.rows_per_cta = cols <= 256 ? 4 : 1;
  if (cols > kTeamCols) s.threads = kNormThreads;
  const int64_t per_sm = cols > kTeamCols ? 512 : s.wide ? 512 : backward ? 512 : 768;
  const int64_t ctas = per_sm / s.threads > 0 ? per_sm / s.threads : 1;
  const int64_t want = ctas * num_sms() * s.rows_per_cta;
  s.groups = gate_mode == kGateChannel ? rows / gate_rows : 1;
  s.plan.group_rows = gate_mode == kGateChannel ? gate_rows : rows;
  int64_t parts = want / s.groups;
  if (parts > s.plan.group_rows) parts = s.plan.group_rows;
  s.plan.parts = parts < 1 ? 1 : parts;
  s.plan.teams = s.plan.parts * s.groups;
  return s;
}

bool aligned(const void* p, int64_t ld, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % (dtype == 1 ? 4 : 8) == 0;
}

// 16-byte accesses are possible (null pointers pass).
bool norm_vectors(const NormArgs& a) {
  if (a.cols % 8 != 0) return false;
  const bool full = a.gate_mode == kGateFull;
  return aligned(a.x, a.ld_x, a.x_dtype) && aligned(a.branch, a.branch ? a.ld_branch : 0, a.branch_dtype) &&
         aligned(full ? a.gate : nullptr, full ? a.ld_gate : 0, a.gate_dtype) &&
         aligned(a.d_stream, a.d_stream ? a.ld_d_stream : 0, a.x_dtype) &&
         aligned(a.d_normed, a.d_normed ? a.ld_d_normed : 0, a.norm_dtype) && aligned(a.stream_out, 0, 0) &&
         aligned(a.norm_out, 0, 0) && aligned(a.d_x, 0, 0) && aligned(a.d_branch, 0, 0) &&
         aligned(full ? a.d_gate : nullptr, 0, 0);
}

// The team kernels take the stream's type and one other: of the branch, the norm's output and an
// element-wise gate.  Other mixes and wider rows go through the generic kernels.
bool norm_in_registers(const NormArgs& a) {
  if (a.cols > kTeamCols || (a.branch && a.branch_dtype != a.norm_dtype)) return false;
  if (a.gate_mode == kGateFull && a.gate_dtype != a.norm_dtype) return false;
  return a.x_dtype == a.norm_dtype || a.x_dtype == 1;
}

template <typename TX, typename TU, int NCH, bool VEC>
void launch_team(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  const unsigned grid = unsigned((s.plan.teams + s.rows_per_cta - 1) / s.rows_per_cta);
  if (backward) residual_norm_team_bwd_kernel<TX, TU, NCH, VEC><<<grid, s.threads, 0, stream>>>(a, s.plan, partial);
  else residual_norm_team_kernel<TX, TU, NCH, VEC><<<grid, s.threads, 0, stream>>>(a, s.plan);
}
template <typename TX, typename TU>
void launch_team(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  const bool vec = norm_vectors(a);
  if (s.wide) {
    if (vec) launch_team<TX, TU, 2, true>(a, s, backward, partial, stream);
    else launch_team<TX, TU, 2, false>(a, s, backward, partial, stream);
  } else {
    if (vec) launch_team<TX, TU, 1, true>(a, s, backward, partial, stream);
    else launch_team<TX, TU, 1, false>(a, s, backward, partial, stream);
  }
}
void launch_teams(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  if (a.x_dtype == 1) {
    if (a.norm_dtype == 0) launch_team<float, uint16_t>(a, s, backward, partial, stream);
    else if (a.norm_dtype == 1) launch_team<float, float>(a, s, backward, partial, stream);
    else launch_team<float, __half>(a, s, backward, partial, stream);
  } else if (a.x_dtype == 0) {
    launch_team<uint16_t, uint16_t>(a, s, backward, partial, stream);
  } else {
    launch_team<__half, __half>(a, s, backward, partial, stream);
  }
}

}  // namespace
}  // namespace mcl4

using namespace mcl4;

extern "C" {

int mcl4moe_residual_norm(const mcl4moe_norm_args* a, mcl4moe_stream_t stream) {
  const int st = check_norm(a, false);
  if (st != MCL4MOE_OK) return st;
  if (a->rows == 0) return MCL4MOE_OK;
  const NormShape s = norm_shape(a->rows, a->cols, a->gate_mode, a->gate_rows, false);
  if (s.plan.teams > (int64_t(1) << 30)) return MCL4MOE_ERR_UNSUPPORTED;
  if (norm_in_registers(*a)) {
    launch_teams(*a, s, false, nullptr, stream);
  } else {
    const int64_t grid = a->rows < int64_t(64) * num_sms() ? a->rows : int64_t(64) * num_sms();
    residual_norm_kernel<<<unsigned(grid), kNormThreads, 0, stream>>>(*a);
  }
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

size_t mcl4moe_residual_norm_workspace_size(int64_t rows, int cols, int gate_mode, int64_t gate_rows) {
  if (rows <= 0 || cols <= 0 || cols > kMaxNormCols || (gate_mode == kGateChannel && gate_rows <= 0)) return 0;
  const NormShape s = norm_shape(rows, cols, gate_mode, gate_rows, true);
  return size_t(2 * s.plan.teams + (s.groups > 1 ? s.groups : 0)) * size_t(cols) * sizeof(float);
}

int mcl4moe_residual_norm_backward(const mcl4moe_norm_args* a, void* workspace, size_t workspace_bytes,
                                   mcl4moe_stream_t stream) {
  const int st = check_norm(a, true);
  if (st != MCL4MOE_OK) return st;
  const bool sums = a->d_pre || a->d_post || (a->gate_mode == kGateChannel && a->d_gate);
  if (a->rows == 0) {
    if ((a->d_pre && cudaMemsetAsync(a->d_pre, 0, sizeof(float) * a->cols, stream) != cudaSuccess) ||
        (a->d_post && cudaMemsetAsync(a->d_post, 0, sizeof(float) * a->cols, stream) != cudaSuccess))
      return MCL4MOE_ERR_CUDA;
    return MCL4MOE_OK;
  }
  const NormShape s = norm_shape(a->rows, a->cols, a->gate_mode, a->gate_rows, true);
  if (s.plan.teams > (int64_t(1) << 30) || s.groups > 65533) return MCL4MOE_ERR_UNSUPPORTED;
  if (sums && (!workspace || workspace_bytes < mcl4moe_residual_norm_workspace_size(a->rows, a->cols, a->gate_mode,
                                                                                    a->gate_rows)))
    return MCL4MOE_ERR_WORKSPACE;
  float* partial = sums ? static_cast<float*>(workspace) : nullptr;
  if (norm_in_registers(*a)) {
    launch_teams(*a, s, true, partial, stream);
  } else {
    static std::atomic<uint64_t> raised{0};
    if (!raise_smem_limit(residual_norm_bwd_kernel, 2 * kMaxNormCols * int(sizeof(float)), raised)) return MCL4MOE_ERR_CUDA;
    residual_norm_bwd_kernel<<<unsigned(s.plan.teams / s.plan.parts * s.plan.parts), kNormThreads,
                               2 * a->cols * sizeof(float), stream>>>(*a, s.plan, partial);
  }
  if (sums) {
    const int groups = int(s.groups);
    float* parts_post = partial + 2 * s.plan.teams * a->cols;
    const dim3 block(32, kSumRows);
    norm_columns_kernel<<<dim3((a->cols + 31) / 32, unsigned(groups + 1)), block, 0, stream>>>(*a, s.plan, partial,
                                                                                              groups, parts_post);
    if (groups > 1 && a->d_post)
      norm_groups_kernel<<<(a->cols + 31) / 32, block, 0, stream>>>(parts_post, groups, a->cols, a->d_post);
  }
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

}  // extern "C"
