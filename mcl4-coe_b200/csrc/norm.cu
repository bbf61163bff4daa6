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
// CTA, 8 or 16 columns a thread) between the reductions, and the next rows are under way to shared
// memory meanwhile.  Teams are persistent, which keeps the columns' factors in registers and, in the
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

// Eight float32 as four pairs: one instruction for two products or sums.
struct V8 {
  uint64_t p[4];
  __device__ __forceinline__ float get(int i) const {
    float a, b;
    f2unpack(p[i >> 1], a, b);
    return i & 1 ? b : a;
  }
  __device__ __forceinline__ void fill(float v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = f2pack(v, v);
  }
};
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ V8 mul(const V8& a, const V8& b) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fmul2(a.p[i], b.p[i]);
  return r;
}
__device__ __forceinline__ V8 mul(const V8& a, float s) {
  V8 r;
  const uint64_t ss = f2pack(s, s);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fmul2(a.p[i], ss);
  return r;
}
__device__ __forceinline__ V8 fma(const V8& a, const V8& b, const V8& c) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = ffma2(a.p[i], b.p[i], c.p[i]);
  return r;
}
__device__ __forceinline__ V8 fma(const V8& a, float s, const V8& c) {
  V8 r;
  const uint64_t ss = f2pack(s, s);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = ffma2(a.p[i], ss, c.p[i]);
  return r;
}
__device__ __forceinline__ float total(const V8& a) {
  float x, y;
  f2unpack(fadd2(fadd2(a.p[0], a.p[1]), fadd2(a.p[2], a.p[3])), x, y);
  return x + y;
}

template <bool VEC>
__device__ __forceinline__ int col_of(int chunk, int i, int tid, int team) {
  return VEC ? (chunk * team + tid) * 8 + i : (chunk * 8 + i) * team + tid;
}

template <typename T>
__device__ __forceinline__ V8 unpack8(const Pack8<T>& d) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = f2pack(elem_f(d.v[2 * i]), elem_f(d.v[2 * i + 1]));
  return r;
}

template <typename T>
__device__ __forceinline__ V8 load8(const T* row, int chunk, int tid, int team, int cols) {
  Pack8<T> d;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = col_of<false>(chunk, i, tid, team);
    d.v[i] = c < cols ? __ldg(row + c) : T(0.f);
  }
  return unpack8(d);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, const V8& v, int chunk, int tid, int team, int cols) {
  if (VEC) {
    const int c = (chunk * team + tid) * 8;
    if (c >= cols) return;
    Pack8<T> p;
#pragma unroll
    for (int i = 0; i < 8; ++i) elem_set(p.v[i], v.get(i));
    uint4* dst = reinterpret_cast<uint4*>(row + c);
    const uint4* w = reinterpret_cast<const uint4*>(&p);
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) dst[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<false>(chunk, i, tid, team);
      if (c < cols) elem_set(row[c], v.get(i));
    }
  }
}

// The rows ahead of a thread, in shared memory: it copies its own elements there (cp.async, 16
// bytes each) `depth` rows ahead and reads them back itself, so that no barrier stands between and
// the loads in flight need no registers.  Slots of a row: up to five operands of NCH chunks.
// Without VEC the elements come straight from memory when they are asked for.
template <int NCH, bool VEC>
struct Ahead {
  char* mine;       // this thread's first 16 bytes
  uint32_t stride;  // bytes between the 16-byte pieces of a thread
  uint32_t stage;   // bytes of a row
  int depth, slot;
  template <typename T>
  __device__ __forceinline__ void fetch(const T* row, uint32_t at, int s, int tid, int team, int cols) const {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c = (j * team + tid) * 8;
        if (c >= cols) continue;
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
          const uint32_t dst = uint32_t(__cvta_generic_to_shared(mine + s * stage + (at + j * (sizeof(T) / 2) + i) * stride));
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(row + c + i * (16 / sizeof(T)))
                       : "memory");
        }
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ V8 take(const T* row, uint32_t at, int j, int tid, int team, int cols) const {
    if constexpr (!VEC) {
      return load8(row, j, tid, team, cols);
    } else {
      Pack8<T> d;
      uint4* w = reinterpret_cast<uint4*>(&d);
      const bool in = (j * team + tid) * 8 < cols;
#pragma unroll
      for (int i = 0; i < int(sizeof(T)) / 2; ++i)
        w[i] = in ? *reinterpret_cast<const uint4*>(mine + slot * stage + (at + j * (sizeof(T) / 2) + i) * stride)
                  : make_uint4(0u, 0u, 0u, 0u);
      return unpack8(d);
    }
  }
  __device__ __forceinline__ void commit() const {
    if (VEC) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The oldest of `depth` committed rows is there.
  __device__ __forceinline__ void wait() const {
    if (!VEC) return;
    if (depth >= 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  __device__ __forceinline__ void next() { slot = slot + 1 == depth ? 0 : slot + 1; }
};

// Sums over the team, the same order every time; every thread gets them.  One barrier per call:
// three buffers in turn, so that a buffer is written again only behind the barrier after its reads.
struct TeamSum {
  float* buf;  // [3][2][32] shared, or null for a one-warp team
  int warps, turn;
  __device__ __forceinline__ float across(const float* t) const {
    float s = 0.f;
#pragma unroll 4
    for (int w = 0; w < warps; ++w) s += t[w];
    return s;
  }
  __device__ __forceinline__ float one(float a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (buf == nullptr) return a;
    float* t = buf + turn * 64;
    turn = turn == 2 ? 0 : turn + 1;
    if ((threadIdx.x & 31) == 0) t[threadIdx.x >> 5] = a;
    __syncthreads();
    return across(t);
  }
  __device__ __forceinline__ float2 two(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (buf == nullptr) return make_float2(a, b);
    float* t = buf + turn * 64;
    turn = turn == 2 ? 0 : turn + 1;
    if ((threadIdx.x & 31) == 0) {
      t[threadIdx.x >> 5] = a;
      t[32 + (threadIdx.x >> 5)] = b;
    }
    __syncthreads();
    return make_float2(across(t), across(t + 32));
  }
};

// Column factors of the team: k = bs act(g) w_post (the gate only where it is the columns'), w = w_pre.
template <int NCH, bool VEC>
__device__ __forceinline__ void load_factors(const NormArgs& a, int64_t group, int tid, int team, V8 (&k)[NCH],
                                             V8 (&w)[NCH]) {
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    float kf[8], wf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<VEC>(j, i, tid, team);
      const bool in = c < a.cols;
      float f = in ? a.branch_scale : 0.f;
      if (in && a.post_weight != nullptr) f *= __ldg(a.post_weight + c);
      if (in && a.gate_mode == kGateChannel)
        f *= act_of(load_f(a.gate, a.gate_dtype, group * a.cols + c), a.gate_act);
      kf[i] = f;
      wf[i] = in && a.pre_weight != nullptr ? __ldg(a.pre_weight + c) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[j].p[i] = f2pack(kf[2 * i], kf[2 * i + 1]);
      w[j].p[i] = f2pack(wf[2 * i], wf[2 * i + 1]);
    }
  }
}

struct TeamPlan {
  int64_t parts;       // teams of a group of rows
  int64_t group_rows;
  int64_t teams;       // in all
  int depth;           // rows ahead in shared memory
};

// 16-byte pieces of a thread's row, by operand.
template <typename TX, typename TU, int NCH>
struct Slots {
  static constexpr uint32_t x = 0, px = NCH * sizeof(TX) / 2, pu = NCH * sizeof(TU) / 2;
  static constexpr uint32_t u = px, gate = px + pu, dy = px + 2 * pu, dh = 2 * px + 2 * pu;
  static constexpr uint32_t forward = px + 2 * pu, backward = 2 * px + 3 * pu;
};

// What a team works on: its place in the CTA, its rows and the rows ahead.
template <int NCH, bool VEC>
struct Team {
  int team, tid;
  int64_t id, group, end;
  TeamSum sum;
  Ahead<NCH, VEC> ahead;
  __device__ __forceinline__ Team(const NormArgs& a, const TeamPlan& plan, char* smem, float* buf, uint32_t pieces) {
    const bool warp_team = a.cols <= 256;
    team = warp_team ? 32 : int(blockDim.x);
    tid = warp_team ? int(threadIdx.x & 31) : int(threadIdx.x);
    id = warp_team ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : int64_t(blockIdx.x);
    group = id / plan.parts;
    end = (group + 1) * plan.group_rows;
    sum = TeamSum{warp_team ? nullptr : buf, int(blockDim.x >> 5), 0};
    ahead = Ahead<NCH, VEC>{smem + threadIdx.x * 16, blockDim.x * 16, blockDim.x * 16 * pieces, plan.depth, 0};
  }
};

template <typename TX, typename TU, int NCH, bool VEC, bool FULL>
__global__ void __launch_bounds__(NCH == 1 ? 256 : 512, NCH == 1 ? 3 : 1)
    residual_norm_team_kernel(const NormArgs a, const TeamPlan plan) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float buf[3 * 64];
  using S = Slots<TX, TU, NCH>;
  Team<NCH, VEC> t(a, plan, smem, buf, FULL ? S::forward : S::gate);
  if (t.id >= plan.teams) return;  // a whole team: no barrier is left behind
  const int tid = t.tid, team = t.team, cols = a.cols;
  V8 k[NCH], w[NCH];
  load_factors<NCH, VEC>(a, t.group, tid, team, k, w);
  const float inv = 1.f / float(cols);
  const bool branch = a.branch != nullptr;
  const TX* px = static_cast<const TX*>(a.x);
  const TU* pu = static_cast<const TU*>(a.branch);
  const TU* pg = static_cast<const TU*>(a.gate);
  auto fetch = [&](int64_t r, int s) {
    if (r < t.end) {
      t.ahead.fetch(px + r * a.ld_x, S::x, s, tid, team, cols);
      if (branch) t.ahead.fetch(pu + r * a.ld_branch, S::u, s, tid, team, cols);
      if (FULL) t.ahead.fetch(pg + r * a.ld_gate, S::gate, s, tid, team, cols);
    }
    t.ahead.commit();
  };
  int64_t r = t.group * plan.group_rows + t.id % plan.parts;
  for (int s = 0; s < plan.depth; ++s) fetch(r + s * plan.parts, s);
  for (; r < t.end; r += plan.parts) {
    t.ahead.wait();
    V8 y[NCH], f[NCH];
    float ru = 1.f, s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      y[j] = t.ahead.take(px + r * a.ld_x, S::x, j, tid, team, cols);
      if (!branch) continue;
      const V8 u = t.ahead.take(pu + r * a.ld_branch, S::u, j, tid, team, cols);
      f[j] = mul(u, k[j]);
      if (FULL) {
        const V8 g = t.ahead.take(pg + r * a.ld_gate, S::gate, j, tid, team, cols);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[j].p[i] = fmul2(f[j].p[i], f2pack(act_of(g.get(2 * i), a.gate_act), act_of(g.get(2 * i + 1), a.gate_act)));
      }
      s += total(mul(u, u));
    }
    const float gate = a.gate_mode == kGateRow ? act_of(load_f(a.gate, a.gate_dtype, r), a.gate_act) : 1.f;
    fetch(r + plan.depth * plan.parts, t.ahead.slot);
    t.ahead.next();
    if (branch) {
      if (a.post_weight != nullptr) ru = rsqrtf(t.sum.one(s) * inv + a.eps);
      const float scale = ru * gate;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        y[j] = fma(f[j], scale, mul(y[j], a.residual_scale));
        store8<TX, VEC>(static_cast<TX*>(a.stream_out) + r * cols, y[j], j, tid, team, cols);
      }
    }
    float ry = 1.f;
    if (a.pre_weight != nullptr) {
      s = 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j) s += total(mul(y[j], y[j]));
      ry = rsqrtf(t.sum.one(s) * inv + a.eps);
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        store8<TU, VEC>(static_cast<TU*>(a.norm_out) + r * cols, mul(mul(y[j], ry), w[j]), j, tid, team, cols);
    }
    if (a.stats != nullptr && tid == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(ru, ry);
  }
}

template <typename TX, typename TU, int NCH, bool VEC, bool FULL>
__global__ void __launch_bounds__(NCH == 1 ? 256 : 512, NCH == 1 ? 2 : 1)
    residual_norm_team_bwd_kernel(const NormArgs a, const TeamPlan plan, float* partial) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float buf[3 * 64];
  using S = Slots<TX, TU, NCH>;
  Team<NCH, VEC> t(a, plan, smem, buf, S::backward);
  if (t.id >= plan.teams) return;
  const int tid = t.tid, team = t.team, cols = a.cols;
  V8 k[NCH], w[NCH], acc_pre[NCH], acc_s[NCH];
  load_factors<NCH, VEC>(a, t.group, tid, team, k, w);
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    acc_pre[j].fill(0.f);
    acc_s[j].fill(0.f);
  }
  const float inv = 1.f / float(cols);
  const bool normed = a.d_normed != nullptr, post = a.post_weight != nullptr, branch = a.branch != nullptr;
  const float rs = branch ? a.residual_scale : 1.f;
  const TX* px = static_cast<const TX*>(a.x);
  const TU* pu = static_cast<const TU*>(a.branch);
  const TU* pg = static_cast<const TU*>(a.gate);
  const TX* pdy = static_cast<const TX*>(a.d_stream);
  const TU* pdh = static_cast<const TU*>(a.d_normed);
  auto fetch = [&](int64_t r, int s) {
    if (r < t.end) {
      if (normed) {
        t.ahead.fetch(px + r * a.ld_x, S::x, s, tid, team, cols);
        t.ahead.fetch(pdh + r * a.ld_d_normed, S::dh, s, tid, team, cols);
      }
      if (branch) t.ahead.fetch(pu + r * a.ld_branch, S::u, s, tid, team, cols);
      if (FULL) t.ahead.fetch(pg + r * a.ld_gate, S::gate, s, tid, team, cols);
      if (pdy != nullptr) t.ahead.fetch(pdy + r * a.ld_d_stream, S::dy, s, tid, team, cols);
    }
    t.ahead.commit();
  };
  int64_t r = t.group * plan.group_rows + t.id % plan.parts;
  for (int s = 0; s < plan.depth; ++s) fetch(r + s * plan.parts, s);
  for (; r < t.end; r += plan.parts) {
    float2 st = make_float2(1.f, 1.f);
    if (a.stats != nullptr) st = __ldg(reinterpret_cast<const float2*>(a.stats + 2 * r));
    const float a1 = a.gate_mode == kGateRow ? act_of(load_f(a.gate, a.gate_dtype, r), a.gate_act) : 1.f;
    const float ru = st.x, ry = st.y;
    t.ahead.wait();
    V8 z[NCH], uh[NCH], f[NCH];  // dz; u r_u; k with the row's or the element's gate
    if (branch) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        uh[j] = mul(t.ahead.take(pu + r * a.ld_branch, S::u, j, tid, team, cols), ru);
        f[j] = a.gate_mode == kGateRow ? mul(k[j], a1) : k[j];
        if (FULL) {
          const V8 g = t.ahead.take(pg + r * a.ld_gate, S::gate, j, tid, team, cols);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            f[j].p[i] = fmul2(f[j].p[i], f2pack(act_of(g.get(2 * i), a.gate_act), act_of(g.get(2 * i + 1), a.gate_act)));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if (pdy != nullptr) z[j] = t.ahead.take(pdy + r * a.ld_d_stream, S::dy, j, tid, team, cols);
      else z[j].fill(0.f);
    }
    if (normed) {
      V8 yh[NCH];
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const V8 x = mul(t.ahead.take(px + r * a.ld_x, S::x, j, tid, team, cols), rs);
        yh[j] = mul(branch ? fma(f[j], uh[j], x) : x, ry);
        const V8 d = t.ahead.take(pdh + r * a.ld_d_normed, S::dh, j, tid, team, cols);
        acc_pre[j] = fma(d, yh[j], acc_pre[j]);
        const V8 dw = mul(d, w[j]);
        dot += total(mul(dw, yh[j]));
        z[j] = fma(dw, ry, z[j]);
      }
      const float mean = t.sum.one(dot) * (inv * ry);
#pragma unroll
      for (int j = 0; j < NCH; ++j) z[j] = fma(yh[j], -mean, z[j]);
    }
    float dot_u = 0.f, dot_g = 0.f;
    if (branch) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const V8 zu = mul(z[j], uh[j]);
        if (post) dot_u += total(mul(f[j], zu));
        if (a.gate_mode == kGateRow) dot_g += total(mul(k[j], zu));
        if (FULL) {
          const V8 g = t.ahead.take(pg + r * a.ld_gate, S::gate, j, tid, team, cols);
          V8 dg = mul(k[j], zu), act;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float g0 = act_of(g.get(2 * i), a.gate_act), g1 = act_of(g.get(2 * i + 1), a.gate_act);
            act.p[i] = f2pack(g0, g1);
            dg.p[i] = fmul2(dg.p[i], f2pack(act_slope(g0, a.gate_act), act_slope(g1, a.gate_act)));
          }
          acc_s[j] = fma(act, zu, acc_s[j]);
          if (a.d_gate != nullptr) store8<TU, VEC>(static_cast<TU*>(a.d_gate) + r * cols, dg, j, tid, team, cols);
        } else {
          acc_s[j] = fma(zu, a1, acc_s[j]);
        }
      }
    }
    fetch(r + plan.depth * plan.parts, t.ahead.slot);
    t.ahead.next();
    if (a.d_x != nullptr) {
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        store8<TX, VEC>(static_cast<TX*>(a.d_x) + r * cols, mul(z[j], rs), j, tid, team, cols);
    }
    if (!branch) continue;
    float mean_u = 0.f;
    if (a.gate_mode == kGateRow) {
      const float2 s = t.sum.two(dot_u, dot_g);
      mean_u = s.x * inv;
      if (tid == 0 && a.d_gate != nullptr) static_cast<float*>(a.d_gate)[r] = act_slope(a1, a.gate_act) * s.y;
    } else if (post) {
      mean_u = t.sum.one(dot_u) * inv;
    }
    if (a.d_branch != nullptr) {
      mean_u = post ? -mean_u * ru : 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        store8<TU, VEC>(static_cast<TU*>(a.d_branch) + r * cols, fma(uh[j], mean_u, mul(mul(f[j], z[j]), ru)), j, tid, team,
                        cols);
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < NCH; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<VEC>(j, i, tid, team);
      if (c >= cols) continue;
      partial[t.id * cols + c] = acc_pre[j].get(i);
      partial[(plan.teams + t.id) * cols + c] = acc_s[j].get(i);
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
  int ctas_per_sm;
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
  s.ctas_per_sm = per_sm / s.threads > 0 ? int(per_sm / s.threads) : 1;
  const int64_t want = int64_t(s.ctas_per_sm) * num_sms() * s.rows_per_cta;
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

// Rows ahead: up to four, as many as the CTAs that are resident at once have room for.
constexpr int kAheadBytes = 200 * 1024;  // of an SM's shared memory

template <typename TX, typename TU, int NCH, bool VEC, bool FULL>
int launch_team(const NormArgs& a, NormShape s, bool backward, float* partial, cudaStream_t stream) {
  using S = Slots<TX, TU, NCH>;
  const int stage = s.threads * 16 * int(backward ? S::backward : FULL ? S::forward : S::gate);
  int depth = kAheadBytes / s.ctas_per_sm / stage;
  depth = depth > 4 ? 4 : depth < 1 ? 1 : depth;
  const int smem = VEC ? depth * stage : 0;
  s.plan.depth = VEC ? depth : 0;
  const unsigned grid = unsigned((s.plan.teams + s.rows_per_cta - 1) / s.rows_per_cta);
  if (backward) {
    static std::atomic<uint64_t> raised{0};
    if (VEC && !raise_smem_limit(residual_norm_team_bwd_kernel<TX, TU, NCH, VEC, FULL>, 220 * 1024, raised))
      return MCL4MOE_ERR_CUDA;
    residual_norm_team_bwd_kernel<TX, TU, NCH, VEC, FULL><<<grid, s.threads, smem, stream>>>(a, s.plan, partial);
  } else {
    static std::atomic<uint64_t> raised{0};
    if (VEC && !raise_smem_limit(residual_norm_team_kernel<TX, TU, NCH, VEC, FULL>, 220 * 1024, raised))
      return MCL4MOE_ERR_CUDA;
    residual_norm_team_kernel<TX, TU, NCH, VEC, FULL><<<grid, s.threads, smem, stream>>>(a, s.plan);
  }
  return MCL4MOE_OK;
}
template <typename TX, typename TU, int NCH, bool VEC>
int launch_team(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  return a.gate_mode == kGateFull ? launch_team<TX, TU, NCH, VEC, true>(a, s, backward, partial, stream)
                                  : launch_team<TX, TU, NCH, VEC, false>(a, s, backward, partial, stream);
}
template <typename TX, typename TU>
int launch_team(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  const bool vec = norm_vectors(a);
  if (s.wide)
    return vec ? launch_team<TX, TU, 2, true>(a, s, backward, partial, stream)
               : launch_team<TX, TU, 2, false>(a, s, backward, partial, stream);
  return vec ? launch_team<TX, TU, 1, true>(a, s, backward, partial, stream)
             : launch_team<TX, TU, 1, false>(a, s, backward, partial, stream);
}
int launch_teams(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  if (a.x_dtype == 1) {
    if (a.norm_dtype == 0) return launch_team<float, uint16_t>(a, s, backward, partial, stream);
    if (a.norm_dtype == 1) return launch_team<float, float>(a, s, backward, partial, stream);
    return launch_team<float, __half>(a, s, backward, partial, stream);
  }
  if (a.x_dtype == 0) return launch_team<uint16_t, uint16_t>(a, s, backward, partial, stream);
  return launch_team<__half, __half>(a, s, backward, partial, stream);
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
    const int team = launch_teams(*a, s, false, nullptr, stream);
    if (team != MCL4MOE_OK) return team;
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
    const int team = launch_teams(*a, s, true, partial, stream);
    if (team != MCL4MOE_OK) return team;
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
