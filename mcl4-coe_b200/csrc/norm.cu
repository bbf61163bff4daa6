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
// 32768 x 2048 bf16 with both norms and a channel gate: forward 95 us (5.7 TB/s), backward 159 us
// (5.1 TB/s) with the column sums; issue slots (60% busy) and the reductions' latency are what is
// left.  Single elements (32768 x 1001, float32 stream): 92 and 230 us.
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

// The sigmoid's quotient is approximate (2 ulp): half a bf16 step is 2^15 times that.
__device__ __forceinline__ float act_of(float g, int act) {
  return act == kActSigmoid ? __fdividef(1.f, 1.f + expf(-g)) : act == kActTanh ? tanhf(g) : g;
}
// act'(g) from a = act(g)
__device__ __forceinline__ float act_slope(float a, int act) {
  return act == kActSigmoid ? a * (1.f - a) : act == kActTanh ? 1.f - a * a : 1.f;
}

// ---------------------------------------------------------------- rows in registers

// Eight elements of a row per chunk, so laid out that a warp's accesses lie side by side: eight
// consecutive ones (16-bit operands, 16 bytes a thread), twice four (with a 32-bit stream, where
// eight would leave every other 16 bytes to the next access: 16384 x 2048 float32 forward 135 us),
// or every team-th one (odd widths, strides or addresses).
enum { kSingles = 0, kEights = 1, kFours = 2 };
__device__ __forceinline__ float elem_f(float v) { return v; }
__device__ __forceinline__ float elem_f(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float elem_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void elem_set(float& d, float v) { d = v; }
__device__ __forceinline__ void elem_set(uint16_t& d, float v) { d = f32_to_bf16(v); }
__device__ __forceinline__ void elem_set(__half& d, float v) { d = __float2half_rn(v); }

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
__device__ __forceinline__ V8 act8(const V8& g, int act) {
  if (act == kActNone) return g;
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2unpack(g.p[i], a, b);
    r.p[i] = f2pack(act_of(a, act), act_of(b, act));
  }
  return r;
}
__device__ __forceinline__ V8 slope8(const V8& g, int act) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2unpack(g.p[i], a, b);
    r.p[i] = f2pack(act_slope(a, act), act_slope(b, act));
  }
  return r;
}
__device__ __forceinline__ V8 add(const V8& a, const V8& b) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fadd2(a.p[i], b.p[i]);
  return r;
}
// Sum of the products.
__device__ __forceinline__ float dot8(const V8& a, const V8& b) {
  float x, y;
  f2unpack(fadd2(ffma2(a.p[0], b.p[0], fmul2(a.p[1], b.p[1])), ffma2(a.p[2], b.p[2], fmul2(a.p[3], b.p[3]))), x, y);
  return x + y;
}

template <int LAY>
__device__ __forceinline__ int col_of(int chunk, int i, int tid, int team) {
  if (LAY == kEights) return (chunk * team + tid) * 8 + i;
  if (LAY == kFours) return (chunk * 2 + (i >> 2)) * team * 4 + tid * 4 + (i & 3);
  return (chunk * 8 + i) * team + tid;
}

// Two elements of one 32-bit word.
template <typename T>
__device__ __forceinline__ uint64_t unpack2(uint32_t w);
template <>
__device__ __forceinline__ uint64_t unpack2<uint16_t>(uint32_t w) {
  return f2pack(bf16x2_lo(w), bf16x2_hi(w));
}
template <>
__device__ __forceinline__ uint64_t unpack2<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2pack(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(uint64_t v);
template <>
__device__ __forceinline__ uint32_t pack2<uint16_t>(uint64_t v) {
  float a, b;
  f2unpack(v, a, b);
  return pack_bf16x2(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(uint64_t v) {
  float a, b;
  f2unpack(v, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ V8 load8(const T* row, int chunk, int tid, int team, int cols) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = col_of<kSingles>(chunk, i, tid, team);
    v[i] = c < cols ? elem_f(__ldg(row + c)) : 0.f;
  }
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = f2pack(v[2 * i], v[2 * i + 1]);
  return r;
}
template <typename T, int LAY>
__device__ __forceinline__ void store8(T* row, const V8& v, int chunk, int tid, int team, int cols) {
  if constexpr (LAY == kSingles) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<kSingles>(chunk, i, tid, team);
      if (c < cols) elem_set(row[c], v.get(i));
    }
  } else if constexpr (LAY == kEights) {
    const int c = col_of<kEights>(chunk, 0, tid, team);
    if (c >= cols) return;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 lo = *reinterpret_cast<const uint2*>(&v.p[2 * h]), hi = *reinterpret_cast<const uint2*>(&v.p[2 * h + 1]);
        *reinterpret_cast<uint4*>(row + c + 4 * h) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    } else {
      *reinterpret_cast<uint4*>(row + c) = make_uint4(pack2<T>(v.p[0]), pack2<T>(v.p[1]), pack2<T>(v.p[2]), pack2<T>(v.p[3]));
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = col_of<kFours>(chunk, 4 * h, tid, team);
      if (c >= cols) continue;
      if constexpr (sizeof(T) == 4) {
        const uint2 lo = *reinterpret_cast<const uint2*>(&v.p[2 * h]), hi = *reinterpret_cast<const uint2*>(&v.p[2 * h + 1]);
        *reinterpret_cast<uint4*>(row + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      } else {
        *reinterpret_cast<uint2*>(row + c) = make_uint2(pack2<T>(v.p[2 * h]), pack2<T>(v.p[2 * h + 1]));
      }
    }
  }
}

// First element of a row: one wide multiply-add from launch constants, so that a row costs no
// registers between its uses.
template <typename T>
__device__ __forceinline__ T* row_at(T* base, uint32_t row, uint32_t ld_bytes) {
  return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(base) + uint64_t(row) * ld_bytes);
}

// The rows ahead of a thread, in shared memory: it copies its own elements there (cp.async, 16
// bytes each) `depth` rows ahead and reads them back itself, so that no barrier stands between and
// the loads in flight need no registers.  A row has a 16-byte piece for each eight 16-bit or four
// 32-bit elements of an operand; a thread's pieces lie `stride` bytes apart.
// Single elements come straight from memory when they are asked for.
template <int NCH, int LAY>
struct Ahead {
  uint32_t mine;    // shared address of this thread's first piece
  uint32_t stride, stage, end;  // bytes: between pieces, of a row, of all rows
  uint32_t slot;    // offset of the row at work
  int depth, tid, team, cols;
  bool in[2 * NCH];  // the half chunk lies inside the row

  template <int BYTES>
  static __device__ __forceinline__ void copy(uint32_t to, const void* from) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
  }
  template <typename T>
  __device__ __forceinline__ void fetch(const T* row, uint32_t at, uint32_t to) const {
    if constexpr (LAY == kEights) {
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        if (in[2 * j]) copy<16>(mine + to + (at + j) * stride, row + col_of<LAY>(j, 0, tid, team));
    } else if constexpr (LAY == kFours) {
#pragma unroll
      for (int h = 0; h < 2 * NCH; ++h)
        if (in[h]) {
          const T* from = row + col_of<LAY>(h >> 1, 4 * (h & 1), tid, team);
          if constexpr (sizeof(T) == 4) copy<16>(mine + to + (at + h) * stride, from);
          else copy<8>(mine + to + (at + (h >> 1)) * stride + 8 * (h & 1), from);
        }
    }
  }
  template <typename T>
  __device__ __forceinline__ V8 take(const T* row, uint32_t at, int j) const {
    if constexpr (LAY == kSingles) {
      return load8(row, j, tid, team, cols);
    } else {
      V8 r;
      const uint32_t from = mine + slot + (at + j * uint32_t(sizeof(T) / 2)) * stride;
      const uint4 w = lds16(from);
      if constexpr (sizeof(T) == 4) {
        const uint4 v = lds16(from + stride);
        r.p[0] = f2pack(__uint_as_float(w.x), __uint_as_float(w.y));
        r.p[1] = f2pack(__uint_as_float(w.z), __uint_as_float(w.w));
        r.p[2] = f2pack(__uint_as_float(v.x), __uint_as_float(v.y));
        r.p[3] = f2pack(__uint_as_float(v.z), __uint_as_float(v.w));
      } else {
        r.p[0] = unpack2<T>(w.x);
        r.p[1] = unpack2<T>(w.y);
        r.p[2] = unpack2<T>(w.z);
        r.p[3] = unpack2<T>(w.w);
      }
      return r;
    }
  }
  static __device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
    return w;
  }
  // Chunks behind the row's end are never fetched: zero once, zero for all rows.
  __device__ __forceinline__ void clear() const {
    if constexpr (LAY != kSingles) {
      bool all = true;
#pragma unroll
      for (int j = 0; j < 2 * NCH; ++j) all = all && in[j];
      if (!all)
        for (uint32_t at = 0; at < end; at += stride)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(mine + at), "r"(0) : "memory");
    }
  }
  // Eight values of this thread's own, behind the rows.
  __device__ __forceinline__ void keep(int which, const V8& v) const {
    const uint32_t to = mine + end + uint32_t(2 * which) * stride;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float a, b, c, d;
      f2unpack(v.p[2 * h], a, b);
      f2unpack(v.p[2 * h + 1], c, d);
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + h * stride), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
    }
  }
  __device__ __forceinline__ V8 kept(int which) const {
    V8 r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 w = lds16(mine + end + uint32_t(2 * which + h) * stride);
      r.p[2 * h] = f2pack(__uint_as_float(w.x), __uint_as_float(w.y));
      r.p[2 * h + 1] = f2pack(__uint_as_float(w.z), __uint_as_float(w.w));
    }
    return r;
  }
  __device__ __forceinline__ void commit() const {
    if (LAY != kSingles) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The oldest of `depth` committed rows is there.
  __device__ __forceinline__ void wait() const {
    if (LAY == kSingles) return;
    if (depth >= 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  __device__ __forceinline__ void next() { slot = slot + stage == end ? 0 : slot + stage; }
};

// Sums over the team, the same order every time; every thread gets them.  One barrier per call:
// three buffers in turn, so that a buffer is written again only behind the barrier after its reads.
template <int WARPS>
struct TeamSum {
  float* buf;  // [3][2][WARPS] shared, zero where there is no such warp; or null for a one-warp team
  int turn;
  static __device__ __forceinline__ float across(const float* t) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w += 4) {
      const float4 v = *reinterpret_cast<const float4*>(t + w);
      s += (v.x + v.y) + (v.z + v.w);
    }
    return s;
  }
  __device__ __forceinline__ float one(float a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (buf == nullptr) return a;
    float* t = buf + turn;
    turn = turn == 4 * WARPS ? 0 : turn + 2 * WARPS;
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
    float* t = buf + turn;
    turn = turn == 4 * WARPS ? 0 : turn + 2 * WARPS;
    if ((threadIdx.x & 31) == 0) {
      t[threadIdx.x >> 5] = a;
      t[WARPS + (threadIdx.x >> 5)] = b;
    }
    __syncthreads();
    return make_float2(across(t), across(t + WARPS));
  }
};

// Column factors of the team: k = bs act(g) w_post (the gate only where it is the columns'), w = w_pre.
template <int NCH, int LAY>
__device__ __forceinline__ void load_factors(const NormArgs& a, int64_t group, int tid, int team, V8 (&k)[NCH],
                                             V8 (&w)[NCH]) {
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    float kf[8], wf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<LAY>(j, i, tid, team);
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
  static constexpr uint32_t u = px, dy = px + pu, dh = 2 * px + pu, gate_b = 2 * px + 2 * pu;
  static constexpr uint32_t gate = px + pu, forward = px + 2 * pu, plain = 2 * px + 2 * pu, backward = 2 * px + 3 * pu;
};

constexpr int kBwdCtas = 3;  // of the backward's small teams, resident together

// Warps of the largest team.
template <int NCH>
constexpr int kTeamWarps = NCH == 1 ? 8 : 16;

// What a team works on: its place in the CTA, its rows and the rows ahead.
template <int NCH, int LAY>
struct Team {
  int team, tid;
  int64_t id, group;
  uint32_t row;  // the first
  int rows;
  TeamSum<kTeamWarps<NCH>> sum;
  Ahead<NCH, LAY> ahead;
  __device__ __forceinline__ Team(const NormArgs& a, const TeamPlan& plan, char* smem, float* buf, uint32_t pieces) {
    const bool warp_team = a.cols <= 256;
    team = warp_team ? 32 : int(blockDim.x);
    tid = warp_team ? int(threadIdx.x & 31) : int(threadIdx.x);
    id = warp_team ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : int64_t(blockIdx.x);
    group = id / plan.parts;
    sum = TeamSum<kTeamWarps<NCH>>{warp_team ? nullptr : buf, 0};
    if (!warp_team) {
      for (int i = threadIdx.x; i < 6 * kTeamWarps<NCH>; i += blockDim.x) buf[i] = 0.f;
      __syncthreads();
    }
    ahead.mine = uint32_t(__cvta_generic_to_shared(smem)) + threadIdx.x * 16;
    ahead.stride = blockDim.x * 16;
    ahead.stage = ahead.stride * pieces;
    ahead.end = ahead.stage * plan.depth;
    ahead.slot = 0;
    ahead.depth = plan.depth;
    ahead.tid = tid;
    ahead.team = team;
    ahead.cols = a.cols;
#pragma unroll
    for (int h = 0; h < 2 * NCH; ++h) ahead.in[h] = col_of<LAY>(h >> 1, 4 * (h & 1), tid, team) < a.cols;
    ahead.clear();
    const int64_t part = id % plan.parts;
    row = uint32_t(group * plan.group_rows + part);
    rows = int((plan.group_rows - part + plan.parts - 1) / plan.parts);
  }
};

template <typename TX, typename TU, int NCH, int LAY, bool GATED>
__global__ void __launch_bounds__(NCH == 1 ? 256 : 512, NCH == 1 ? 3 : 1)
    residual_norm_team_kernel(const NormArgs a, const TeamPlan plan) {
  extern __shared__ __align__(16) char smem[];
  __shared__ __align__(16) float buf[3 * 2 * kTeamWarps<NCH>];
  using S = Slots<TX, TU, NCH>;
  Team<NCH, LAY> t(a, plan, smem, buf, GATED ? S::forward : S::gate);
  if (t.id >= plan.teams) return;  // a whole team: no barrier is left behind
  const int tid = t.tid, team = t.team, cols = a.cols;
  V8 k[NCH], w[NCH];
  load_factors<NCH, LAY>(a, t.group, tid, team, k, w);
  const float inv = 1.f / float(cols);
  const bool branch = a.branch != nullptr;
  Ahead<NCH, LAY>& ahead = t.ahead;
  uint32_t r = t.row;
  const uint32_t parts = uint32_t(plan.parts);
  const int rows = t.rows, depth = plan.depth;
  // GATED: a gate of rows or elements; the columns' is in k
  const bool full = GATED && a.gate_mode == kGateFull, by_row = GATED && a.gate_mode == kGateRow;
  const uint32_t ld_x = uint32_t(a.ld_x * sizeof(TX)), ld_u = uint32_t(a.ld_branch * sizeof(TU));
  const uint32_t ld_g = uint32_t(a.ld_gate * sizeof(TU)), out_x = uint32_t(cols * sizeof(TX)), out_u = uint32_t(cols * sizeof(TU));
  auto x_row = [&](uint32_t row) { return row_at(static_cast<const TX*>(a.x), row, ld_x); };
  auto u_row = [&](uint32_t row) { return row_at(static_cast<const TU*>(a.branch), row, ld_u); };
  auto g_row = [&](uint32_t row) { return row_at(static_cast<const TU*>(a.gate), row, ld_g); };
  auto fetch = [&](bool there, uint32_t row, uint32_t to) {
    if (there) {
      ahead.fetch(x_row(row), S::x, to);
      if (branch) ahead.fetch(u_row(row), S::u, to);
      if (full) ahead.fetch(g_row(row), S::gate, to);
    }
    ahead.commit();
  };
  float g1 = by_row ? load_f(a.gate, a.gate_dtype, r) : 1.f;
  for (int s = 0; s < depth; ++s) fetch(s < rows, r + s * parts, s * ahead.stage);
  for (int n = 0; n < rows; ++n, r += parts) {
    ahead.wait();
    V8 y[NCH], f[NCH];
    float ru = 1.f, s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      y[j] = ahead.take(x_row(r), S::x, j);
      if (!branch) continue;
      const V8 v = ahead.take(u_row(r), S::u, j);
      f[j] = mul(v, k[j]);
      if (full) f[j] = mul(f[j], act8(ahead.take(g_row(r), S::gate, j), a.gate_act));
      s += dot8(v, v);
    }
    const float gate = by_row ? act_of(g1, a.gate_act) : 1.f;
    if (by_row && n + 1 < rows) g1 = load_f(a.gate, a.gate_dtype, r + parts);
    fetch(n + depth < rows, r + depth * parts, ahead.slot);
    ahead.next();
    if (branch) {
      if (a.post_weight != nullptr) ru = rsqrtf(t.sum.one(s) * inv + a.eps);
      const float scale = ru * gate;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        y[j] = fma(f[j], scale, mul(y[j], a.residual_scale));
        store8<TX, LAY>(row_at(static_cast<TX*>(a.stream_out), r, out_x), y[j], j, tid, team, cols);
      }
    }
    float ry = 1.f;
    if (a.pre_weight != nullptr) {
      s = 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j) s += dot8(y[j], y[j]);
      ry = rsqrtf(t.sum.one(s) * inv + a.eps);
#pragma unroll
      for (int j = 0; j < NCH; ++j)
        store8<TU, LAY>(row_at(static_cast<TU*>(a.norm_out), r, out_u), mul(mul(y[j], ry), w[j]), j, tid, team, cols);
    }
    if (a.stats != nullptr && tid == 0) *row_at(reinterpret_cast<float2*>(a.stats), r, 8u) = make_float2(ru, ry);
  }
}

// The columns' factors lie in shared memory behind the rows ahead, each thread's its own, so that
// the registers hold two column sums and the row (three values a column) alone: 3 CTAs of 256
// threads an SM instead of 2, and no spills with 16 columns a thread.  TG: type of an element-wise
// gate's gradient, float for a caller that adds it up over rows (in one kernel with both types the
// token gates' gradient with a float32 stream took 245 us for 236).
template <typename TX, typename TU, int NCH, int LAY, bool GATED, typename TG>
__global__ void __launch_bounds__(NCH == 1 ? 256 : 512, NCH == 1 ? kBwdCtas : 1)
    residual_norm_team_bwd_kernel(const NormArgs a, const TeamPlan plan, float* partial) {
  extern __shared__ __align__(16) char smem[];
  __shared__ __align__(16) float buf[3 * 2 * kTeamWarps<NCH>];
  using S = Slots<TX, TU, NCH>;
  Team<NCH, LAY> t(a, plan, smem, buf, GATED ? S::backward : S::plain);
  if (t.id >= plan.teams) return;
  const int tid = t.tid, team = t.team, cols = a.cols;
  Ahead<NCH, LAY>& ahead = t.ahead;
  V8 acc_pre[NCH], acc_s[NCH];
  {
    V8 k[NCH], w[NCH];
    load_factors<NCH, LAY>(a, t.group, tid, team, k, w);
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      ahead.keep(2 * j, k[j]);
      ahead.keep(2 * j + 1, w[j]);
      acc_pre[j].fill(0.f);
      acc_s[j].fill(0.f);
    }
  }
  const float inv = 1.f / float(cols);
  const bool normed = a.d_normed != nullptr, post = a.post_weight != nullptr, branch = a.branch != nullptr;
  const bool streamed = a.d_stream != nullptr;
  const float rs = branch ? a.residual_scale : 1.f;
  uint32_t r = t.row;
  const uint32_t parts = uint32_t(plan.parts);
  const int rows = t.rows, depth = plan.depth;
  // GATED: a gate of rows or elements; the columns' is in k
  const bool full = GATED && a.gate_mode == kGateFull, by_row = GATED && a.gate_mode == kGateRow;
  const uint32_t ld_x = uint32_t(a.ld_x * sizeof(TX)), ld_u = uint32_t(a.ld_branch * sizeof(TU));
  const uint32_t ld_g = uint32_t(a.ld_gate * sizeof(TU)), out_x = uint32_t(cols * sizeof(TX)), out_u = uint32_t(cols * sizeof(TU));
  auto x_row = [&](uint32_t row) { return row_at(static_cast<const TX*>(a.x), row, ld_x); };
  auto u_row = [&](uint32_t row) { return row_at(static_cast<const TU*>(a.branch), row, ld_u); };
  auto g_row = [&](uint32_t row) { return row_at(static_cast<const TU*>(a.gate), row, ld_g); };
  const uint32_t ld_dy = uint32_t(a.ld_d_stream * sizeof(TX)), ld_dh = uint32_t(a.ld_d_normed * sizeof(TU));
  auto dy_row = [&](uint32_t row) { return row_at(static_cast<const TX*>(a.d_stream), row, ld_dy); };
  auto dh_row = [&](uint32_t row) { return row_at(static_cast<const TU*>(a.d_normed), row, ld_dh); };
  auto fetch = [&](bool there, uint32_t row, uint32_t to) {
    if (there) {
      if (normed) {
        ahead.fetch(x_row(row), S::x, to);
        ahead.fetch(dh_row(row), S::dh, to);
      }
      if (branch) ahead.fetch(u_row(row), S::u, to);
      if (full) ahead.fetch(g_row(row), S::gate_b, to);
      if (streamed) ahead.fetch(dy_row(row), S::dy, to);
    }
    ahead.commit();
  };
  float2 st = make_float2(1.f, 1.f);
  float g1 = 1.f;
  auto scalars = [&](uint32_t row) {
    if (a.stats != nullptr) st = __ldg(row_at(reinterpret_cast<const float2*>(a.stats), row, 8u));
    if (by_row) g1 = load_f(a.gate, a.gate_dtype, row);
  };
  scalars(r);
  for (int s = 0; s < depth; ++s) fetch(s < rows, r + s * parts, s * ahead.stage);
  for (int n = 0; n < rows; ++n, r += parts) {
    const float ru = st.x, ry = st.y, a1 = by_row ? act_of(g1, a.gate_act) : 1.f;
    if (n + 1 < rows) scalars(r + parts);  // the next row's, a row ahead
    ahead.wait();
    V8 z[NCH], uh[NCH], act[NCH];  // dz; u r_u; the element's gate
    // single elements come from memory: all of them are asked for before the first is used
    V8 x1[NCH], dh1[NCH];
    if constexpr (LAY == kSingles) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        if (branch) uh[j] = ahead.take(u_row(r), S::u, j);
        if (streamed) z[j] = ahead.take(dy_row(r), S::dy, j);
        if (normed) {
          x1[j] = ahead.take(x_row(r), S::x, j);
          dh1[j] = ahead.take(dh_row(r), S::dh, j);
        }
      }
    }
    if (branch) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        uh[j] = mul(LAY == kSingles ? uh[j] : ahead.take(u_row(r), S::u, j), ru);
        if (full) act[j] = act8(ahead.take(g_row(r), S::gate_b, j), a.gate_act);
      }
    }
    // k of a column with the row's or the element's gate
    auto factor = [&](int j) {
      V8 k = ahead.kept(2 * j);
      if (by_row) k = mul(k, a1);
      return full ? mul(k, act[j]) : k;
    };
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if (!streamed) z[j].fill(0.f);
      else if (LAY != kSingles) z[j] = ahead.take(dy_row(r), S::dy, j);
    }
    if (normed) {
      V8 yh[NCH];
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const V8 v = mul(LAY == kSingles ? x1[j] : ahead.take(x_row(r), S::x, j), rs);
        yh[j] = mul(branch ? fma(factor(j), uh[j], v) : v, ry);
        const V8 d = LAY == kSingles ? dh1[j] : ahead.take(dh_row(r), S::dh, j);
        acc_pre[j] = fma(d, yh[j], acc_pre[j]);
        const V8 dw = mul(d, ahead.kept(2 * j + 1));
        dot += dot8(dw, yh[j]);
        z[j] = fma(dw, ry, z[j]);
      }
      const float mean = t.sum.one(dot) * (inv * ry);
#pragma unroll
      for (int j = 0; j < NCH; ++j) z[j] = fma(yh[j], -mean, z[j]);
    }
    fetch(n + depth < rows, r + depth * parts, ahead.slot);
    ahead.next();
    if (a.d_x != nullptr) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) store8<TX, LAY>(row_at(static_cast<TX*>(a.d_x), r, out_x), mul(z[j], rs), j, tid, team, cols);
    }
    if (!branch) continue;
    float dot_u = 0.f, dot_g = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const V8 zu = mul(z[j], uh[j]);
      if (by_row) dot_g += dot8(ahead.kept(2 * j), zu);
      if (full && a.d_gate != nullptr) {
        const V8 g = mul(mul(ahead.kept(2 * j), zu), slope8(act[j], a.gate_act));
        store8<TG, LAY>(row_at(static_cast<TG*>(a.d_gate), r, uint32_t(cols * sizeof(TG))), g, j, tid, team, cols);
      }
      acc_s[j] = full ? fma(act[j], zu, acc_s[j]) : by_row ? fma(zu, a1, acc_s[j]) : add(zu, acc_s[j]);
      z[j] = mul(factor(j), z[j]);
      if (post) dot_u += dot8(z[j], uh[j]);
    }
    float mean_u = 0.f;
    if (by_row) {
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
        store8<TU, LAY>(row_at(static_cast<TU*>(a.d_branch), r, out_u), fma(uh[j], mean_u, mul(z[j], ru)), j, tid, team, cols);
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < NCH; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<LAY>(j, i, tid, team);
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
        store_f(a.d_gate, a.gate_grad_f32 ? 1 : a.gate_dtype, r * a.cols + c, kzu * act_slope(g, a.gate_act));
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
  if (a->cols > kMaxNormCols || a->rows > (int64_t(1) << 31) - 1) return MCL4MOE_ERR_UNSUPPORTED;
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

NormShape norm_shape(int64_t rows, int cols, int gate_mode, int64_t gate_rows, bool backward, bool wide) {
  NormShape s{};
  s.wide = wide;
  const int per = s.wide ? 16 : 8;
  const int need = (cols + per - 1) / per;
  s.threads = cols <= 256 ? 128 : (need + 31) / 32 * 32;
  s.rows_per_cta = cols <= 256 ? 4 : 1;
  if (cols > kTeamCols) s.threads = kNormThreads;
  const int64_t per_sm = cols > kTeamCols ? 512 : s.wide ? 512 : backward ? 256 * kBwdCtas : 768;
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
  const int64_t far = int64_t(1) << 30;  // byte strides in 32 bits
  if (a.ld_x >= far || a.ld_branch >= far || a.ld_gate >= far || a.ld_d_stream >= far || a.ld_d_normed >= far) return false;
  if (a.gate_mode == kGateFull && a.gate_dtype != a.norm_dtype) return false;
  return a.x_dtype == a.norm_dtype || a.x_dtype == 1;
}

// Rows ahead: up to four, as many as the CTAs that are resident at once have room for.
constexpr int kAheadBytes = 200 * 1024;  // of an SM's shared memory
constexpr int kTeamSmem = 224 * 1024;    // of a CTA: one float32 row of 8192 with an element-wise gate and the factors

// 16 columns a thread: needed from 2049 columns on; from 1025 on where a row has more operands or
// wider ones, or a third reduction (a token gate's gradient), which then weigh more than the warps in
// flight.  32768 x 2048, forward / backward in us, 8 against 16 columns a thread: bf16 97 / 162 against
// 103 / 168; token gate 97 / 245 against 88 / 191; element-wise gate 120 / 261 against 120 / 208; float32
// stream 149 / 234 against 138 / 215.  Single elements stay narrow: 32768 x 1501 with a float32 stream
// 135 / 334 against 169 / 521, 32768 x 2047 bf16 204 / 456 against 206 / 730.
bool norm_wide(const NormArgs& a) {
  if (a.cols > 2048 || a.cols <= 1024) return a.cols > 2048;
  return norm_vectors(a) && (a.x_dtype == 1 || a.gate_mode >= kGateRow);
}

template <typename TX, typename TU, int NCH, int LAY, bool GATED>
int launch_team(const NormArgs& a, NormShape s, bool backward, float* partial, cudaStream_t stream) {
  using S = Slots<TX, TU, NCH>;
  const int stage = s.threads * 16 * int(backward ? (GATED ? S::backward : S::plain) : GATED ? S::forward : S::gate);
  const int kept = backward ? s.threads * 16 * 4 * NCH : 0;
  int depth = (kAheadBytes / s.ctas_per_sm - kept) / stage;
  depth = depth > 4 ? 4 : depth < 1 ? 1 : depth;
  const int smem = kept + (LAY != kSingles ? depth * stage : 0);
  s.plan.depth = LAY != kSingles ? depth : 0;
  const unsigned grid = unsigned((s.plan.teams + s.rows_per_cta - 1) / s.rows_per_cta);
  if (backward) {
    const auto launch = [&](auto kernel, std::atomic<uint64_t>& raised) {
      if (!raise_smem_limit(kernel, kTeamSmem, raised)) return MCL4MOE_ERR_CUDA;
      kernel<<<grid, s.threads, smem, stream>>>(a, s.plan, partial);
      return MCL4MOE_OK;
    };
    static std::atomic<uint64_t> raised{0}, raised_f32{0};
    if constexpr (GATED && sizeof(TU) == 2)
      if (a.gate_grad_f32) return launch(residual_norm_team_bwd_kernel<TX, TU, NCH, LAY, GATED, float>, raised_f32);
    return launch(residual_norm_team_bwd_kernel<TX, TU, NCH, LAY, GATED, TU>, raised);
  } else {
    static std::atomic<uint64_t> raised{0};
    if (LAY != kSingles && !raise_smem_limit(residual_norm_team_kernel<TX, TU, NCH, LAY, GATED>, kTeamSmem, raised))
      return MCL4MOE_ERR_CUDA;
    residual_norm_team_kernel<TX, TU, NCH, LAY, GATED><<<grid, s.threads, smem, stream>>>(a, s.plan);
  }
  return MCL4MOE_OK;
}
template <typename TX, typename TU, int NCH, int LAY>
int launch_team(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  return a.gate_mode >= kGateRow ? launch_team<TX, TU, NCH, LAY, true>(a, s, backward, partial, stream)
                                 : launch_team<TX, TU, NCH, LAY, false>(a, s, backward, partial, stream);
}
template <typename TX, typename TU>
int launch_team(const NormArgs& a, const NormShape& s, bool backward, float* partial, cudaStream_t stream) {
  constexpr int kLay = sizeof(TX) == 4 ? kFours : kEights;
  const bool vec = norm_vectors(a);
  if (s.wide)
    return vec ? launch_team<TX, TU, 2, kLay>(a, s, backward, partial, stream)
               : launch_team<TX, TU, 2, kSingles>(a, s, backward, partial, stream);
  return vec ? launch_team<TX, TU, 1, kLay>(a, s, backward, partial, stream)
             : launch_team<TX, TU, 1, kSingles>(a, s, backward, partial, stream);
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
  const NormShape s = norm_shape(a->rows, a->cols, a->gate_mode, a->gate_rows, false, norm_wide(*a));
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
  if (rows <= 0 || cols <= 0 || cols > kMaxNormCols ||
      (gate_mode == kGateChannel && (gate_rows <= 0 || rows % gate_rows != 0)))
    return 0;
  int64_t teams = 0, groups = 0;  // of either width of the teams
  for (int wide = cols > 2048; wide < 2; ++wide) {
    const NormShape s = norm_shape(rows, cols, gate_mode, gate_rows, true, wide != 0);
    teams = s.plan.teams > teams ? s.plan.teams : teams;
    groups = s.groups;
  }
  return size_t(2 * teams + (groups > 1 ? groups : 0)) * size_t(cols) * sizeof(float);
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
  const NormShape s = norm_shape(a->rows, a->cols, a->gate_mode, a->gate_rows, true, norm_wide(*a));
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
