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
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace mcl4 {
namespace {

constexpr int kMaxNormCols = 16384;
constexpr int kNormThreads = 256;

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
  __device__ float n(int c) const { return a.post_weight ? u(c) * ru * __ldg(a.post_weight + c) : u(c); }
  __device__ float y(int c) const {
    if (a.branch == nullptr) return x(c);
    return a.residual_scale * x(c) + a.branch_scale * (gate(c) * n(c));
  }
};

__global__ void __launch_bounds__(kNormThreads) residual_norm_kernel(const NormArgs a) {
  __shared__ float tmp[32];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    Row row{a, r, 0.f, 0.f};
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
    if (a.pre_weight == nullptr) continue;
    row.ry = rsqrtf(cta_sum(sum, tmp) / float(a.cols) + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += kNormThreads)
      store_f(a.norm_out, a.norm_dtype, r * a.cols + c, row.y(c) * row.ry * __ldg(a.pre_weight + c));
  }
}

// One CTA per part of a gate group's rows; the column sums of the part stay in shared memory
// (each column belongs to one thread) and leave as one row of `partial` per sum.
__global__ void __launch_bounds__(kNormThreads) residual_norm_bwd_kernel(const NormArgs a, int parts, float* partial) {
  extern __shared__ float acc[];  // [3][cols]: pre, post, gate
  __shared__ float tmp[32];
  const int64_t group_rows = a.gate_mode == kGateChannel ? a.gate_rows : a.rows;
  const int64_t group = blockIdx.x / parts, part = blockIdx.x % parts;
  const int64_t each = (group_rows + parts - 1) / parts;
  const int64_t first = group * group_rows + part * each;
  const int64_t end = min(first + each, (group + 1) * group_rows);
  for (int c = threadIdx.x; c < 3 * a.cols; c += kNormThreads) acc[c] = 0.f;
  __syncthreads();
  const float inv = 1.f / float(a.cols);
  for (int64_t r = first; r < end; ++r) {
    Row row{a, r, 0.f, 0.f};
    const bool normed = a.pre_weight != nullptr && a.d_normed != nullptr;
    if (a.branch != nullptr && a.post_weight != nullptr) {
      float sum = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += kNormThreads) sum += row.u(c) * row.u(c);
      row.ru = rsqrtf(cta_sum(sum, tmp) * inv + a.eps);
    }
    float mean_t = 0.f;
    if (normed) {
      float sum = 0.f, dot = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
        const float y = row.y(c);
        sum += y * y;
        dot += load_f(a.d_normed, a.norm_dtype, r * a.ld_d_normed + c) * __ldg(a.pre_weight + c) * y;
      }
      row.ry = rsqrtf(cta_sum(sum, tmp) * inv + a.eps);
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
      const float g = row.gate(c), n = row.n(c), bz = a.branch_scale * z, dn = bz * g;
      if (a.gate_mode != kGateNone) {
        const float dg = bz * n * act_slope(g, a.gate_act);
        if (a.gate_mode == kGateChannel) acc[2 * a.cols + c] += dg;
        else if (a.gate_mode == kGateRow) dot_g += dg;
        else if (a.d_gate != nullptr) store_f(a.d_gate, a.gate_dtype, r * a.cols + c, dg);
      }
      if (a.post_weight != nullptr) {
        const float uh = row.u(c) * row.ru;
        acc[a.cols + c] += dn * uh;
        dot_u += dn * __ldg(a.post_weight + c) * uh;
      } else if (a.d_branch != nullptr) {
        store_f(a.d_branch, a.branch_dtype, r * a.cols + c, dn);
      }
    }
    if (a.branch == nullptr) continue;
    if (a.gate_mode == kGateRow) {
      const float sum = cta_sum(dot_g, tmp);
      if (threadIdx.x == 0 && a.d_gate != nullptr) static_cast<float*>(a.d_gate)[r] = sum;
    }
    if (a.post_weight != nullptr) {
      const float mean_u = cta_sum(dot_u, tmp) * inv;
      if (a.d_branch != nullptr)
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
          const float dn = a.branch_scale * dz(c) * row.gate(c);
          store_f(a.d_branch, a.branch_dtype, r * a.cols + c,
                  row.ru * (dn * __ldg(a.post_weight + c) - row.u(c) * row.ru * mean_u));
        }
    }
  }
  if (partial == nullptr) return;
  __syncthreads();
  for (int s = 0; s < 3; ++s)
    for (int c = threadIdx.x; c < a.cols; c += kNormThreads)
      partial[(int64_t(s) * gridDim.x + blockIdx.x) * a.cols + c] = acc[s * a.cols + c];
}

// Adds the partial rows in their order: the weights' over all of them, the channel gate's over its group's.
__global__ void __launch_bounds__(256) norm_partials_kernel(const float* partial, int blocks, int parts, int cols,
                                                            float* d_pre, float* d_post, float* d_gate) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  const int which = int(blockIdx.y);
  float* out = which == 0 ? d_pre : which == 1 ? d_post : d_gate;
  if (out == nullptr) return;
  const float* src = partial + int64_t(min(which, 2)) * blocks * cols + c;
  int first = 0, end = blocks;
  if (which >= 2) {
    first = (which - 2) * parts;
    end = first + parts;
    out += int64_t(which - 2) * cols;
  }
  float sum = 0.f;
  for (int b = first; b < end; ++b) sum += src[int64_t(b) * cols];
  out[c] = sum;
}

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
  if (!backward && some &&
      ((a->pre_weight && !a->norm_out) || (a->branch && !a->stream_out) || (!a->branch && !a->pre_weight)))
    return MCL4MOE_ERR_INVALID;
  if (backward && some &&
      ((a->d_stream && a->ld_d_stream < a->cols) || (a->d_normed && (!a->pre_weight || a->ld_d_normed < a->cols))))
    return MCL4MOE_ERR_INVALID;
  if (a->cols > kMaxNormCols) return MCL4MOE_ERR_UNSUPPORTED;
  return MCL4MOE_OK;
}

// CTAs per gate group in the backward (one group without a channel gate), and groups.
void norm_parts(int64_t rows, int gate_mode, int64_t gate_rows, int64_t& groups, int64_t& parts) {
  groups = gate_mode == kGateChannel ? rows / gate_rows : 1;
  const int64_t group_rows = gate_mode == kGateChannel ? gate_rows : rows;
  const int64_t want = 2 * num_sms();
  parts = groups >= want ? 1 : want / groups;
  if (parts > group_rows) parts = group_rows;
  if (parts < 1) parts = 1;
}

}  // namespace
}  // namespace mcl4

using namespace mcl4;

extern "C" {

int mcl4moe_residual_norm(const mcl4moe_norm_args* a, mcl4moe_stream_t stream) {
  const int st = check_norm(a, false);
  if (st != MCL4MOE_OK) return st;
  if (a->rows == 0) return MCL4MOE_OK;
  const int64_t grid = a->rows < int64_t(64) * num_sms() ? a->rows : int64_t(64) * num_sms();
  residual_norm_kernel<<<unsigned(grid), kNormThreads, 0, stream>>>(*a);
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

size_t mcl4moe_residual_norm_workspace_size(int64_t rows, int cols, int gate_mode, int64_t gate_rows) {
  if (rows <= 0 || cols <= 0 || cols > kMaxNormCols || (gate_mode == kGateChannel && gate_rows <= 0)) return 0;
  int64_t groups, parts;
  norm_parts(rows, gate_mode, gate_rows, groups, parts);
  return size_t(3) * size_t(groups * parts) * size_t(cols) * sizeof(float);
}

int mcl4moe_residual_norm_backward(const mcl4moe_norm_args* a, void* workspace, size_t workspace_bytes,
                                   mcl4moe_stream_t stream) {
  const int st = check_norm(a, true);
  if (st != MCL4MOE_OK) return st;
  float* d_gate = a->gate_mode == kGateChannel ? static_cast<float*>(a->d_gate) : nullptr;
  const bool sums = a->d_pre || a->d_post || d_gate;
  if (a->rows == 0) {
    if ((a->d_pre && cudaMemsetAsync(a->d_pre, 0, sizeof(float) * a->cols, stream) != cudaSuccess) ||
        (a->d_post && cudaMemsetAsync(a->d_post, 0, sizeof(float) * a->cols, stream) != cudaSuccess))
      return MCL4MOE_ERR_CUDA;
    return MCL4MOE_OK;
  }
  int64_t groups, parts;
  norm_parts(a->rows, a->gate_mode, a->gate_rows, groups, parts);
  if (groups * parts > (int64_t(1) << 30) || groups > 65533) return MCL4MOE_ERR_UNSUPPORTED;
  if (sums && (!workspace || workspace_bytes < mcl4moe_residual_norm_workspace_size(a->rows, a->cols, a->gate_mode,
                                                                                    a->gate_rows)))
    return MCL4MOE_ERR_WORKSPACE;
  const int smem = 3 * a->cols * int(sizeof(float));
  static std::atomic<uint64_t> raised{0};
  if (!raise_smem_limit(residual_norm_bwd_kernel, 3 * kMaxNormCols * int(sizeof(float)), raised)) return MCL4MOE_ERR_CUDA;
  float* partial = sums ? static_cast<float*>(workspace) : nullptr;
  residual_norm_bwd_kernel<<<unsigned(groups * parts), kNormThreads, smem, stream>>>(*a, int(parts), partial);
  if (sums) {
    const dim3 grid((a->cols + 255) / 256, unsigned(d_gate ? 2 + groups : 2));
    norm_partials_kernel<<<grid, 256, 0, stream>>>(partial, int(groups * parts), int(parts), a->cols, a->d_pre,
                                                   a->d_post, d_gate);
  }
  return cudaGetLastError() == cudaSuccess ? MCL4MOE_OK : MCL4MOE_ERR_CUDA;
}

}  // extern "C"
