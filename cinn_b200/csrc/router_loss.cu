// A router's balance loss, its gradient and the per-expert counts.  x is [tokens, experts], w the tokens' weights,
// c the number of tokens that chose each expert, f = c / sum c; per token q = softmax(x):
//
//   loss = E sum_e f_e sum_t w_t q_te        dx_te = w_t E q_te (f_e - sum_e' f_e' q_te')
//
// The gradient needs the counts alone, so it and the column sums of w q share one pass over the logits: a warp per
// token, the row in registers, the column sums in registers over the tokens of a warp, one partial row per CTA
// (expert_load), and a small kernel that folds the partial rows and the counts into the loss (balance_fold).  Nothing
// is accumulated by floating-point atomics: results do not depend on the order of CTAs.  A token of weight 0 is out:
// it adds nothing, and its gradient row is 0 whatever its logits hold.
#include "device_math.cuh"
#include "kernel_registry.h"

namespace cinn_b200 {
namespace {

constexpr int kWarps = 8;
constexpr int kPer   = 32;  // columns per lane: rows of up to 1024

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    k_router_loss(const T* __restrict__ x, const float* __restrict__ weight, const int* __restrict__ counts,
                  float* __restrict__ out_load, T* __restrict__ out_grad, long long rows, long long cols_ll,
                  double weight_value) {
  grid_dependency_sync();
  __shared__ float f[1024];
  __shared__ float part[kWarps][1024];
  __shared__ float scratch[32];
  const int cols = (int)cols_ll, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (out_grad) {
    // Shares of the choices, less their mean: sum_e q_e = 1, so a constant taken off f changes nothing in
    // f_e - sum f q but its cancellation.
    float total = 0.0f;
    for (int e = threadIdx.x; e < cols; e += blockDim.x) total += (float)counts[e];
    total = cta_allreduce<SumOp>(total, scratch);
    for (int e = threadIdx.x; e < cols; e += blockDim.x)
      f[e] = total > 0.0f ? (float)counts[e] / total - 1.0f / (float)cols : 0.0f;
    __syncthreads();
  }
  float acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.0f;
  for (long long t = (long long)blockIdx.x * kWarps + warp; t < rows; t += (long long)gridDim.x * kWarps) {
    const float w = weight ? weight[t] : (float)weight_value;
    float q[kPer], m = -INFINITY, s = 0.0f, inner = 0.0f;
    if (w != 0.0f) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        q[i]        = e < cols ? Io<T>::load1(x + t * cols + e) : -INFINITY;
        m           = fmaxf(m, q[i]);
      }
      m = warp_allreduce<MaxOp>(m);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        q[i] = lane + 32 * i < cols ? expf(q[i] - m) : 0.0f;
        s += q[i];
      }
      const float inv = 1.0f / warp_allreduce<SumOp>(s);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        q[i] *= inv;
        acc[i] += w * q[i];
        if (out_grad && e < cols) inner += q[i] * f[e];
      }
      inner = warp_allreduce<SumOp>(inner);
    }
    if (!out_grad) continue;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < cols) Io<T>::store1(out_grad + t * cols + e, w != 0.0f ? (float)cols * w * q[i] * (f[e] - inner) : 0.0f);
    }
  }
  if (!out_load) return;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 32 * i < cols) part[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < cols; e += blockDim.x) {
    float v = 0.0f;
    for (int k = 0; k < kWarps; ++k) v += part[k][e];
    out_load[(long long)blockIdx.x * cols + e] = v;
  }
}

// One CTA: a histogram in shared memory (whole numbers: the order of the additions does not show).
__global__ void __launch_bounds__(1024)
    k_expert_counts(const void* __restrict__ index, const float* __restrict__ weight, int* __restrict__ counts,
                    long long rows, long long slots, long long experts, long long wide, double weight_value) {
  grid_dependency_sync();
  __shared__ int bins[1024];
  for (int e = threadIdx.x; e < experts; e += blockDim.x) bins[e] = 0;
  __syncthreads();
  for (long long i = threadIdx.x; i < rows * slots; i += blockDim.x) {
    const long long e = wide ? reinterpret_cast<const long long*>(index)[i] : reinterpret_cast<const int*>(index)[i];
    const float w     = weight ? weight[i / slots] : (float)weight_value;
    if (w != 0.0f && e >= 0 && e < experts) atomicAdd(&bins[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[e] = bins[e];
}

__global__ void __launch_bounds__(1024)
    k_balance_fold(const float* __restrict__ load, const int* __restrict__ counts, float* __restrict__ out,
                   long long slices, long long experts) {
  grid_dependency_sync();
  __shared__ float scratch[32];
  float total = 0.0f, sum = 0.0f;
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    total += (float)counts[e];
    float v = 0.0f;
    for (long long k = 0; k < slices; ++k) v += load[k * experts + e];
    sum += (float)counts[e] * v;
  }
  total = cta_allreduce<SumOp>(total, scratch);
  sum   = cta_allreduce<SumOp>(sum, scratch);
  if (threadIdx.x == 0) out[0] = total > 0.0f ? (float)experts * (sum / total) : 0.0f;
}

}  // namespace

CINN_B200_REGISTER_KERNEL_PDL("router_loss_f32", 8, kWarps * 32, k_router_loss<float>);
CINN_B200_REGISTER_KERNEL_PDL("router_loss_f16", 8, kWarps * 32, k_router_loss<__half>);
CINN_B200_REGISTER_KERNEL_PDL("router_loss_bf16", 8, kWarps * 32, k_router_loss<__nv_bfloat16>);
CINN_B200_REGISTER_KERNEL_PDL("expert_counts", 8, 1024, k_expert_counts);
CINN_B200_REGISTER_KERNEL_PDL("balance_fold", 5, 1024, k_balance_fold);

}  // namespace cinn_b200
