// Losses over rows of logits and their gradients: the log-probability of a chosen token, the clipped policy loss with
// a KL term, distillation from a teacher's top logits.  x is [rows, cols]; per row, with z = x / temperature:
//
//   lse = log sum_j exp z_j,   q_j = exp(z_j - lse),   w = the row's weight
//   token_logprob   lp = z_a - lse                       dx_j = w / temperature * ([j = a] - q_j)   (w: d loss / d lp)
//   policy_loss     r = exp(lp - old), gap = ref - lp
//                   loss = w (kl (exp(gap) - gap - 1) - min(r A, clip(r, 1 - lo, 1 + hi) A))
//                   d loss / d lp = w (kl (1 - exp(gap)) - A r [r A is the minimum]), dx as above
//   distill_loss    p = softmax over the row's teacher entries / temperature
//                   loss = w sum_k p_k (log p_k - log q_{i_k}),   dx_j = w / temperature * (q_j - sum_{i_k = j} p_k)
//
// A row whose weight is 0, whose token id lies outside [0, cols), or whose teacher entries are all outside is out: its
// loss is 0 and its gradient row 0 whatever its operands hold.  token_logprob needs no weight.
//
// One CTA per row: maximum, sum of exponentials, then the gradient, three passes over the row of which the later two
// find it in L2.
#include "device_math.cuh"
#include "kernel_registry.h"

namespace cinn_b200 {
namespace {

enum Kind { kLogprob = 0, kPolicy = 1, kDistill = 2 };

__device__ __forceinline__ long long load_index(const void* p, long long i, int wide) {
  return wide ? __ldg(reinterpret_cast<const long long*>(p) + i) : (long long)__ldg(reinterpret_cast<const int*>(p) + i);
}
__device__ __forceinline__ float load_float(const void* p, long long i, int type) {
  if (type == 0) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (type == 1) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

struct Policy {
  float lo, hi, kl;  // clip bounds of the ratio (1 - clip_low, 1 + clip_high), weight of the KL term
};
// The policy loss of one token (without its weight) and its derivative with respect to the log-probability.
__device__ __forceinline__ void policy_terms(float lp, float old, float ref, float adv, const Policy& c, float* loss,
                                             float* slope) {
  const float r = expf(lp - old), free = r * adv, held = fminf(fmaxf(r, c.lo), c.hi) * adv;
  *loss  = -fminf(free, held);
  *slope = free <= held ? -free : 0.0f;
  if (r != r || adv != adv) *loss = *slope = r * adv;  // fminf drops a NaN
  if (c.kl != 0.0f) {
    const float gap = ref - lp, e = expm1f(gap);  // expm1: gap is near 0 while the policy is near the reference
    *loss += c.kl * (e - gap);
    *slope -= c.kl * e;
  }
}

template <typename T, int KIND>
__global__ void __launch_bounds__(256)
    k_row_loss(const T* __restrict__ x, const void* __restrict__ ids, const void* __restrict__ a0,
               const float* __restrict__ a1, const float* __restrict__ a2, const float* __restrict__ weight,
               float* __restrict__ out_loss, float* __restrict__ out_lp, T* __restrict__ out_grad, long long rows,
               long long cols, long long entries, long long wide, long long teacher, double weight_value,
               double temperature, double clip_low, double clip_high, double kl_coef) {
  grid_dependency_sync();
  __shared__ float scratch[32];
  const float inv_t = (float)(1.0 / temperature);
  const Policy pol  = {(float)(1.0 - clip_low), (float)(1.0 + clip_high), (float)kl_coef};
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr   = x + row * cols;
    const float w = weight ? weight[row] : (float)weight_value;
    const bool weighted = KIND != kLogprob || out_grad != nullptr;
    bool live     = weighted && w != 0.0f;
    bool need     = live;
    long long a   = 0;
    float tmax = -INFINITY, tsum = 0.0f;
    if (KIND != kDistill) {
      a               = load_index(ids, row, (int)wide);
      const bool good = a >= 0 && a < cols;
      live            = live && good;
      need            = live || (out_lp && good);
    } else {
      for (long long k = 0; k < entries; ++k) {
        const long long i = load_index(ids, row * entries + k, (int)wide);
        if (i >= 0 && i < cols) tmax = fmaxf(tmax, load_float(a0, row * entries + k, (int)teacher) * inv_t);
      }
      live = need = live && tmax > -INFINITY;
      for (long long k = 0; k < entries && live; ++k) {
        const long long i = load_index(ids, row * entries + k, (int)wide);
        if (i >= 0 && i < cols) tsum += expf(load_float(a0, row * entries + k, (int)teacher) * inv_t - tmax);
      }
    }
    float m = -INFINITY, s = 0.0f;
    if (need) {
      for (long long j = threadIdx.x; j < cols; j += blockDim.x) m = fmaxf(m, Io<T>::load1(xr + j) * inv_t);
      m = cta_allreduce<MaxOp>(m, scratch);
      for (long long j = threadIdx.x; j < cols; j += blockDim.x) s += expf(Io<T>::load1(xr + j) * inv_t - m);
      s = cta_allreduce<SumOp>(s, scratch);
    }
    const float ls = logf(s);
    float slope = 0.0f, loss = 0.0f;  // slope: d loss / d z_a, or the weight of the softmax for the distillation
    if (KIND != kDistill) {
      const float lp = need ? Io<T>::load1(xr + a) * inv_t - m - ls : 0.0f;
      if (out_lp && threadIdx.x == 0) out_lp[row] = lp;
      if (KIND == kLogprob) {
        slope = w;
      } else if (live) {
        policy_terms(lp, static_cast<const float*>(a0)[row], pol.kl != 0.0f ? a1[row] : 0.0f, a2[row], pol, &loss, &slope);
        slope *= w;
      }
    } else if (live) {
      const float lt = logf(tsum);
      for (long long k = threadIdx.x; k < entries; k += blockDim.x) {
        const long long i = load_index(ids, row * entries + k, (int)wide);
        if (i < 0 || i >= cols) continue;
        const float lp = load_float(a0, row * entries + k, (int)teacher) * inv_t - tmax - lt, p = expf(lp);
        if (p > 0.0f) loss += p * (lp - (Io<T>::load1(xr + i) * inv_t - m - ls));
      }
      loss  = cta_allreduce<SumOp>(loss, scratch);
      slope = w;
    }
    if (out_loss && threadIdx.x == 0) out_loss[row] = live ? w * loss : 0.0f;
    if (!out_grad) continue;
    T* gr = out_grad + row * cols;
    const float inv_s = 1.0f / s, c = slope * inv_t;
    for (long long j = threadIdx.x; j < cols; j += blockDim.x) {
      float v = 0.0f;
      if (live) {
        const float q = expf(Io<T>::load1(xr + j) * inv_t - m) * inv_s;
        v             = KIND == kDistill ? c * q : c * ((j == a ? 1.0f : 0.0f) - q);
      }
      Io<T>::store1(gr + j, v);
    }
    if (KIND == kDistill && live) {
      __syncthreads();  // the entries below are stored over what another thread stored above
      const float it = 1.0f / tsum;
      for (long long k = threadIdx.x; k < entries; k += blockDim.x) {
        const long long i = load_index(ids, row * entries + k, (int)wide);
        if (i < 0 || i >= cols) continue;
        float p = 0.0f;  // every entry of a column adds up the column in the same order: equal values are stored
        for (long long n = 0; n < entries; ++n)
          if (load_index(ids, row * entries + n, (int)wide) == i) p += expf(load_float(a0, row * entries + n, (int)teacher) * inv_t - tmax) * it;
        Io<T>::store1(gr + i, c * (expf(Io<T>::load1(xr + i) * inv_t - m) * inv_s - p));
      }
    }
  }
}

}  // namespace

#define REG_ROW_LOSS(TNAME, T)                                                                        \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_logprob_" TNAME, 19, 256, k_row_loss<T, kLogprob>);         \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_policy_" TNAME, 19, 256, k_row_loss<T, kPolicy>);           \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_distill_" TNAME, 19, 256, k_row_loss<T, kDistill>)
REG_ROW_LOSS("f32", float);
REG_ROW_LOSS("f16", __half);
REG_ROW_LOSS("bf16", __nv_bfloat16);

}  // namespace cinn_b200
