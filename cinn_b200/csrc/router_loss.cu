// A router's balance loss, its gradient and the per-expert counts.  x is [tokens, experts], w the tokens' weights,
// c the number of tokens that chose each expert, f = c / sum c; per token q = softmax(x):
//
//   loss = E sum_e f_e sum_t w_t q_te        dx_te = w_t E q_te (f_e - sum_e' f_e' q_te')
//
// The gradient needs the counts alone, so it and the column sums of w q share one pass over the logits: the row of a
// token in the registers of L lanes (L <= 32 lanes, NV vectors of V elements each), the column sums in the same lanes'
// registers over all tokens of the warp, one partial row per CTA (expert_load), and a small kernel that folds the
// partial rows and the counts into the loss (balance_fold).  No floating-point atomics: results do not depend on the
// order of CTAs.  A token of weight 0 is out: it adds nothing and is not read, and its gradient row is 0.
#include <type_traits>
#include "device_math.cuh"
#include "kernel_registry.h"

namespace cinn_b200 {
namespace {

constexpr int kRouterThreads = 512;
constexpr int kMaxExperts    = 1024;

// V elements at p, as floats: one vector, or one element.
template <typename T, int V>
struct Raw {
  typedef typename std::conditional<V == 1, T, uint4>::type type;
};
template <typename T, int V>
__device__ __forceinline__ void widen(const typename Raw<T, V>::type& r, float* f) {
  if constexpr (V == 1) f[0] = Io<T>::load1(&r);
  else Io<T>::unpack(r, f);
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(kRouterThreads)
    k_router_loss(const T* __restrict__ x, const float* __restrict__ weight, const int* __restrict__ counts,
                  float* __restrict__ out_load, T* __restrict__ out_grad, long long rows, long long cols_ll,
                  double weight_value, long long lanes_ll) {
  grid_dependency_sync();
  typedef typename Raw<T, V>::type R;
  constexpr int K = V * NV;  // elements per lane
  extern __shared__ float part[];  // [warps][cols]
  __shared__ float scratch[32];
  const int cols = (int)cols_ll, L = (int)lanes_ll, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  const int per_warp = 32 / L, sub = lane & (L - 1), group = lane / L;
  const int nvec     = cols / V;
  float f[K], acc[K];
#pragma unroll
  for (int i = 0; i < K; ++i) f[i] = acc[i] = 0.0f;
  if (out_grad) {
    // Shares of the choices, less their mean: sum_e q_e = 1, so a constant taken off f changes nothing in
    // f_e - sum f q but its cancellation.
    float total = 0.0f;
    for (int e = threadIdx.x; e < cols; e += blockDim.x) total += (float)counts[e];
    total = cta_allreduce<SumOp>(total, scratch);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int v = sub + (i / V) * L;
      if (v < nvec && total > 0.0f) f[i] = (float)counts[v * V + i % V] / total - 1.0f / (float)cols;
    }
  }
  auto weight_of = [&](long long t) { return t < rows ? (weight ? __ldg(weight + t) : (float)weight_value) : 0.0f; };
  auto load      = [&](long long t, bool on, R (&r)[NV]) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int v = sub + n * L;
      if (on && v < nvec) {
        if constexpr (V == 1) r[n] = x[t * cols + v];
        else r[n] = ld_stream16(x + t * cols + (long long)v * V);
      }
    }
  };
  // Tokens of this lane's group; the weights are fetched two tokens ahead, the logits one.
  const long long step = (long long)gridDim.x * W * per_warp;
  long long t = ((long long)blockIdx.x * W + warp) * per_warp + group;
  float w = weight_of(t), w1 = weight_of(t + step);
  R r[NV], r1[NV];
  load(t, w != 0.0f, r);
  for (long long base = t - group; base < rows; base += step, t += step) {  // the same trips for all lanes of a warp
    const float w2 = weight_of(t + 2 * step);
    load(t + step, w1 != 0.0f, r1);
    float q[K], m = -INFINITY, s = 0.0f, inner = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const bool on = w != 0.0f && sub + n * L < nvec;
      widen<T, V>(r[n], q + n * V);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!on) q[n * V + j] = -INFINITY;
        m = fmaxf(m, q[n * V + j]);
      }
    }
    for (int o = L >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base_m = w != 0.0f ? m : 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      float e;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((q[i] - base_m) * 1.4426950408889634f));
      q[i] = e;
      s += e;
    }
#pragma unroll
    for (int i = 0; i < K; ++i) inner = fmaf(q[i], f[i], inner);
    for (int o = L >> 1; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      inner += __shfl_xor_sync(0xffffffffu, inner, o);
    }
    const float inv = 1.0f / s, wq = w != 0.0f ? w * inv : 0.0f;
    inner *= inv;
    const float factor = (float)cols * wq;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int v = sub + n * L;
      float d[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = n * V + j;
        if (w != 0.0f) acc[i] = fmaf(wq, q[i], acc[i]);
        d[j] = w != 0.0f ? factor * q[i] * (f[i] - inner) : 0.0f;
      }
      if (out_grad && t < rows && v < nvec) {
        if constexpr (V == 1) Io<T>::store1(out_grad + t * cols + v, d[0]);
        else st_stream16(out_grad + t * cols + (long long)v * V, Io<T>::pack(d));
      }
    }
    w  = w1;
    w1 = w2;
#pragma unroll
    for (int n = 0; n < NV; ++n) r[n] = r1[n];
  }
  if (!out_load) return;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    for (int o = L; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);  // the warp's groups
    const int v = sub + (i / V) * L;
    if (group == 0 && v < nvec) part[warp * cols + v * V + i % V] = acc[i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < cols; e += blockDim.x) {
    float v = 0.0f;
    for (int k = 0; k < W; ++k) v += part[k * cols + e];
    out_load[(long long)blockIdx.x * cols + e] = v;
  }
}

// Counts of the choices in shared memory, a thread per token (whole numbers: the order of the additions does not show).
// One CTA writes the result; several add to one that k_expert_zero has cleared.
__global__ void __launch_bounds__(1024)
    k_expert_counts(const void* __restrict__ index, const float* __restrict__ weight, int* __restrict__ counts,
                    long long rows, long long slots, long long experts, long long wide, double weight_value) {
  grid_dependency_sync();
  __shared__ int bins[kMaxExperts];
  for (int e = threadIdx.x; e < experts; e += blockDim.x) bins[e] = 0;
  __syncthreads();
  for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < rows; t += (long long)gridDim.x * blockDim.x) {
    if ((weight ? __ldg(weight + t) : (float)weight_value) == 0.0f) continue;
#pragma unroll 4
    for (long long i = t * slots; i < (t + 1) * slots; ++i) {
      const long long e = wide ? __ldg(reinterpret_cast<const long long*>(index) + i) : (long long)__ldg(reinterpret_cast<const int*>(index) + i);
      if (e >= 0 && e < experts) atomicAdd(&bins[e], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    if (gridDim.x == 1) counts[e] = bins[e];
    else if (bins[e]) atomicAdd(counts + e, bins[e]);
  }
}
__global__ void __launch_bounds__(1024) k_expert_zero(int* __restrict__ counts, long long experts) {
  grid_dependency_sync();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[e] = 0;
}

// All warps of the cluster, each of them together.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// loss = E / sum c * sum over slices and experts of c_e load_ke: one flat dot product, over the CTAs of one cluster.
__global__ void __launch_bounds__(1024)
    k_balance_fold(const float* __restrict__ load, const int* __restrict__ counts, float* __restrict__ out,
                   long long slices, long long experts) {
  grid_dependency_sync();
  __shared__ float scratch[32];
  __shared__ float meet[8];
  int C, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  // A thread keeps to one column, or to four neighbouring ones, and walks down every `down`-th slice.
  const int E = (int)experts, K = (int)slices, tid = threadIdx.x;
  const bool four = E % 4 == 0 && (reinterpret_cast<uintptr_t>(load) & 15) == 0;
  const int across = four ? E / 4 : E, down = blockDim.x / across * C, col = tid % across;
  const int first = tid / across < blockDim.x / across ? tid / across * C + rank : K;
  float total = 0.0f, sum = 0.0f;
  for (int e = tid; e < E; e += blockDim.x) total += (float)counts[e];
  if (four) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int k = first; k < K; k += down) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(load) + (long long)k * across + col);
      v[0] += u.x;
      v[1] += u.y;
      v[2] += u.z;
      v[3] += u.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fmaf((float)counts[4 * col + j], v[j], sum);
  } else {
    float v = 0.0f;
#pragma unroll 8
    for (int k = first; k < K; k += down) v += __ldg(load + (long long)k * E + col);
    sum = (float)counts[col] * v;
  }
  total = cta_allreduce<SumOp>(total, scratch);
  sum = cta_allreduce<SumOp>(sum, scratch);
  if (C > 1) {
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(meet + rank)));
    cluster_barrier();  // no CTA writes to the first one's shared memory before that one runs
    if (threadIdx.x == 0) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(sum) : "memory");
    cluster_barrier();
    sum = 0.0f;
    if (rank == 0)
      for (int k = 0; k < C; ++k) sum += meet[k];
  }
  if (rank == 0 && threadIdx.x == 0) out[0] = total > 0.0f ? (float)experts * (sum / total) : 0.0f;
}

}  // namespace

#define REG_ROUTER(TNAME, T, VN, V, NV) \
  CINN_B200_REGISTER_KERNEL_PDL("router_loss_" TNAME VN "_n" #NV, 9, kRouterThreads, k_router_loss<T, V, NV>)
#define REG_ROUTER_TYPE(TNAME, T, V)   \
  REG_ROUTER(TNAME, T, "_s", 1, 1);    \
  REG_ROUTER(TNAME, T, "_s", 1, 2);    \
  REG_ROUTER(TNAME, T, "_s", 1, 4);    \
  REG_ROUTER(TNAME, T, "_s", 1, 8);    \
  REG_ROUTER(TNAME, T, "_s", 1, 16);   \
  REG_ROUTER(TNAME, T, "_s", 1, 32);   \
  REG_ROUTER(TNAME, T, "_v", V, 1);    \
  REG_ROUTER(TNAME, T, "_v", V, 2);    \
  REG_ROUTER(TNAME, T, "_v", V, 4)
REG_ROUTER_TYPE("f32", float, 4);
REG_ROUTER("f32", float, "_v", 4, 8);
REG_ROUTER_TYPE("f16", __half, 8);
REG_ROUTER_TYPE("bf16", __nv_bfloat16, 8);
CINN_B200_REGISTER_KERNEL_PDL("expert_counts", 8, 1024, k_expert_counts);
CINN_B200_REGISTER_KERNEL_PDL("expert_zero", 2, 1024, k_expert_zero);
CINN_B200_REGISTER_KERNEL_PDL("balance_fold", 5, 1024, k_balance_fold);

}  // namespace cinn_b200
