// A router's balance loss, its gradient and the per-expert counts.  x is [tokens, experts], w the tokens' weights,
// c the number of tokens that chose each expert, f = c / sum c; per token q = softmax(x):
//
//   loss = E sum_t w_t (sum_e f_e q_te)        dx_te = w_t E q_te (f_e - sum_e' f_e' q_te')
//
// The counts come first (they are a constant of the differentiation); loss and gradient then share one pass over the
// logits, because the sum over the experts that the gradient subtracts is the token's term of the loss: a token's row in
// the registers of L lanes (NV vectors of V elements each), the terms added up per CTA (balance_part) and then over the
// CTAs by an ordinary row reduction.  No floating-point atomics: results do not depend on the order of CTAs.  A token of
// weight 0 is out: it adds nothing and is not read, and its gradient row is 0.
//
// Bound by HBM for long batches and, at these row lengths, by instructions nearly as much: three reductions over a token's
// lanes for eight elements per lane.  Measured with counts, loss and gradient, 65536 x 256 fp32, 8 choices: 29 us (119 MB,
// 0.63 of the copy bandwidth), of which 6 us are the three small launches around this kernel; 480 us before the row lay
// in registers as vectors, 34 with 16 elements per lane, 32 with column sums (which the loss does not need) kept too, 33 with two tokens
// per trip (84 registers: one CTA per SM).
#include <type_traits>
#include "device_math.cuh"
#include "kernel_registry.h"
#include "pair_math.cuh"

namespace cinn_b200 {
namespace {

constexpr int kRouterThreads = 512;
constexpr int kMaxExperts    = 1024;

// What a lane loads at once: a vector of V elements, or one element (V = 1).
template <typename T, int V>
struct Raw {
  typedef typename std::conditional<V == 1, T, uint4>::type type;
  __device__ static __forceinline__ void widen(const type& r, float* f) {
    if constexpr (V == 1) f[0] = Io<T>::load1(&r);
    else Io<T>::unpack(r, f);
  }
  __device__ static __forceinline__ type fill(float v) {
    if constexpr (V == 1) {
      T one;
      Io<T>::store1(&one, v);
      return one;
    } else {
      float f[V];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = v;
      return Io<T>::pack(f);
    }
  }
};

template <typename T, int V, int NV>
__global__ void __launch_bounds__(V * NV > 16 ? kRouterThreads / 2 : kRouterThreads, V > 1 && (V * NV <= 8 || V * NV == 32) ? 2 : 1)
    k_router_loss(const T* __restrict__ x, const float* __restrict__ weight, const int* __restrict__ counts,
                  float* __restrict__ out_part, T* __restrict__ out_grad, long long rows, long long cols_ll,
                  double weight_value, long long lanes_ll) {
  grid_dependency_sync();
  typedef Raw<T, V> Io1;
  typedef typename Io1::type R;
  constexpr int K = V * NV;          // elements per lane, a pair at a time (an odd last one is paired with nothing)
  constexpr int P = (K + 1) / 2;
  __shared__ float scratch[32];
  const int cols = (int)cols_ll, L = (int)lanes_ll, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  const int shift = 31 - __clz(L), per_warp = 32 >> shift, sub = lane & (L - 1), group = lane >> shift;
  const int nvec  = cols / V;
  // Shares of the choices.  In f_e - sum f q a constant may be taken off f, because sum q = 1: less their mean, shares
  // that are nearly alike do not cancel.  The loss is summed without that, and by lanes: its terms are all positive.
  float total = 0.0f, sum = 0.0f;
  for (int e = threadIdx.x; e < cols; e += blockDim.x) total += (float)counts[e];
  total             = cta_allreduce<SumOp>(total, scratch);
  const float scale = total > 0.0f ? 1.0f / total : 0.0f, mean = total > 0.0f ? 1.0f / (float)cols : 0.0f;
  F2 f[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float g[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = 2 * i + j, v = sub + (e / V) * L;
      g[j]        = e < K && v < nvec ? (float)counts[v * V + e % V] * scale : 0.0f;
    }
    f[i] = pair(g[0], g[1]);
  }
  // Tokens of this lane's group; the weights are fetched two tokens ahead, the logits one.  A token that is out is not
  // read: zeros stand for it, and its weight of 0 makes everything it gives 0.
  const long long step = (long long)gridDim.x * W * per_warp, jump = step * cols;
  long long t = ((long long)blockIdx.x * W + warp) * per_warp + group;
  const T* px = x + t * cols + sub * V;
  T* pg       = out_grad ? out_grad + t * cols + sub * V : nullptr;
  auto weight_of = [&](long long t) { return t < rows ? (weight ? __ldg(weight + t) : (float)weight_value) : 0.0f; };
  auto load      = [&](const T* p, bool on, R (&r)[NV]) {
    if (__all_sync(0xffffffffu, on)) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (sub + n * L < nvec) {  // the others stay minus infinity
          if constexpr (V == 1) r[n] = p[n * L];
          else r[n] = ld_stream16(p + n * L * V);
        }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (sub + n * L < nvec) {
          r[n] = Io1::fill(0.0f);
          if (on) {
            if constexpr (V == 1) r[n] = p[n * L];
            else r[n] = ld_stream16(p + n * L * V);
          }
        }
    }
  };
  const F2 log2e    = pair(1.4426950408889634f, 1.4426950408889634f);
  const float fcols = (float)cols;
  const F2 less_mean = pair(-mean, -mean);
  // One token: its row is `r`, its weight `w`.
  auto token = [&](const R (&r)[NV], float w) {
    float y[2 * P], m = -INFINITY;
    y[2 * P - 1] = -INFINITY;
#pragma unroll
    for (int n = 0; n < NV; ++n) Io1::widen(r[n], y + n * V);
#pragma unroll
    for (int i = 0; i < K; ++i) m = fmaxf(m, y[i]);
    if (L == 32) {
      asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(m));
    } else {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
        if (o < L) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (L > 16) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    }
    F2 q[P], s2 = pair(0.0f, 0.0f), dot2 = pair(0.0f, 0.0f), inner2 = pair(0.0f, 0.0f);
    const F2 nm = pair(-m, -m);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float a, b;
      unpair(mul2(add2(pair(y[2 * i], y[2 * i + 1]), nm), log2e), a, b);
      q[i] = pair(ex2(a), ex2(b));
      s2   = add2(s2, q[i]);
      dot2 = fma2(q[i], f[i], dot2);
    }
    float s0, s1, i0, i1, d0, d1;
    unpair(s2, s0, s1);
    unpair(dot2, d0, d1);
    if (!out_grad) {
      s0 += s1;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < L) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      sum = fmaf(w, (d0 + d1) * __fdividef(1.0f, s0), sum);
      return;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) inner2 = fma2(q[i], add2(f[i], less_mean), inner2);
    unpair(inner2, i0, i1);
    F2 both = add2(pair(s0, i0), pair(s1, i1));  // the sum of the exponentials and their product with f, side by side
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (o < L) {
        unpair(both, s0, i0);
        both = add2(both, pair(__shfl_xor_sync(0xffffffffu, s0, o), __shfl_xor_sync(0xffffffffu, i0, o)));
      }
    unpair(both, s0, i0);
    const float inv = __fdividef(1.0f, s0), less_inner = -i0 * inv;
    sum = fmaf(w, (d0 + d1) * inv, sum);
    const float factor = fcols * w * inv;
    const F2 factor2 = pair(factor, factor), less = pair(less_inner, less_inner);
#pragma unroll
    for (int i = 0; i < P; ++i)
      unpair(mul2(mul2(factor2, q[i]), add2(add2(f[i], less_mean), less)), y[2 * i], y[2 * i + 1]);
    if (t < rows) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (sub + n * L < nvec) {
          if constexpr (V == 1) Io<T>::store1(pg + n * L, y[n]);
          else st_stream16(pg + n * L * V, Io<T>::pack(y + n * V));
        }
    }
  };
  float w = weight_of(t), w1 = weight_of(t + step);
  R r[NV], r1[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) r[n] = r1[n] = Io1::fill(-INFINITY);
  load(px, w != 0.0f, r);
  for (long long base = t - group; base < rows; base += step, t += step) {  // the same trips for all lanes of a warp
    const float w2 = weight_of(t + 2 * step);
    px += jump;
    load(px, w1 != 0.0f, r1);
    token(r, w);
    pg += jump;
    w  = w1;
    w1 = w2;
#pragma unroll
    for (int n = 0; n < NV; ++n) r[n] = r1[n];
  }
  if (!out_part) return;
  sum = cta_allreduce<SumOp>(sum, scratch);
  if (threadIdx.x == 0) out_part[blockIdx.x] = (float)cols * sum;
}

// Adds this thread's choices to the CTA's bins, eight read before the first is counted (compared as they come, each load
// waited for the one before: 16384 x 4 choices on 8 CTAs 5.5 us, now 4.2).  Neighbouring threads take neighbouring choices.
// There are fewer than 2^31 choices and at most 2^17 threads: 32 bits hold every position.  Bins per lane, without bank
// conflicts, are no faster (5.1 us).
template <class Index>
__device__ __forceinline__ void count_choices(int* bins, const Index* __restrict__ index, const float* __restrict__ weight,
                                              float weight_value, unsigned n, unsigned slots, unsigned experts) {
  constexpr int kAhead = 8;
  const unsigned step = gridDim.x * blockDim.x, step_t = step / slots, step_s = step - step_t * slots;
  unsigned i = blockIdx.x * blockDim.x + threadIdx.x, t = i / slots, s = i - t * slots;
  while (i < n) {
    Index chosen[kAhead];
    float w[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      chosen[u] = -1;
      w[u]      = weight_value;
      if (i < n) {
        chosen[u] = __ldg(index + i);
        if (weight) w[u] = __ldg(weight + t);
      }
      i += step;
      t += step_t;
      s += step_s;
      if (s >= slots) {
        s -= slots;
        ++t;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (w[u] != 0.0f && chosen[u] >= 0 && chosen[u] < (Index)experts) atomicAdd(&bins[(int)chosen[u]], 1);
  }
}

// Counts of the choices in shared memory (whole numbers: the order of the additions does not show).  The CTAs of one
// cluster add up each other's bins and write the result; the CTAs of a larger grid add theirs to one that k_expert_zero
// has cleared.
__global__ void __launch_bounds__(1024)
    k_expert_counts(const void* __restrict__ index, const float* __restrict__ weight, int* __restrict__ counts,
                    long long choices, long long slots, long long experts, long long wide, double weight_value) {
  grid_dependency_sync();
  __shared__ int bins[kMaxExperts];
  int C, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  for (int e = threadIdx.x; e < experts; e += blockDim.x) bins[e] = 0;
  __syncthreads();
  if (wide) count_choices(bins, static_cast<const long long*>(index), weight, (float)weight_value, choices, slots, experts);
  else count_choices(bins, static_cast<const int*>(index), weight, (float)weight_value, choices, slots, experts);
  __syncthreads();
  if (gridDim.x > C) {
    for (int e = threadIdx.x; e < experts; e += blockDim.x)
      if (bins[e]) atomicAdd(counts + e, bins[e]);
    return;
  }
  if (C > 1) cluster_barrier();  // every CTA's bins are complete
  for (int e = rank * blockDim.x + threadIdx.x; e < experts; e += C * blockDim.x) {
    const unsigned mine = (unsigned)__cvta_generic_to_shared(bins + e);
    int sum             = 0;
    for (int c = 0; c < C; ++c) {
      unsigned there;
      int v;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(mine), "r"(c));
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
      sum += v;
    }
    counts[e] = sum;
  }
  if (C > 1) cluster_barrier();  // no CTA leaves while another reads its bins
}
__global__ void __launch_bounds__(1024) k_expert_zero(int* __restrict__ counts, long long experts) {
  grid_dependency_sync();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[e] = 0;
}

}  // namespace

#define REG_ROUTER(TNAME, T, VN, V, NV) \
  CINN_B200_REGISTER_KERNEL_PDL("router_loss_" TNAME VN "_n" #NV, 9, V * NV > 16 ? kRouterThreads / 2 : kRouterThreads, k_router_loss<T, V, NV>)
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

}  // namespace cinn_b200
