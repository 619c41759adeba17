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
// loss is 0 and its gradient row 0 whatever its operands hold, and it is not read.  token_logprob needs no weight.
//
// What bounds it: HBM.  A logit is read once and its gradient written once, 2 to 8 bytes for about ten instructions,
// one or two of them exponentials (at 16 bits those alone take three quarters of the special-function units' rate).
// Layout: a row belongs to one CTA, or to a cluster of C CTAs when there are few rows.  A CTA has W warps that compute
// and one whose first lane brings the row's 16-byte vectors through a ring of N shared-memory slots (four vectors per
// computing thread each) with bulk asynchronous copies.  Pass 1 keeps a running reference and sum per lane; the warps'
// (reference, sum) pairs meet once, in shared memory or in distributed shared memory across the cluster.  Pass 2 turns
// the row into its gradient: first the last chunks, which are still in the ring, then the others, which come through
// the ring again from L2, the last one first.  Copies that will be wanted again ask L2 to keep them (evict_last), the
// others let go (evict_first).  CTAs are not persistent: the hardware deals rows to SMs as they come free, which rows
// that are out make uneven, and co-resident CTAs cover one another's ends.
//
// Measured on 4096 x 131072 bf16 logits, single launches / back to back at the power cap, of the measured copy bandwidth:
// the log-probability alone 0.97 / 0.92, with its gradient 0.90 / 0.84.  Without the L2 hints half of pass 2's reads miss L2:
// 0.76.  4 slots of 8 warps against 3 / 6 slots: level on long rows, 0.64 against 0.64 / 0.55 at 1000 x 50021 fp16; 16 warps
// 0.78, 4 warps 0.80.  Pass 2 without the chunks that are still there 0.825.  The row held on chip by a cluster of 2 or 4
// CTAs: 0.68; rings in clusters of 2 / 4: 0.80 / 0.74.  Persistent CTAs that fetch the next row ahead, rows dealt statically
// or by cluster launch control: 0.75, 0.77.  Plain loads into registers: 0.81.
//
// Every wait on a copy is bounded: a warp that gives up records it (cinn_b200_device_status) and goes on through the
// barriers it shares with others; the copying lane waits for all its copies, bounded, before it leaves.
#include "device_math.cuh"
#include "kernel_registry.h"
#include "tma_utils.cuh"

namespace cinn_b200 {

CINN_B200_DEFINE_ASYNC_TIMEOUT_COUNTER(g_row_loss_wait_timeouts);

namespace {

enum Kind { kLogprob = 0, kPolicy = 1, kDistill = 2 };
constexpr int kMaxWarps = 16;
constexpr int kUnroll   = 4;   // 16-byte vectors per thread of a ring slot

__device__ __forceinline__ long long load_index(const void* p, long long i, int wide) {
  return wide ? __ldg(reinterpret_cast<const long long*>(p) + i) : (long long)__ldg(reinterpret_cast<const int*>(p) + i);
}
__device__ __forceinline__ float load_float(const void* p, long long i, int type) {
  if (type == 0) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (type == 1) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Pairs of floats in one 64-bit register, for the two-wide arithmetic of sm_100.
typedef unsigned long long F2;
__device__ __forceinline__ F2 pair(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(F2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The largest element of N words of packed elements, as float (a NaN is passed over: the sum of exponentials keeps it).
template <typename T, int N>
__device__ __forceinline__ float words_max(const uint32_t* w) {
  if constexpr (sizeof(T) == 4) {
    float m = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, __uint_as_float(w[i]));
    return m;
  } else {
    typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
    const T2* t = reinterpret_cast<const T2*>(w);
    T2 m        = t[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = __hmax2(m, t[i]);
    return fmaxf(__low2float(m), __high2float(m));
  }
}
// Elements 2 i and 2 i + 1 of packed words.
template <typename T>
__device__ __forceinline__ F2 elements(const uint32_t* w, int i) {
  float lo, hi;
  if constexpr (sizeof(T) == 4) return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else if constexpr (std::is_same<T, __half>::value) unpack_h2(w[i], lo, hi);
  else unpack_bf2(w[i], lo, hi);
  return pair(lo, hi);
}
// A vector of -infinity.
template <typename T>
__device__ __forceinline__ uint4 minus_infinity() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// A sum of 2^((x - m) c) known by its reference m and its value s.  The reference is any value not far below the
// largest x: -infinity while nothing but -infinity has been seen.
struct Sum {
  float m, s;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Sum warp_join(Sum v, float c) {
  const float m = warp_max(v.m);
  v.s           = v.s * ex2((v.m - finite_ref(m)) * c);
  return {m, warp_allreduce<SumOp>(v.s)};
}

// The sum a lane keeps while it walks a row: two pairs of partial sums of 2^((x + nm) c), nm = -(its reference).
struct Walk {
  float m, nm;
  F2 s0, s1;
};
// NV vectors into the sum.  The reference moves only when their maximum exceeds it by a factor of 2^24, which the
// partial sums bear; the first vectors that are not all -infinity set it.
template <typename T, int NV>
__device__ __forceinline__ void walk(const uint4 (&u)[NV], float c, float margin, Walk& k) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
  const float top   = words_max<T, 4 * NV>(w);
  if (top > k.m + margin) {
    const float f = ex2((k.m - top) * c);
    k.s0          = mul2(k.s0, pair(f, f));
    k.s1          = mul2(k.s1, pair(f, f));
    k.m           = top;
    k.nm          = -finite_ref(top);
  }
  const F2 c2 = pair(c, c), nm2 = pair(k.nm, k.nm);
  constexpr int kPairs = NV * 8 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < kPairs; i += 2) {
    float a0, a1, b0, b1;
    unpair(mul2(add2(elements<T>(w, i), nm2), c2), a0, a1);
    unpair(mul2(add2(elements<T>(w, i + 1), nm2), c2), b0, b1);
    k.s0 = add2(k.s0, pair(ex2(a0), ex2(a1)));
    k.s1 = add2(k.s1, pair(ex2(b0), ex2(b1)));
  }
}
// NV vectors of logits into as many of the gradient's common part, q0 2^((x + nm) c).
template <typename T, int NV>
__device__ __forceinline__ void common_part(uint4 (&u)[NV], float nm, float c, float q0) {
  constexpr int V = 16 / sizeof(T);
  const F2 c2 = pair(c, c), q2 = pair(q0, q0), nm2 = pair(nm, nm);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
    float f[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float a0, a1;
      unpair(mul2(add2(elements<T>(w, i), nm2), c2), a0, a1);
      unpair(mul2(pair(ex2(a0), ex2(a1)), q2), f[2 * i], f[2 * i + 1]);
    }
    u[v] = Io<T>::pack(f);
  }
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
  if (free != free) *loss = *slope = free;  // fminf drops a NaN
  if (c.kl != 0.0f) {
    const float gap = ref - lp, e = expm1f(gap);  // expm1: gap is near 0 while the policy is near the reference
    *loss += c.kl * (e - gap);
    *slope -= c.kl * e;
  }
}

// How long L2 should keep what a copy brings: past other data, when the row comes through a second time, or not at all.
__device__ __forceinline__ uint64_t l2_keep() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t l2_pass() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void bulk_load_hint(void* smem_dst, const void* gmem_src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
                   smem_addr(smem_dst)),
               "l"(gmem_src), "r"(bytes), "r"(smem_addr(bar)), "l"(policy)
               : "memory");
}
// All warps of the cluster, each of them together.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Where a row's vectors lie: `head` elements in front of the first 16-byte boundary, `nvec` vectors, `tail` elements;
// and this CTA's stretch of the vectors, `count` from `start` on (`per` to a CTA).
struct Row {
  const char* body;
  int head, tail, nvec, per, start, count;
};
template <typename T>
__device__ __forceinline__ Row row_at(const T* x, long long row, int cols, int rank, int C) {
  constexpr int V = 16 / sizeof(T);
  const T* p      = x + row * cols;
  const int skew  = (int)(reinterpret_cast<uintptr_t>(p) & 15) / (int)sizeof(T);
  Row r;
  r.head  = min(skew ? V - skew : 0, cols);
  r.nvec  = (cols - r.head) / V;
  r.tail  = cols - r.head - r.nvec * V;
  r.per   = (((r.nvec + C - 1) >> (31 - __clz(C))) + 31) & ~31;  // C is a power of two
  r.start = min(rank * r.per, r.nvec);
  r.count = min(r.per, r.nvec - r.start);
  r.body  = reinterpret_cast<const char*>(p + r.head);
  return r;
}

template <typename T, int KIND, bool GRAD>
__global__ void __launch_bounds__(kMaxWarps * 32 + 32, 1)
    k_row_loss(const T* __restrict__ x, const void* __restrict__ ids, const void* __restrict__ a0,
               const float* __restrict__ a1, const float* __restrict__ a2, const float* __restrict__ weight,
               float* __restrict__ out_loss, float* __restrict__ out_lp, T* __restrict__ out_grad, long long rows,
               long long cols_ll, long long entries_ll, long long wide_ll, long long teacher_ll, double weight_value,
               double temperature, double clip_low, double clip_high, double kl_coef, long long slots_ll) {
  grid_dependency_sync();
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  const int cols = (int)cols_ll, entries = (int)entries_ll, wide = (int)wide_ll, teacher = (int)teacher_ll;
  const int N = (int)slots_ll, W = (blockDim.x >> 5) - 1, T32 = W * 32, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int C, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int G = C * W, g = rank * W + warp, slot_bytes = T32 * kUnroll * 16;
  const long long row = blockIdx.x / C;
  uint64_t* full  = reinterpret_cast<uint64_t*>(smem + (size_t)N * slot_bytes);
  uint64_t* empty = full + N;
  uint64_t* met   = empty + N;                             // completes when the pairs of all G warps are here
  float2* meet    = reinterpret_cast<float2*>(met + 1);    // [G]
  int* kept_id    = reinterpret_cast<int*>(meet + G);      // [entries], the distillation's
  float* kept_t   = reinterpret_cast<float*>(kept_id + entries);
  float* kept_x   = kept_t + entries;
  const float c   = (float)(1.4426950408889634 / temperature);
  const T* xr     = x + row * cols;

  const float w  = weight ? __ldg(weight + row) : (float)weight_value;
  long long id   = KIND == kDistill ? 0 : load_index(ids, row, wide);
  const int a    = id >= 0 && id < cols ? (int)id : -1;
  bool live      = (GRAD || KIND != kLogprob) && w != 0.0f && a >= 0;  // whether the row counts
  const bool need = live || (KIND != kDistill && out_lp && a >= 0);    // whether it is read
  const Row r    = row_at(x, row, cols, rank, C);
  // The element in front of or behind the vectors that this lane holds, if any (first warp of the row).
  const int edge = g == 0 && lane < r.head ? lane : g == 0 && lane >= 8 && lane - 8 < r.tail ? cols - r.tail + lane - 8 : -1;

  T* gr      = GRAD ? out_grad + row * cols : nullptr;
  char* body = GRAD ? reinterpret_cast<char*>(gr + r.head) + (size_t)r.start * 16 : nullptr;
  auto put   = [&](int v, uint4 u) {  // a vector of the gradient
    if ((reinterpret_cast<uintptr_t>(body) & 15) == 0) {
      st_stream16(body + (size_t)v * 16, u);
    } else {  // the gradient is not aligned as the logits are
      const uint32_t t[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < V; ++j) {
        T one;
        if constexpr (sizeof(T) == 4) one = __uint_as_float(t[j]);
        else reinterpret_cast<unsigned short&>(one) = (unsigned short)(t[j / 2] >> (16 * (j & 1)));
        reinterpret_cast<T*>(body)[v * V + j] = one;
      }
    }
  };
  if (!need) {  // the same for every warp of the row: no barrier is left waiting
    if (g == 0 && lane == 0) {
      if (out_loss) out_loss[row] = 0.0f;
      if (out_lp) out_lp[row] = 0.0f;
    }
    if (GRAD) {
      for (int v = tid; v < r.count; v += blockDim.x) put(v, make_uint4(0, 0, 0, 0));
      if (edge >= 0) Io<T>::store1(gr + edge, 0.0f);
    }
    return;
  }

  const int chunk  = T32 * kUnroll;                               // vectors of a slot
  const int chunks = (r.count + chunk - 1) / chunk;
  const int held   = GRAD ? min(chunks, N) : 0;                   // pass 2 finds the last ones still in the ring
  const int total  = GRAD ? 2 * chunks - held : chunks;           // and has the others fetched again, last one first
  const bool producer = warp == W;
  auto copy = [&](int i, int s) {
    const int at         = (i < chunks ? i : total - 1 - i) * chunk;
    const uint32_t bytes = (uint32_t)min(r.count - at, chunk) * 16u;
    mbar_arrive_expect_tx(&full[s], bytes);
    bulk_load_hint(smem + (size_t)s * slot_bytes, r.body + (size_t)(r.start + at) * 16, bytes, &full[s],
                   i < total - chunks ? l2_keep() : l2_pass());
  };
  if (producer && lane == 0) {
    for (int s = 0; s < N; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], W);
    }
    mbar_init(met, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (C > 1) mbar_arrive_expect_tx(met, (uint32_t)G * 8u);
    for (int i = 0; i < min(N, total); ++i) copy(i, i);
  }
  __syncwarp();
  __syncthreads();
  if (C > 1) cluster_barrier();  // no CTA writes to another's shared memory before that one runs
  if (producer) {
    bool ok  = true;  // (the warp stays together: the barriers of a cluster are passed by warps, not by lanes)
    int made = min(N, total);
    for (int i = made, s = 0, n = 0; i < total && ok; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], n & 1));
      if (ok) {
        if (lane == 0) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the slot's readers before its refill
          copy(i, s);
        }
        __syncwarp();
        ++made;
      }
      if (++s == N) s = 0, ++n;
    }
    // Every copy lands before the warp that issued it leaves.
    for (int i = max(0, made - N); i < made; ++i) ok = mbar_wait_bounded(&full[i % N], (i / N) & 1) && ok;
    if (!__all_sync(0xffffffffu, ok) && lane == 0) atomicAdd(&g_row_loss_wait_timeouts, 1u);
    if (C > 1) cluster_barrier();
    return;
  }
  float xe = -INFINITY, xa = 0.0f, old = 0.0f, ref = 0.0f, adv = 0.0f;
  if (edge >= 0) xe = Io<T>::load1(xr + edge);
  if (KIND != kDistill) xa = Io<T>::load1(xr + a);
  if (KIND == kPolicy) {
    old = __ldg(static_cast<const float*>(a0) + row);
    ref = kl_coef != 0.0 ? __ldg(a1 + row) : 0.0f;
    adv = __ldg(a2 + row);
  }
  if (KIND == kDistill) {  // the teacher's entries into L2; they are wanted after pass 1
    const char* p0 = static_cast<const char*>(ids) + row * entries * (wide ? 8 : 4);
    const char* p1 = static_cast<const char*>(a0) + row * entries * (teacher ? 2 : 4);
    for (int b = tid * 128; b < entries * (wide ? 8 : 4); b += T32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p0 + b));
    for (int b = tid * 128; b < entries * (teacher ? 2 : 4); b += T32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p1 + b));
  }

  // Pass 1.
  Walk k;
  k.m  = xe == xe ? xe : -INFINITY;
  k.nm = -finite_ref(k.m);
  k.s0 = pair(ex2((xe + k.nm) * c), 0.0f);
  k.s1 = pair(0.0f, 0.0f);
  const float margin = 24.0f / c;
  int slot = 0;  // next slot to read, and the parity of its phase
  uint32_t phase = 0;
  bool dead = false;
  auto wait = [&]() {
    if (!dead && !mbar_wait_bounded(&full[slot], phase)) dead = true;
  };
  auto leave = [&](int s) {  // the warp has read its part of slot s
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&empty[s])) : "memory");
  };
  auto next_slot = [&]() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1;
    }
  };
  for (int i = 0; i < chunks; ++i) {
    const int left = r.count - i * chunk;
    wait();
    const uint4* src = reinterpret_cast<const uint4*>(smem + (size_t)slot * slot_bytes) + tid;
    if (left >= chunk) {
      uint4 u[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) u[j] = src[j * T32];
      walk<T, kUnroll>(u, c, margin, k);
    } else {
      for (int j = tid; j < left; j += T32) {
        const uint4 u[1] = {src[j - tid]};
        walk<T, 1>(u, c, margin, k);
      }
    }
    if (i < chunks - held) leave(slot);
    next_slot();
  }
  float p0, p1;
  unpair(add2(k.s0, k.s1), p0, p1);
  Sum t = warp_join({k.m, p0 + p1}, c);
  if (KIND == kDistill) {  // the entries and the student's logits at them, for every warp of this CTA
    for (int n = tid; n < entries; n += T32) {
      const long long i = load_index(ids, row * entries + n, wide);
      const float tn    = load_float(a0, row * entries + n, teacher);
      const bool good   = i >= 0 && i < cols;
      kept_id[n]        = good ? (int)i : -1;
      kept_t[n]         = good ? tn : -INFINITY;
      kept_x[n]         = good ? Io<T>::load1(xr + i) : 0.0f;
    }
  }
  if (G > 1) {
    if (C == 1) {
      if (lane == 0) meet[warp] = make_float2(t.m, t.s);
      asm volatile("bar.sync 1, %0;" ::"r"(T32) : "memory");
    } else {
      if (lane < C) {
        uint32_t there, bar;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_addr(meet + g)), "r"(lane));
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_addr(met)), "r"(lane));
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(there), "l"(pair(t.m, t.s)), "r"(bar)
                     : "memory");
      }
      __syncwarp();
      if (KIND == kDistill) asm volatile("bar.sync 1, %0;" ::"r"(T32) : "memory");  // the entries above
      if (!dead && !mbar_wait_bounded(met, 0)) dead = true;
    }
    Sum u = {-INFINITY, 0.0f};
    for (int n = lane; n < G; n += 32) {
      const float2 o = meet[n];
      const float hi = fmaxf(u.m, o.x), hf = finite_ref(hi);
      u.s = u.s * ex2((u.m - hf) * c) + o.y * ex2((o.x - hf) * c);
      u.m = hi;
    }
    t = warp_join(u, c);
  } else {
    __syncwarp();
  }
  const float nM = -finite_ref(t.m), S = t.s, lg = log2f(S), inv_t = (float)(1.0 / temperature);
  auto logq = [&](float v) { return ((v + nM) * c - lg) * 0.6931471805599453f; };

  float slope = w, loss = 0.0f;  // slope: d loss / d lp, or the factor of the softmax for the distillation
  float tmax = -INFINITY, tsum = 0.0f;
  if (KIND != kDistill) {
    const float lp = logq(xa);
    if (KIND == kPolicy && live) {
      const Policy pol = {(float)(1.0 - clip_low), (float)(1.0 + clip_high), (float)kl_coef};
      policy_terms(lp, old, ref, adv, pol, &loss, &slope);
      slope *= w;
    }
    if (g == 0 && lane == 0) {
      if (out_lp) out_lp[row] = lp;
      if (out_loss) out_loss[row] = live ? w * loss : 0.0f;
    }
  } else {
    for (int n = lane; n < entries; n += 32) tmax = fmaxf(tmax, kept_t[n]);
    tmax = warp_max(tmax);
    live = tmax > -INFINITY;  // otherwise the teacher keeps nothing, and the row is out
    for (int n = lane; n < entries && live; n += 32) tsum += ex2((kept_t[n] - tmax) * c);
    tsum = warp_allreduce<SumOp>(tsum);
    if (out_loss && g == G - 1) {  // one warp of the row
      const float lt = log2f(tsum);
      for (int n = lane; n < entries && live; n += 32) {
        const float lp2 = (kept_t[n] - tmax) * c - lt, p = ex2(lp2);
        if (p > 0.0f) loss += p * (lp2 * 0.6931471805599453f - logq(kept_x[n]));
      }
      loss = warp_allreduce<SumOp>(loss);
      if (lane == 0) out_loss[row] = live ? w * loss : 0.0f;
    }
  }

  if (GRAD) {
    // Pass 2: factor * 2^((x - M) c) / S everywhere, then the few columns that have a term of their own.
    const float coef = KIND == kDistill ? slope * inv_t : -slope * inv_t, q0 = coef / S;
    int kept = (chunks - held) % N;  // slot of the first chunk that is still there
    for (int i = 0; i < chunks; ++i) {
      const int at = (i < held ? chunks - held + i : chunks - 1 - i) * chunk, left = r.count - at;
      int s        = kept;
      if (i < held) {
        kept = kept + 1 == N ? 0 : kept + 1;
      } else {
        wait();
        s = slot;
        next_slot();
      }
      const uint4* src = reinterpret_cast<const uint4*>(smem + (size_t)s * slot_bytes) + tid;
      if (!live) {
        for (int j = tid; j < min(left, chunk); j += T32) put(at + j, make_uint4(0, 0, 0, 0));
        leave(s);
      } else if (left >= chunk) {
        uint4 u[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) u[j] = src[j * T32];
        leave(s);
        common_part<T, kUnroll>(u, nM, c, q0);
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) put(at + tid + j * T32, u[j]);
      } else {
        for (int j = tid; j < left; j += T32) {
          uint4 u[1] = {src[j - tid]};
          common_part<T, 1>(u, nM, c, q0);
          put(at + j, u[0]);
        }
        leave(s);
      }
    }
    if (edge >= 0) Io<T>::store1(gr + edge, live ? ex2((xe + nM) * c) * q0 : 0.0f);
    // Columns are stored again by the warp that stored them above (ordered by the warp barrier).
    __syncwarp();
    auto mine = [&](int i) {
      const int e = i - r.head;
      if (e < 0 || e >= r.nvec * V) return g == 0;
      const int at = e / V - r.start;
      return at >= 0 && at < r.count && (at % T32) / 32 == warp;
    };
    if (KIND != kDistill) {
      if (live && lane == 0 && mine(a)) Io<T>::store1(gr + a, slope * inv_t * (1.0f - ex2((xa + nM) * c) / S));
    } else if (live) {
      const float it = 1.0f / tsum;
      for (int n0 = 0; n0 < entries; n0 += 32) {
        const int i   = n0 + lane < entries ? kept_id[n0 + lane] : -1;
        unsigned todo = __ballot_sync(0xffffffffu, i >= 0 && mine(i));
        while (todo) {  // one column at a time: the warp adds up all of its entries
          const int n   = __ffs(todo) - 1;
          const int col = __shfl_sync(0xffffffffu, i, n);
          todo &= todo - 1;
          float p = 0.0f;
          for (int n2 = lane; n2 < entries; n2 += 32)
            if (kept_id[n2] == col) p += ex2((kept_t[n2] - tmax) * c);
          p = warp_allreduce<SumOp>(p) * it;
          if (lane == 0) Io<T>::store1(gr + col, coef * (ex2((kept_x[n0 + n] + nM) * c) / S - p));
        }
      }
    }
  }
  if (__any_sync(0xffffffffu, dead) && lane == 0) atomicAdd(&g_row_loss_wait_timeouts, 1u);
  if (C > 1) cluster_barrier();  // no CTA leaves while another may still write to its shared memory
}

}  // namespace

#define REG_ROW_LOSS(KNAME, KIND, TNAME, T)                                                                          \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_" KNAME "_" TNAME, 20, kMaxWarps * 32 + 32, k_row_loss<T, KIND, false>);         \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_" KNAME "_grad_" TNAME, 20, kMaxWarps * 32 + 32, k_row_loss<T, KIND, true>)
#define REG_ROW_LOSS_KINDS(TNAME, T)             \
  REG_ROW_LOSS("logprob", kLogprob, TNAME, T);   \
  REG_ROW_LOSS("policy", kPolicy, TNAME, T);     \
  REG_ROW_LOSS("distill", kDistill, TNAME, T)
REG_ROW_LOSS_KINDS("f32", float);
REG_ROW_LOSS_KINDS("f16", __half);
REG_ROW_LOSS_KINDS("bf16", __nv_bfloat16);

}  // namespace cinn_b200
