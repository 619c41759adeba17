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
// A row whose weight is 0, whose token id lies outside [0, cols), or whose teacher entries are all outside or -infinity is
// out: its loss is 0 and its gradient row 0 whatever its operands hold (in the first two cases it is not read).
// token_logprob needs no weight.
//
// What bounds it: HBM.  A logit is read once and its gradient written once, 2 to 8 bytes for about ten instructions,
// one or two of them exponentials (at 16 bits those alone take three quarters of the special-function units' rate).
// Layout: a row belongs to one CTA, or to a cluster of C CTAs when there are few rows.  A CTA has W warps that compute
// and one whose first lane brings the row's 16-byte vectors through a ring of N shared-memory slots (four vectors per
// computing thread each) with bulk asynchronous copies.  Pass 1 keeps a running maximum (over whole chunks the warp's) and a
// sum per lane; the warps' (maximum, sum) pairs meet once, in shared memory or in distributed shared memory across the
// cluster.  Pass 2 turns the row into its gradient: first the last chunks, which are still in the ring, then the others,
// which come through the ring again from L2, the last one first.  Copies that will be wanted again ask L2 to keep them
// (evict_last), the others let go (evict_first).  CTAs are not persistent: the hardware deals rows to SMs as they come free,
// which rows that are out make uneven, and co-resident CTAs cover one another's ends.
//
// Measured on 4096 x 131072 bf16 logits back to back at the power cap, of the measured copy bandwidth: the log-probability
// alone 0.91 to 0.97 (GPUs differ), with the gradient 0.82 to 0.85.  Variants of the latter, single launches on one GPU, 0.90
// as built there: without the L2 hints half of pass 2's reads miss L2, 0.76.  4 slots of 8 warps against 3 / 6 slots: level
// on long rows, 0.64 against 0.64 / 0.55 at 1000 x 50021 fp16; 16 warps 0.78, 4 warps 0.80.  Pass 2 without the chunks that
// are still there 0.825.  The row held on chip by a cluster of 2 or 4 CTAs: 0.68; rings in clusters of 2 / 4: 0.80 / 0.74.
// Persistent CTAs that fetch the next row ahead, rows dealt statically or by cluster launch control: 0.75, 0.77.  Plain loads
// into registers: 0.81.
//
// Every wait on a copy is bounded: a warp that gives up records it (cinn_b200_device_status) and goes on through the
// barriers it shares with others; the copying lane waits for all its copies, bounded, before it leaves.
#include "device_math.cuh"
#include "kernel_registry.h"
#include "pair_math.cuh"
#include "tma_utils.cuh"

namespace cinn_b200 {

CINN_B200_DEFINE_ASYNC_TIMEOUT_COUNTER(g_row_loss_wait_timeouts);

namespace {

enum Kind { kLogprob = 0, kPolicy = 1, kDistill = 2 };
constexpr int kMaxWarps = 8;
constexpr int kUnroll   = 4;   // 16-byte vectors per thread of a ring slot

__device__ __forceinline__ long long load_index(const void* p, long long i, int wide) {
  return wide ? __ldg(reinterpret_cast<const long long*>(p) + i) : (long long)__ldg(reinterpret_cast<const int*>(p) + i);
}
__device__ __forceinline__ float load_float(const void* p, long long i, int type) {
  if (type == 0) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (type == 1) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
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

// A sum of 2^((x - m) c) known by the largest x, m, and its value s.  m is -infinity while nothing but -infinity has
// been seen.
struct Sum {
  float m, s;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Sum warp_join(Sum v, float c) {
  const float m = warp_max(v.m);
  v.s           = v.s * ex2((v.m - finite_ref(m)) * c);
  return {m, warp_allreduce<SumOp>(v.s)};
}

// The sum a lane keeps while it walks a row: two pairs of partial sums of 2^((x + nm) c), nm = -(its largest x).
struct Walk {
  float m, nm;
  F2 s0, s1;
};
// NV vectors into the sum.  The reference is the maximum itself, moved as soon as it is exceeded: a token that the model
// is sure of then has 2^0 = 1 exactly in a sum little above 1, and its log-probability, near 0, keeps its digits.  (Moved
// only when exceeded by 2^24, the logarithm was the small difference of two numbers near 24, 2e-6 off.)
// WARP: all lanes are here and take the warp's maximum, which moves seldom (128 x 131072 bf16 forward 10.7 us, 10.9 with a
// maximum per lane, 10.4 with the reference left behind); otherwise a lane its own.
template <typename T, int NV, bool WARP>
__device__ __forceinline__ void walk(const uint4 (&u)[NV], float c, Walk& k) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
  const float top   = WARP ? warp_max(words_max<T, 4 * NV>(w)) : words_max<T, 4 * NV>(w);
  if (top > k.m) {
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
// The policy loss of one token (without its weight) and its derivative with respect to the log-probability.  In float32: old
// and ref come as float32 log-probabilities, off by half a step each, which moves ratio and gap as much as lp's own
// rounding does; wider arithmetic behind them would add no digits.
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
// Asks for [from, to) in L2.  A hint: nothing is read, so it need not wait for the kernel before this one, which may still
// be writing there.
__device__ __forceinline__ void hint_l2(const void* from, const void* to) {
  const uintptr_t a = (reinterpret_cast<uintptr_t>(from) + 15) & ~(uintptr_t)15, b = reinterpret_cast<uintptr_t>(to) & ~(uintptr_t)15;
  if (b > a) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"((uint32_t)(b - a)) : "memory");
}
__device__ __forceinline__ unsigned sm_count() {
  unsigned n;
  asm("mov.u32 %0, %%nsmid;" : "=r"(n));
  return n;
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

// The operands of a call, as the kernels get them.
template <typename T>
struct Call {
  const T* x;
  const void *ids, *a0;
  const float *a1, *a2, *weight;
  float *out_loss, *out_lp;
  T* out_grad;
  int cols, entries, wide, teacher;
  float weight_value;
  float inv_t, c;  // 1 / temperature; the exponentials are 2^(c (x - largest x))
  Policy policy;
};
#define ROW_LOSS_PARAMS                                                                                                  \
  const T *__restrict__ x, const void *__restrict__ ids, const void *__restrict__ a0, const float *__restrict__ a1,       \
      const float *__restrict__ a2, const float *__restrict__ weight, float *__restrict__ out_loss,                       \
      float *__restrict__ out_lp, T *__restrict__ out_grad, long long rows, long long cols, long long entries,            \
      long long wide, long long teacher, double weight_value, double inv_t, double c, double clip_low, double clip_high,   \
      double kl_coef
#define ROW_LOSS_CALL                                                                                                    \
  {x, ids, a0, a1, a2, weight, out_loss, out_lp, out_grad, (int)cols, (int)entries, (int)wide, (int)teacher,              \
   (float)weight_value, (float)inv_t, (float)c, {(float)clip_low, (float)clip_high, (float)kl_coef}}

// What a row's scalar operands say.
struct Head {
  float w;
  int a;      // the token's column, -1 outside
  bool live;  // whether the row counts
  bool need;  // whether it is read
};
template <typename T, int KIND, bool GRAD>
__device__ __forceinline__ Head head_of(const Call<T>& o, long long row) {
  Head h;
  h.w                = o.weight ? __ldg(o.weight + row) : o.weight_value;
  const long long id = KIND == kDistill ? 0 : load_index(o.ids, row, o.wide);
  h.a                = id >= 0 && id < o.cols ? (int)id : -1;
  h.live             = (GRAD || KIND != kLogprob) && h.w != 0.0f && h.a >= 0;
  h.need             = h.live || (KIND != kDistill && o.out_lp && h.a >= 0);
  return h;
}
struct PolicyOperands {
  float old, ref, adv;
};
template <typename T, int KIND>
__device__ __forceinline__ PolicyOperands policy_operands(const Call<T>& o, long long row) {
  if (KIND != kPolicy) return {0.0f, 0.0f, 0.0f};
  return {__ldg(static_cast<const float*>(o.a0) + row), o.policy.kl != 0.0f ? __ldg(o.a1 + row) : 0.0f, __ldg(o.a2 + row)};
}

// A row's teacher entries in shared memory, four arrays of `padded` values: their columns (-1: unused, -2: behind the last
// one), their logits, the student's logits there, and (before the columns are stored) what all entries of a column have
// together, over 2^(c (the largest)).
struct Kept {
  int* id;
  float *t, *x, *mass;
  int padded;
};
__device__ __forceinline__ Kept kept_at(void* p, int entries) {
  const int n = (entries + 3) & ~3;
  float* f    = static_cast<float*>(p);
  return {static_cast<int*>(p), f + n, f + 2 * n, f + 3 * n, n};
}
template <typename T>
__device__ __forceinline__ void keep_entries(const Call<T>& o, long long row, const Kept& k, int thread, int threads) {
  for (int n = thread; n < k.padded; n += threads) {
    if (n >= o.entries) {
      k.id[n] = -2;
      continue;
    }
    const long long i = load_index(o.ids, row * o.entries + n, o.wide);
    const float t     = load_float(o.a0, row * o.entries + n, o.teacher);
    const bool good   = i >= 0 && i < o.cols;
    k.id[n]           = good ? (int)i : -1;
    k.t[n]            = good ? t : -INFINITY;
    k.x[n]            = good ? Io<T>::load1(o.x + row * o.cols + i) : 0.0f;
  }
}
// The same with one entry per thread, fetched early: its column and logit when the row begins, the student's logit there
// (which needs the column) while the row is being read, stored once the row has been.
struct EarlyEntry {
  long long id;
  float t, x;
};
template <typename T>
__device__ __forceinline__ EarlyEntry fetch_entry(const Call<T>& o, long long row, int thread) {
  if (thread >= o.entries) return {-2, 0.0f, 0.0f};
  const long long at = row * o.entries + thread;
  return {load_index(o.ids, at, o.wide), load_float(o.a0, at, o.teacher), 0.0f};
}
template <typename T>
__device__ __forceinline__ void fetch_student(const Call<T>& o, const T* xr, int thread, EarlyEntry& e) {
  const bool good = e.id >= 0 && e.id < o.cols;
  if (good) e.x = Io<T>::load1(xr + e.id);
  else if (thread < o.entries) e.id = -1, e.t = -INFINITY;
}
__device__ __forceinline__ void keep_entry(const Kept& k, int thread, const EarlyEntry& e) {
  if (thread >= k.padded) return;
  k.id[thread] = (int)e.id;
  k.t[thread]  = e.t;
  k.x[thread]  = e.x;
}
template <typename T>
__device__ __forceinline__ void prefetch_entries(const Call<T>& o, long long row, int thread, int threads) {
  const int wi = o.wide ? 8 : 4, wt = o.teacher ? 2 : 4;
  const char* p0 = static_cast<const char*>(o.ids) + row * o.entries * wi;
  const char* p1 = static_cast<const char*>(o.a0) + row * o.entries * wt;
  for (int b = thread * 128; b < o.entries * wi; b += threads * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p0 + b));
  for (int b = thread * 128; b < o.entries * wt; b += threads * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p1 + b));
}

// What follows from a row's sum: q_j = 2^(c (x_j + nm)) / S, the gradient's common part coef * q_j.  The divisions are few, one
// or two to a thread and row, and rounded ones: the approximate one took the error of a float32 gradient, 777 x 50021,
// from 4.2e-8 to 5e-8 (2-norm, a maximum-subtracted softmax in float32 2.7e-8), at the same times.
struct Terms {
  float nm, S, slope, coef, tmax, tsum;
  bool live;
};
// Loss and log-probability are written by the lane for which `writes` holds (of the warp for which `sums` does, for the
// distillation, whose sum over the entries a whole warp takes).
template <typename T, int KIND>
__device__ __forceinline__ Terms row_terms(const Call<T>& o, long long row, const Head& h, const Sum& t, float xa,
                                           const PolicyOperands& po, const Kept& kept, bool writes, bool sums, int lane) {
  Terms k        = {-finite_ref(t.m), t.s, h.w, 0.0f, -INFINITY, 0.0f, h.live};
  const float lg = logf(t.s);
  auto logq      = [&](float v) { return fmaf(v + k.nm, o.inv_t, -lg); };
  float loss     = 0.0f;
  if (KIND != kDistill) {
    const float lp = logq(xa);
    if (KIND == kPolicy && h.live) {
      policy_terms(lp, po.old, po.ref, po.adv, o.policy, &loss, &k.slope);
      k.slope *= h.w;
    }
    if (writes) {
      if (o.out_lp) o.out_lp[row] = lp;
      if (o.out_loss) o.out_loss[row] = h.live ? h.w * loss : 0.0f;
    }
    k.coef = -k.slope * o.inv_t;
    return k;
  }
  bool nan = false;  // the maxima pass over it
  for (int n = lane; n < o.entries; n += 32) {
    const float v = kept.t[n];
    k.tmax        = fmaxf(k.tmax, v);
    nan |= v != v;
  }
  k.tmax = warp_max(k.tmax);
  k.live = __any_sync(0xffffffffu, nan) || k.tmax > -INFINITY;  // otherwise the teacher keeps nothing, and the row is out
  for (int n = lane; n < o.entries && k.live; n += 32) k.tsum += ex2((kept.t[n] - k.tmax) * o.c);
  k.tsum = warp_allreduce<SumOp>(k.tsum);
  if (o.out_loss && sums) {
    const float lt = logf(k.tsum);
    for (int n = lane; n < o.entries && k.live; n += 32) {
      const float d = kept.t[n] - k.tmax, p = ex2(d * o.c) / k.tsum;
      if (p != 0.0f) loss += p * (fmaf(d, o.inv_t, -lt) - logq(kept.x[n]));
    }
    loss = warp_allreduce<SumOp>(loss);
    if (lane == 0) o.out_loss[row] = k.live ? h.w * loss : 0.0f;
  }
  k.coef = k.slope * o.inv_t;
  return k;
}
// Every entry adds up its whole column, in the same order: entries of one column get the same value.  A column that no
// other entry has (four are compared at a time) is its own sum.
__device__ __forceinline__ void column_masses(const Kept& kept, int entries, const Terms& k, float c, int thread, int threads) {
  for (int n = thread; n < entries; n += threads) {
    const int id = kept.id[n];
    int same     = 0;
    for (int i = 0; i < kept.padded; i += 4) {
      const int4 v = *reinterpret_cast<const int4*>(kept.id + i);
      same += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
    }
    float mass = ex2((kept.t[n] - k.tmax) * c);
    if (same > 1 && id >= 0) {
      mass = 0.0f;
      for (int i = 0; i < entries; ++i)
        if (kept.id[i] == id) mass += ex2((kept.t[i] - k.tmax) * c);
    }
    kept.mass[n] = mass;
  }
}
// The columns that have a term of their own, stored again by the warp that stored their vectors (`mine`).
template <typename T, int KIND, class Mine>
__device__ __forceinline__ void special_columns(const Call<T>& o, T* gr, const Terms& k, const Head& h, float xa,
                                                const Kept& kept, int lane, Mine mine) {
  if (KIND != kDistill) {
    // 1 - q as (S - e) / S: a difference of near numbers is exact.
    if (k.live && lane == 0 && mine(h.a)) Io<T>::store1(gr + h.a, k.slope * o.inv_t * ((k.S - ex2((xa + k.nm) * o.c)) / k.S));
  } else if (k.live) {
    const float it = 1.0f / k.tsum;
    for (int n = lane; n < o.entries; n += 32) {
      const int id = kept.id[n];
      if (id >= 0 && mine(id)) Io<T>::store1(gr + id, k.coef * (ex2((kept.x[n] + k.nm) * o.c) / k.S - kept.mass[n] * it));
    }
  }
}
// A vector of the gradient at `p`, which may not be aligned as the logits are.
template <typename T>
__device__ __forceinline__ void put(char* p, uint4 u) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    st_stream16(p, u);
    return;
  }
  const uint32_t t[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(T); ++j) {
    T one;
    if constexpr (sizeof(T) == 4) one = __uint_as_float(t[j]);
    else reinterpret_cast<unsigned short&>(one) = (unsigned short)(t[j / 2] >> (16 * (j & 1)));
    reinterpret_cast<T*>(p)[j] = one;
  }
}
// The element in front of or behind a row's vectors that a lane of its first warp holds, -1 if none.
__device__ __forceinline__ int edge_of(const Row& r, int cols, bool first_warp, int lane) {
  if (!first_warp) return -1;
  return lane < r.head ? lane : lane >= 8 && lane - 8 < r.tail ? cols - r.tail + lane - 8 : -1;
}
__device__ __forceinline__ Walk start_walk(float xe, float c) {
  Walk k;
  k.m  = xe == xe ? xe : -INFINITY;
  k.nm = -finite_ref(k.m);
  k.s0 = pair(ex2((xe + k.nm) * c), 0.0f);
  k.s1 = pair(0.0f, 0.0f);
  return k;
}
__device__ __forceinline__ Sum end_walk(const Walk& k, float c) {
  float lo, hi;
  unpair(add2(k.s0, k.s1), lo, hi);
  return warp_join({k.m, lo + hi}, c);
}
__device__ __forceinline__ Sum join_all(const float2* meet, int n, int lane, float c) {
  Sum u = {-INFINITY, 0.0f};
  for (int i = lane; i < n; i += 32) {
    const float2 v = meet[i];
    const float hi = fmaxf(u.m, v.x), hf = finite_ref(hi);
    u.s = u.s * ex2((u.m - hf) * c) + v.y * ex2((v.x - hf) * c);
    u.m = hi;
  }
  return warp_join(u, c);
}
// The barrier of one row's threads (numbers that the compiler knows: a number at run time reserves all sixteen).
__device__ __forceinline__ void barrier_of(int group, int threads) {
  switch (group) {
    case 0: asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); break;
    case 1: asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory"); break;
    case 2: asm volatile("bar.sync 3, %0;" ::"r"(threads) : "memory"); break;
    default: asm volatile("bar.sync 4, %0;" ::"r"(threads) : "memory"); break;
  }
}

template <typename T, int KIND, bool GRAD>
__global__ void __launch_bounds__(kMaxWarps * 32 + 32, 3) k_row_loss(ROW_LOSS_PARAMS, long long slots_ll) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  const Call<T> o = ROW_LOSS_CALL;
  const int N = (int)slots_ll, W = (blockDim.x >> 5) - 1, T32 = W * 32, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int C, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int G = C * W, g = rank * W + warp, slot_bytes = T32 * kUnroll * 16;
  const long long row = blockIdx.x / C;
  const Kept kept = kept_at(smem + (size_t)N * slot_bytes, o.entries);
  uint64_t* full  = reinterpret_cast<uint64_t*>(kept.mass + kept.padded);
  uint64_t* empty = full + N;
  uint64_t* met   = empty + N;                           // completes when the pairs of all G warps are here
  float2* meet    = reinterpret_cast<float2*>(met + 1);  // [G]
  const T* xr     = x + row * cols;
  const Row r     = row_at(x, row, o.cols, rank, C);
  const int chunk = T32 * kUnroll;  // vectors of a slot
  const bool producer = warp == W;
  // While the kernel before this one ends: barriers, and the first wave's rows into L2 (1000 x 50021 fp16 with the gradient
  // 41 -> 39 us back to back).
  if (producer && lane == 0) {
    for (int s = 0; s < N; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], W);
    }
    mbar_init(met, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (C > 1) mbar_arrive_expect_tx(met, (uint32_t)G * 8u);
    const char* p = r.body + (size_t)r.start * 16;
    if (blockIdx.x < 3 * sm_count()) hint_l2(p, p + (size_t)min(r.count, N * chunk) * 16);
  }
  grid_dependency_sync();
  const Head h    = head_of<T, KIND, GRAD>(o, row);
  const int edge  = edge_of(r, o.cols, g == 0, lane);
  T* gr           = GRAD ? out_grad + row * cols : nullptr;
  char* body      = GRAD ? reinterpret_cast<char*>(gr + r.head) + (size_t)r.start * 16 : nullptr;
  if (!h.need) {  // the same for every warp of the row: no barrier is left waiting
    if (g == 0 && lane == 0) {
      if (out_loss) out_loss[row] = 0.0f;
      if (out_lp) out_lp[row] = 0.0f;
    }
    if (GRAD) {
      for (int v = tid; v < r.count; v += blockDim.x) put<T>(body + (size_t)v * 16, make_uint4(0, 0, 0, 0));
      if (edge >= 0) Io<T>::store1(gr + edge, 0.0f);
    }
    return;
  }

  const int chunks = (r.count + chunk - 1) / chunk;
  const int held   = GRAD ? min(chunks, N) : 0;              // pass 2 finds the last ones still in the ring
  const int total  = GRAD ? 2 * chunks - held : chunks;      // and has the others fetched again, last one first
  auto copy = [&](int i, int s) {
    const int at         = (i < chunks ? i : total - 1 - i) * chunk;
    const uint32_t bytes = (uint32_t)min(r.count - at, chunk) * 16u;
    mbar_arrive_expect_tx(&full[s], bytes);
    bulk_load_hint(smem + (size_t)s * slot_bytes, r.body + (size_t)(r.start + at) * 16, bytes, &full[s],
                   i < total - chunks ? l2_keep() : l2_pass());
  };
  if (producer && lane == 0)
    for (int i = 0; i < min(N, total); ++i) copy(i, i);
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
  float xe = -INFINITY, xa = 0.0f;
  if (edge >= 0) xe = Io<T>::load1(xr + edge);
  if (KIND != kDistill) xa = Io<T>::load1(xr + h.a);
  const PolicyOperands po = policy_operands<T, KIND>(o, row);
  EarlyEntry entry = {-2, 0.0f, 0.0f};
  if (KIND == kDistill) {
    if (o.entries <= T32) {
      entry = fetch_entry(o, row, tid);
      fetch_student(o, xr, tid, entry);
    } else {
      prefetch_entries(o, row, tid, T32);  // they are fetched after pass 1
    }
  }

  // Pass 1.
  Walk k   = start_walk(xe, o.c);
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
      walk<T, kUnroll, true>(u, o.c, k);
    } else {
      for (int j = tid; j < left; j += T32) {
        const uint4 u[1] = {src[j - tid]};
        walk<T, 1, false>(u, o.c, k);
      }
    }
    if (i < chunks - held) leave(slot);
    next_slot();
  }
  Sum t = end_walk(k, o.c);
  if (KIND == kDistill) {  // for every warp of this CTA
    if (o.entries <= T32) keep_entry(kept, tid, entry);
    else keep_entries(o, row, kept, tid, T32);
  }
  if (G > 1) {
    if (C == 1) {
      if (lane == 0) meet[warp] = make_float2(t.m, t.s);
      barrier_of(0, T32);
    } else {
      if (lane < C) {
        uint32_t there, bar;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_addr(meet + g)), "r"(lane));
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_addr(met)), "r"(lane));
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(there), "l"(pair(t.m, t.s)), "r"(bar)
                     : "memory");
      }
      __syncwarp();
      if (KIND == kDistill) barrier_of(0, T32);  // the entries above
      if (!dead && !mbar_wait_bounded(met, 0)) dead = true;
    }
    t = join_all(meet, G, lane, o.c);
  } else {
    __syncwarp();
  }
  const Terms m = row_terms<T, KIND>(o, row, h, t, xa, po, kept, g == 0 && lane == 0, g == G - 1, lane);

  if (GRAD) {
    if (KIND == kDistill) column_masses(kept, o.entries, m, o.c, tid, T32);
    // Pass 2: coef * q_j everywhere, then the few columns that have a term of their own.
    const float q0 = m.coef / m.S;
    int there      = (chunks - held) % N;  // slot of the first chunk that is still there
    for (int i = 0; i < chunks; ++i) {
      const int at = (i < held ? chunks - held + i : chunks - 1 - i) * chunk, left = r.count - at;
      int s        = there;
      if (i < held) {
        there = there + 1 == N ? 0 : there + 1;
      } else {
        wait();
        s = slot;
        next_slot();
      }
      const uint4* src = reinterpret_cast<const uint4*>(smem + (size_t)s * slot_bytes) + tid;
      char* dst        = body + (size_t)(at + tid) * 16;
      if (!m.live) {
        for (int j = tid; j < min(left, chunk); j += T32) put<T>(dst + (size_t)(j - tid) * 16, make_uint4(0, 0, 0, 0));
        leave(s);
      } else if (left >= chunk) {
        uint4 u[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) u[j] = src[j * T32];
        leave(s);
        common_part<T, kUnroll>(u, m.nm, o.c, q0);
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) put<T>(dst + (size_t)j * T32 * 16, u[j]);
      } else {
        for (int j = tid; j < left; j += T32) {
          uint4 u[1] = {src[j - tid]};
          common_part<T, 1>(u, m.nm, o.c, q0);
          put<T>(dst + (size_t)(j - tid) * 16, u[0]);
        }
        leave(s);
      }
    }
    if (edge >= 0) Io<T>::store1(gr + edge, m.live ? ex2((xe + m.nm) * o.c) * q0 : 0.0f);
    __syncwarp();  // the vectors before what is stored over them
    if (KIND == kDistill) barrier_of(0, T32);  // the masses
    special_columns<T, KIND>(o, gr, m, h, xa, kept, lane, [&](int i) {
      const int e = i - r.head;
      if (e < 0 || e >= r.nvec * V) return g == 0;
      const int at = e / V - r.start;
      return at >= 0 && at < r.count && (at & (T32 - 1)) / 32 == warp;
    });
  }
  if (__any_sync(0xffffffffu, dead) && lane == 0) atomicAdd(&g_row_loss_wait_timeouts, 1u);
  if (C > 1) cluster_barrier();  // no CTA leaves while another may still write to its shared memory
}

// Rows of at most 16 KiB, in registers: W = 2^shift warps per row (1, 2 or 4), 8 / W rows per CTA, up to NV vectors per thread, all
// of them loaded at once.  A row's warps meet at a barrier of their own.
template <typename T, int KIND, bool GRAD, int NV>
__global__ void __launch_bounds__(256, NV == 8 ? 2 : 4) k_row_loss_short(ROW_LOSS_PARAMS, long long shift_ll) {
  if (threadIdx.x == 0 && blockIdx.x < 4 * sm_count()) {  // the first wave's rows into L2 while the kernel before this one ends
    const long long first = (long long)blockIdx.x * (8 >> (int)shift_ll);
    hint_l2(x + first * cols, x + min(rows, first + (8 >> (int)shift_ll)) * cols);
  }
  grid_dependency_sync();
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float2 meet[8];
  const Call<T> o = ROW_LOSS_CALL;
  const int W = 1 << (int)shift_ll, T32 = 32 * W, group = threadIdx.x >> (5 + (int)shift_ll), tid = threadIdx.x - group * T32, lane = tid & 31, warp = tid >> 5;
  const long long row = (long long)blockIdx.x * (8 >> (int)shift_ll) + group;
  if (row >= rows) return;
  const Kept kept = kept_at(smem + group * ((o.entries + 3) & ~3) * 16, o.entries);
  const T* xr     = x + row * cols;
  const Head h    = head_of<T, KIND, GRAD>(o, row);
  const Row r     = row_at(x, row, o.cols, 0, 1);
  const int edge  = edge_of(r, o.cols, warp == 0, lane);
  T* gr           = GRAD ? out_grad + row * cols : nullptr;
  char* body      = GRAD ? reinterpret_cast<char*>(gr + r.head) : nullptr;
  if (!h.need) {
    if (tid == 0) {
      if (out_loss) out_loss[row] = 0.0f;
      if (out_lp) out_lp[row] = 0.0f;
    }
    if (GRAD) {
      for (int v = tid; v < r.nvec; v += T32) put<T>(body + (size_t)v * 16, make_uint4(0, 0, 0, 0));
      if (edge >= 0) Io<T>::store1(gr + edge, 0.0f);
    }
    return;
  }
  EarlyEntry entry = {-2, 0.0f, 0.0f};
  if (KIND == kDistill && o.entries <= T32) entry = fetch_entry(o, row, tid);
  uint4 u[NV];
  const uint4* src = reinterpret_cast<const uint4*>(r.body) + tid;
#pragma unroll
  for (int j = 0; j < NV; ++j) u[j] = tid + j * T32 < r.nvec ? ld_stream16(src + j * T32) : minus_infinity<T>();
  float xe = -INFINITY, xa = 0.0f;
  if (edge >= 0) xe = Io<T>::load1(xr + edge);
  if (KIND != kDistill) xa = Io<T>::load1(xr + h.a);
  const PolicyOperands po = policy_operands<T, KIND>(o, row);
  if (KIND == kDistill) {
    if (o.entries <= T32) fetch_student(o, xr, tid, entry);
    else keep_entries(o, row, kept, tid, T32);
  }
  Walk k = start_walk(xe, o.c);
  if constexpr (NV == 8) {
    walk<T, 4, false>(reinterpret_cast<const uint4(&)[4]>(u[0]), o.c, k);
    walk<T, 4, false>(reinterpret_cast<const uint4(&)[4]>(u[4]), o.c, k);
  } else {
    walk<T, NV, false>(u, o.c, k);
  }
  Sum t = end_walk(k, o.c);
  if (KIND == kDistill && o.entries <= T32) keep_entry(kept, tid, entry);
  if (W > 1) {
    if (lane == 0) meet[group * W + warp] = make_float2(t.m, t.s);
    barrier_of(group, T32);
    t = join_all(meet + group * W, W, lane, o.c);
  } else {
    __syncwarp();
  }
  const Terms m = row_terms<T, KIND>(o, row, h, t, xa, po, kept, tid == 0, warp == W - 1, lane);
  if (!GRAD) return;
  if (KIND == kDistill) column_masses(kept, o.entries, m, o.c, tid, T32);
  const float q0 = m.coef / m.S;
  if (m.live) {
    common_part<T, NV>(u, m.nm, o.c, q0);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) u[j] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (tid + j * T32 < r.nvec) put<T>(body + (size_t)(tid + j * T32) * 16, u[j]);
  if (edge >= 0) Io<T>::store1(gr + edge, m.live ? ex2((xe + m.nm) * o.c) * q0 : 0.0f);
  __syncwarp();  // the vectors before what is stored over them
  if (KIND == kDistill && W > 1) barrier_of(group, T32);  // the masses
  special_columns<T, KIND>(o, gr, m, h, xa, kept, lane, [&](int i) {
    const int e = i - r.head;
    return e < 0 || e >= r.nvec * V ? warp == 0 : ((e / V) & (T32 - 1)) / 32 == warp;
  });
}

}  // namespace

#define REG_ROW_LOSS(KNAME, KIND, GNAME, GRAD, TNAME, T)                                                                      \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_" KNAME GNAME "_" TNAME, 21, kMaxWarps * 32 + 32, k_row_loss<T, KIND, GRAD>);         \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_" KNAME GNAME "_" TNAME "_n2", 21, 256, k_row_loss_short<T, KIND, GRAD, 2>);          \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_" KNAME GNAME "_" TNAME "_n4", 21, 256, k_row_loss_short<T, KIND, GRAD, 4>);          \
  CINN_B200_REGISTER_KERNEL_PDL("row_loss_" KNAME GNAME "_" TNAME "_n8", 21, 256, k_row_loss_short<T, KIND, GRAD, 8>)
#define REG_ROW_LOSS_KINDS(TNAME, T)                           \
  REG_ROW_LOSS("logprob", kLogprob, "", false, TNAME, T);      \
  REG_ROW_LOSS("logprob", kLogprob, "_grad", true, TNAME, T);  \
  REG_ROW_LOSS("policy", kPolicy, "", false, TNAME, T);        \
  REG_ROW_LOSS("policy", kPolicy, "_grad", true, TNAME, T);    \
  REG_ROW_LOSS("distill", kDistill, "", false, TNAME, T);      \
  REG_ROW_LOSS("distill", kDistill, "_grad", true, TNAME, T)
REG_ROW_LOSS_KINDS("f32", float);
REG_ROW_LOSS_KINDS("f16", __half);
REG_ROW_LOSS_KINDS("bf16", __nv_bfloat16);

}  // namespace cinn_b200
