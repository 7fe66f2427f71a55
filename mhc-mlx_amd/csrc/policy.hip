// Clipped policy loss with a KL term, from the logits, and its gradient.
//
//   lp = z_a - log sum_v exp z_v;  r = exp(lp - old);  q = exp(ref - lp)
//   L  = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (q - 1 - log q)
//   c  = dL / dlp = -A r [r A <= clip(r) A] + beta (1 - q)
//   dz_v = w c / D ([v = a] - exp(z_v) / sum)
//
// Bound by memory: the logits have to be read and the gradient written.  A
// workgroup holds a row in registers (up to 128 K 16-bit logits), so that
// loss and gradient together read it once; through autograd the gradient
// needs the upstream scalar and is a second call, which reads the row again.
// Rows of weight 0, and rows whose c is 0 (a clipped token without a KL term),
// are not read for it: their gradient is zeros.  Loss and gradient of 8192 x
// 50257 bf16, a quarter of the rows masked: 338 us, 4.3 TB/s; through autograd
// 1000 x 32768 fp32 27 us for the loss (4.9 TB/s) and 39 for the gradient, which
// finds the logits in the last-level cache.
#include "mhc_device.hpp"
#include "mhc_host.hpp"
#include "mhc_plan.hpp"

namespace mhc {
namespace {

constexpr int kRowThreads = 1024;  // of the kernels for rows of any length
constexpr int kMaxRows = 1 << 20;  // workgroups of a launch; further rows go round again

// A row as vectors of 16 bytes at 16-byte boundaries, with the elements
// before the first and after the last taken one by one (rows of an odd width
// start anywhere).
template <typename T>
struct Row {
  static constexpr int kE = 16 / (int)sizeof(T);
  int head, vecs, tail;
  MHC_DEV Row(const T* p, int V) {
    head = min(V, (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)));
    vecs = (V - head) / kE;
    tail = V - head - vecs * kE;
  }
};

// vector v from p on: a 32-bit offset from an address that the workgroup shares
template <typename T>
MHC_DEV const T* vec_at(const T* p, uint32_t v) { return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + v * 16u); }
template <typename T>
MHC_DEV T* vec_at(T* p, uint32_t v) { return reinterpret_cast<T*>(reinterpret_cast<char*>(p) + v * 16u); }

// sum and largest of what a thread has seen; exponentials are taken below `top`
struct Running {
  float top = -__builtin_inff(), sum = 0.f;
};

// exp(x - top), 0 for x = -inf whatever the top
MHC_DEV float exp_below(float x, float top) {
  return __builtin_amdgcn_exp2f((x - top) * 1.44269504f);
}

// top as it is subtracted: a row part of -inf alone has none, and -inf - -inf would be NaN
MHC_DEV float base_of(float top) { return top == -__builtin_inff() ? 0.f : top; }

template <int E>
MHC_DEV void take(Running& r, const float (&x)[E]) {
  float top = x[0];
#pragma unroll
  for (int k = 1; k < E; ++k) top = fmaxf(top, x[k]);
  if (top > r.top) {
    r.sum *= exp_below(r.top, top);
    r.top = top;
  }
  const float base = base_of(r.top);
#pragma unroll
  for (int k = 0; k < E; ++k) r.sum += exp_below(x[k], base);
}

MHC_DEV void join(Running& r, float top, float sum) {
  const float t = fmaxf(r.top, top), base = base_of(t);
  r.sum = r.sum * exp_below(r.top, base) + sum * exp_below(top, base);
  r.top = t;
}

// one result for a workgroup of THREADS, in every thread, joined in a fixed order
template <int THREADS>
MHC_DEV Running join_workgroup(Running r, float (&lds)[32]) {
  constexpr int kWaves = THREADS / kWave;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) join(r, __shfl_xor(r.top, d), __shfl_xor(r.sum, d));
  if constexpr (kWaves == 1) return r;
  const int wave = threadIdx.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) {
    lds[wave] = r.top;
    lds[16 + wave] = r.sum;
  }
  __syncthreads();
  Running all;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) join(all, lds[w], lds[16 + w]);
  return all;
}

// a sum over a workgroup's threads, in every thread, in a fixed order
template <int THREADS, typename S, int N>
MHC_DEV S sum_workgroup(S s, S (&lds)[N]) {
  static_assert(N >= THREADS / kWave);
  constexpr int kWaves = THREADS / kWave;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  if constexpr (kWaves == 1) return s;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  S all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += lds[w];
  return all;
}

MHC_DEV float weight_of(const mhc_policy_args& a, int64_t t) {
  if (a.weights == nullptr) return 1.f;
  return a.weights_dtype == MHC_DTYPE_U8 ? (static_cast<const uint8_t*>(a.weights)[t] != 0 ? 1.f : 0.f)
                                         : static_cast<const float*>(a.weights)[t];
}

struct Token {
  float loss, logp, coef;  // without the weight
  float logit;
};

// The differences of log probabilities are small beside them, and the mean of
// ratio times advantage is small beside its terms: lp's rounding to fp32 (5e-7
// at -11) would be most of the loss's error.  So lp is put together in fp64,
// from log sum = e log 2 + log m, whose fp32 part, of m around 1, is below 0.35.
template <typename T>
MHC_DEV Token token_of(const mhc_policy_args& a, int64_t t, const T* row, float top, float sum) {
  const int64_t at = a.actions[t];
  const float nan = __builtin_nanf("");
  const float z = at >= 0 && at < a.V ? load1(row + at) : nan;
  int e;
  float m = frexpf(sum, &e);
  if (m < 0.70710678f) m *= 2.f, --e;
  const double lp = (double)z - (double)top - ((double)e * 0.6931471805599453 + (double)logf(m));
  const float ratio = expf((float)(lp - (double)a.old_logp[t])), adv = a.advantages[t];
  // (a NaN ratio stays one: fminf and fmaxf would drop it)
  const float held_ratio = ratio < 1.f - a.clip_low ? 1.f - a.clip_low : ratio > 1.f + a.clip_high ? 1.f + a.clip_high : ratio;
  // (a ratio past fp32's range is still nothing without an advantage, and so is a KL term without a coefficient)
  const float free = adv == 0.f && ratio == __builtin_inff() ? 0.f : ratio * adv, held = held_ratio * adv;
  Token r;
  r.logp = (float)lp;
  r.logit = z;
  r.loss = -(free <= held ? free : held);
  r.coef = free <= held ? -free : 0.f;
  if (!(free == free)) r.loss = r.coef = nan;
  if (a.ref_logp != nullptr && a.kl_coef != 0.f) {
    const float gap = (float)((double)a.ref_logp[t] - lp), over = expm1f(gap);  // q - 1 without cancellation near q = 1
    r.loss += a.kl_coef * (over - gap);
    r.coef -= a.kl_coef * over;
  }
  return r;
}

// D: the caller's, or the sum of the weights (1 if that is 0)
template <int THREADS>
MHC_DEV float denominator_of(const mhc_policy_args& a, float (&lds)[32]) {
  if (a.denominator > 0.f) return a.denominator;
  float d = (float)a.T;
  if (a.weights != nullptr) {
    d = 0.f;
#pragma unroll 8
    for (int64_t t = threadIdx.x; t < a.T; t += THREADS) d += weight_of(a, t);
    d = sum_workgroup<THREADS>(d, lds);
  }
  return d != 0.f ? d : 1.f;
}

// element `k` of those before a row's first vector and after its last
template <typename T>
MHC_DEV int edge_of(const Row<T>& at, int V, int k) { return k < at.head ? k : V - at.tail + (k - at.head); }

// 16 bytes at p; along: p is a multiple of 16
template <typename T>
MHC_DEV void store_vec(T* p, const float (&x)[16 / sizeof(T)], bool along) {
  u32x4 o;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) o[k] = __builtin_bit_cast(uint32_t, x[k]);
    else o[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
  }
  if (along) *reinterpret_cast<u32x4*>(p) = o;
  else __builtin_memcpy(p, &o, 16);
}

template <typename T>
MHC_DEV void zero_row(T* out, int V, int threads) {
  const Row<T> at(out, V);
  for (int v = threadIdx.x; v < at.vecs; v += threads)
    reinterpret_cast<u32x4*>(out + at.head)[v] = u32x4{0, 0, 0, 0};
  if ((int)threadIdx.x < at.head + at.tail) out[edge_of(at, V, threadIdx.x)] = (T)0;
}

// Rows of up to THREADS * NV vectors, held in registers from the sums to the
// gradient (GRAD: stored times `scale` / D; else what the backward reads).  A
// workgroup takes rows in turn, so that those of a CU load, compute and store
// at different times, and sums the weights once.
template <typename T, int THREADS, int NV, bool GRAD>
__global__ __launch_bounds__(THREADS) void policy_held_kernel(const mhc_policy_args a, float* logp, float* stats, float* terms, float scale,
                                                              T* dlogits) {
  using R = Row<T>;
  __shared__ float lds[32];
  const float unit = GRAD ? scale / denominator_of<THREADS>(a, lds) : 1.f;
  const int V = (int)a.V;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const float w = weight_of(a, t);
    if (w == 0.f) {
      if (threadIdx.x == 0) {
        logp[t] = terms[t] = 0.f;
        if constexpr (!GRAD) stats[3 * t] = stats[3 * t + 1] = stats[3 * t + 2] = 0.f;
      }
      if constexpr (GRAD) zero_row(dlogits + t * a.V, V, THREADS);
      continue;
    }
    const T* const row = static_cast<const T*>(a.logits) + t * a.row_stride;
    const R at(row, V);
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (or every vector's place would have a register for all rows)
    Vec<T, R::kE> q[NV] = {};
    if (at.vecs > 0) {  // (threads past the last vector read it once more: a load under a condition waits for itself)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        q[i].template load<GRAD>(vec_at(row + at.head, (uint32_t)min(i * THREADS + tid, at.vecs - 1)));  // (else read again soon)
    }
    const bool on_edge = tid < at.head + at.tail;
    const int edge = on_edge ? edge_of(at, V, tid) : 0;
    float x1[1] = {on_edge ? load1(row + edge) : -__builtin_inff()};
    Running r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * THREADS + tid >= at.vecs) break;
      float x[R::kE];
#pragma unroll
      for (int k = 0; k < R::kE; ++k) x[k] = q[i].get(k);
      take(r, x);
      __builtin_amdgcn_sched_barrier(0);  // one vector after the other, or the unpacked row would need the registers twice
    }
    take(r, x1);
    r = join_workgroup<THREADS>(r, lds);
    const Token k = token_of(a, t, row, r.top, r.sum);
    if (threadIdx.x == 0) {
      logp[t] = k.logp;
      terms[t] = w * k.loss;
      if constexpr (!GRAD) {
        stats[3 * t] = r.top;
        stats[3 * t + 1] = 1.f / r.sum;
        stats[3 * t + 2] = w * k.coef;
      }
    }
    if constexpr (GRAD) {
      T* const out = dlogits + t * a.V;
      const float coef = w * k.coef * unit, each = -coef / r.sum;
      if (w * k.coef == 0.f) {
        zero_row(out, V, THREADS);
        continue;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(q[i].w[j]));  // (or the row would be kept unpacked from the sums on)
      const int action = (int)a.actions[t];
      const bool along = ((uintptr_t)(out + at.head) & 15) == 0;  // the gradient's vectors line up with the logits'
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = i * THREADS + tid;
        if (v >= at.vecs) break;
        float x[R::kE];
#pragma unroll
        for (int j = 0; j < R::kE; ++j) x[j] = each * exp_below(q[i].get(j), r.top);
        store_vec(vec_at(out + at.head, (uint32_t)v), x, along);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (on_edge) store1(out + edge, each * exp_below(x1[0], r.top));
      // the action's, once more, by the thread that stored it: the later of a thread's stores to one place stays
      const int vec = action - at.head;
      const bool mine = vec >= 0 && vec < at.vecs * R::kE ? vec / R::kE % THREADS == tid : on_edge && edge == action;
      if (mine) store1(out + action, each * exp_below(k.logit, r.top) + coef);
    }
  }
}

// Rows of any length: the sums of a row in one pass, for the backward.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void policy_rows_kernel(const mhc_policy_args a, float* logp, float* stats,
                                                                  float* terms) {
  __shared__ float lds[32];
  using R = Row<T>;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const float w = weight_of(a, t);
    if (w == 0.f) {
      if (threadIdx.x == 0) {
        logp[t] = terms[t] = 0.f;
        stats[3 * t] = stats[3 * t + 1] = stats[3 * t + 2] = 0.f;
      }
      continue;
    }
    const T* const row = static_cast<const T*>(a.logits) + t * a.row_stride;
    const R at(row, (int)a.V);
    Running r;
#pragma unroll 4
    for (int v = threadIdx.x; v < at.vecs; v += kRowThreads) {
      Vec<T, R::kE> q;
      q.template load<false>(row + at.head + v * R::kE);
      float x[R::kE];
#pragma unroll
      for (int k = 0; k < R::kE; ++k) x[k] = q.get(k);
      take(r, x);
    }
    if ((int)threadIdx.x < at.head + at.tail) {
      const float x[1] = {load1(row + edge_of(at, (int)a.V, threadIdx.x))};
      take(r, x);
    }
    r = join_workgroup<kRowThreads>(r, lds);
    if (threadIdx.x == 0) {
      const Token k = token_of(a, t, row, r.top, r.sum);
      logp[t] = k.logp;
      terms[t] = w * k.loss;
      stats[3 * t] = r.top;
      stats[3 * t + 1] = 1.f / r.sum;
      stats[3 * t + 2] = w * k.coef;
    }
  }
}

// loss = sum of the terms / D, and 1 / D for the backward (if asked for): one workgroup, a fixed order
__global__ __launch_bounds__(kRowThreads) void policy_loss_kernel(const mhc_policy_args a, const float* terms, float* loss,
                                                                  float* inv) {
  __shared__ float lds[32];
  __shared__ double lds_terms[kRowThreads / kWave];
  double s = 0;  // (terms of both signs)
#pragma unroll 8
  for (int64_t t = threadIdx.x; t < a.T; t += kRowThreads) s += (double)terms[t];
  s = sum_workgroup<kRowThreads>(s, lds_terms);
  const float den = denominator_of<kRowThreads>(a, lds);
  if (threadIdx.x == 0) {
    loss[0] = (float)(s / (double)den);
    if (inv != nullptr) inv[0] = 1.f / den;
  }
}

// The gradient from the rows' sums, one pass over rows of any length.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void policy_grad_kernel(const mhc_policy_args a, const float* stats,
                                                                  const float* dloss, float scale, T* dlogits) {
  using R = Row<T>;
  const float unit = (dloss != nullptr ? dloss[0] : scale) * stats[3 * a.T];
  const int V = (int)a.V;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    T* const out = dlogits + t * a.V;
    if (stats[3 * t + 2] == 0.f) {
      zero_row(out, V, kRowThreads);
      continue;
    }
    const T* const row = static_cast<const T*>(a.logits) + t * a.row_stride;
    const float top = stats[3 * t], coef = stats[3 * t + 2] * unit, each = -coef * stats[3 * t + 1];
    const int action = (int)a.actions[t];
    const R at(out, V);
    const bool along = ((uintptr_t)(row + at.head) & 15) == 0;  // the logits' vectors line up with the gradient's
#pragma unroll 4
    for (int v = threadIdx.x; v < at.vecs; v += kRowThreads) {
      const int first = at.head + v * R::kE;
      Vec<T, R::kE> q;
      if (along) q.load(row + first);
      else __builtin_memcpy(q.w, row + first, 16);
      float x[R::kE];
#pragma unroll
      for (int k = 0; k < R::kE; ++k) x[k] = each * exp_below(q.get(k), top) + (first + k == action ? coef : 0.f);
      store_vec(out + first, x, true);
    }
    if ((int)threadIdx.x < at.head + at.tail) {
      const int v = edge_of(at, V, threadIdx.x);
      store1(out + v, each * exp_below(load1(row + v), top) + (v == action ? coef : 0.f));
    }
  }
}

unsigned grid_of(int64_t T) { return (unsigned)std::min<int64_t>(T, kMaxRows); }

template <typename T, int THREADS, int NV, bool GRAD>
int launch_held(const mhc_policy_args& a, float* logp, float* stats, float* terms, float scale, T* dlogits, hipStream_t s) {
  // as many workgroups as fit the card at once: they go on to further rows
  const int fit = std::max(1, occupancy_blocks(reinterpret_cast<const void*>(policy_held_kernel<T, THREADS, NV, GRAD>), THREADS, 0));
  const unsigned blocks = (unsigned)std::min<int64_t>(a.T, (int64_t)device_cu_count() * fit);
  hipLaunchKernelGGL((policy_held_kernel<T, THREADS, NV, GRAD>), dim3(blocks), dim3(THREADS), 0, s, a, logp, stats, terms, scale, dlogits);
  MHC_CHECK_LAUNCH("policy_held_kernel");
  return MHC_OK;
}

// Whether a row fits a workgroup's registers: 16 vectors of each of 1024 threads.
bool held(const mhc_policy_args& a) { return a.V <= (a.dtype == kF32 ? 65536 : 131072); }

// Long rows are held by 512 threads, so that the rows of two or three
// workgroups of a CU are at different stages (8192 x 50257 bf16: 335 us for
// loss and gradient, 133 for the loss; 1024 threads 365 and 170), unless each
// CU has one at most; short ones by as few as hold them.
template <typename T, bool GRAD>
int run_held(const mhc_policy_args& a, float* logp, float* stats, float* terms, float scale, T* dlogits, hipStream_t s) {
  const int64_t vecs = a.V * (int64_t)sizeof(T) / 16;
  if (vecs <= 64) return launch_held<T, 64, 1, GRAD>(a, logp, stats, terms, scale, dlogits, s);
  if (vecs <= 256) return launch_held<T, 256, 1, GRAD>(a, logp, stats, terms, scale, dlogits, s);
  if (vecs <= 1024) return launch_held<T, 256, 4, GRAD>(a, logp, stats, terms, scale, dlogits, s);
  const bool wide = a.T <= device_cu_count();
  if (vecs <= 4096) {
    return wide ? launch_held<T, 1024, 4, GRAD>(a, logp, stats, terms, scale, dlogits, s)
                : launch_held<T, 512, 8, GRAD>(a, logp, stats, terms, scale, dlogits, s);
  }
  if constexpr (!GRAD) {
    // 13 vectors a thread are the most that leave room for a third workgroup of a CU (78 of 80 registers): the loss of 8192
    // rows of 34000 bf16 120 us, with 16 vectors 134; of 50257 158 and 175; of 53000 158 and 167.  (With the gradient two fit
    // either way, and the time is the same.)
    if (vecs <= 13 * 512 && !wide) return launch_held<T, 512, 13, GRAD>(a, logp, stats, terms, scale, dlogits, s);
  }
  if (vecs <= 8192) {
    return wide ? launch_held<T, 1024, 8, GRAD>(a, logp, stats, terms, scale, dlogits, s)
                : launch_held<T, 512, 16, GRAD>(a, logp, stats, terms, scale, dlogits, s);
  }
  return launch_held<T, 1024, 16, GRAD>(a, logp, stats, terms, scale, dlogits, s);
}

int check_args(const mhc_policy_args* a) {
  MHC_CHECK_ARG(a != nullptr, "null pointer: args");
  MHC_CHECK_ARG(a->T >= 0 && a->V >= 1, "T must be >= 0 and V >= 1 (got %lld, %lld)", (long long)a->T, (long long)a->V);
  MHC_CHECK_ARG(a->V < ((int64_t)1 << 31) - 16, "V %lld is too large", (long long)a->V);
  MHC_CHECK_ARG(a->dtype == kF32 || a->dtype == kBF16 || a->dtype == kF16, "unsupported dtype %d", a->dtype);
  MHC_CHECK_ARG(a->clip_low >= 0 && a->clip_high >= 0, "clip_low and clip_high must be >= 0");
  MHC_CHECK_ARG(a->denominator >= 0, "denominator must be >= 0");
  if (a->T == 0) return MHC_OK;
  MHC_CHECK_ARG(a->logits && a->actions && a->old_logp && a->advantages, "null pointer");
  MHC_CHECK_ARG(a->row_stride >= a->V || a->T == 1, "row_stride must be at least V");
  MHC_CHECK_ARG(a->weights == nullptr || a->weights_dtype == MHC_DTYPE_F32 || a->weights_dtype == MHC_DTYPE_U8,
                "weights must be fp32 or bytes");
  return MHC_OK;
}

int run_loss(const mhc_policy_args& a, const float* terms, float* loss, float* inv, hipStream_t s) {
  hipLaunchKernelGGL(policy_loss_kernel, dim3(1), dim3(kRowThreads), 0, s, a, terms, loss, inv);
  MHC_CHECK_LAUNCH("policy_loss_kernel");
  return MHC_OK;
}

template <typename T>
int run_fwd(const mhc_policy_args& a, float* loss, float* logp, float* stats, float* terms, hipStream_t s) {
  int rc = MHC_OK;
  if (a.T > 0 && held(a)) {
    rc = run_held<T, false>(a, logp, stats, terms, 1.f, nullptr, s);
  } else if (a.T > 0) {
    hipLaunchKernelGGL((policy_rows_kernel<T>), dim3(grid_of(a.T)), dim3(kRowThreads), 0, s, a, logp, stats, terms);
    MHC_CHECK_LAUNCH("policy_rows_kernel");
  }
  return rc != MHC_OK ? rc : run_loss(a, terms, loss, stats + 3 * a.T, s);
}

template <typename T>
int run_bwd(const mhc_policy_args& a, const float* stats, const float* dloss, float scale, void* dlogits, hipStream_t s) {
  hipLaunchKernelGGL((policy_grad_kernel<T>), dim3(grid_of(a.T)), dim3(kRowThreads), 0, s, a, stats, dloss, scale,
                     static_cast<T*>(dlogits));
  MHC_CHECK_LAUNCH("policy_grad_kernel");
  return MHC_OK;
}

template <typename T>
int run_fwd_bwd(const mhc_policy_args& a, float scale, float* loss, float* logp, void* dlogits, float* stats, float* terms, hipStream_t s) {
  if (a.T == 0 || !held(a)) {
    if (const int rc = run_fwd<T>(a, loss, logp, stats, terms, s)) return rc;
    return a.T == 0 ? MHC_OK : run_bwd<T>(a, stats, nullptr, scale, dlogits, s);
  }
  if (const int rc = run_held<T, true>(a, logp, nullptr, terms, scale, static_cast<T*>(dlogits), s)) return rc;
  return run_loss(a, terms, loss, nullptr, s);
}

}  // namespace
}  // namespace mhc

// the terms [T], then (for the call that has no caller's) the stats [3 T + 1]
extern "C" size_t mhc_policy_loss_workspace_bytes(int64_t T) { return T < 0 ? 0 : (size_t)(4 * T + 1) * sizeof(float); }

extern "C" int mhc_policy_loss_fwd(const mhc_policy_args* args, float* loss, float* logp, float* stats, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_args(args)) return rc;
  MHC_CHECK_ARG(loss != nullptr && stats != nullptr && (logp != nullptr || args->T == 0), "null pointer");
  MHC_CHECK_ARG(args->T == 0 || (workspace != nullptr && workspace_bytes >= (size_t)args->T * sizeof(float)),
                "workspace too small");
  float* const terms = static_cast<float*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (args->dtype == kF32) return run_fwd<float>(*args, loss, logp, stats, terms, s);
  if (args->dtype == kBF16) return run_fwd<__bf16>(*args, loss, logp, stats, terms, s);
  return run_fwd<_Float16>(*args, loss, logp, stats, terms, s);
}

extern "C" int mhc_policy_loss_bwd(const mhc_policy_args* args, const float* stats, const float* dloss, void* dlogits,
                                   void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_args(args)) return rc;
  if (args->T == 0) return MHC_OK;
  MHC_CHECK_ARG(stats != nullptr && dlogits != nullptr, "null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (args->dtype == kF32) return run_bwd<float>(*args, stats, dloss, 1.f, dlogits, s);
  if (args->dtype == kBF16) return run_bwd<__bf16>(*args, stats, dloss, 1.f, dlogits, s);
  return run_bwd<_Float16>(*args, stats, dloss, 1.f, dlogits, s);
}

extern "C" int mhc_policy_loss_fwd_bwd(const mhc_policy_args* args, float grad_scale, float* loss, float* logp,
                                       void* dlogits, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_args(args)) return rc;
  MHC_CHECK_ARG(loss != nullptr && ((logp != nullptr && dlogits != nullptr) || args->T == 0), "null pointer");
  MHC_CHECK_ARG(workspace != nullptr && workspace_bytes >= mhc_policy_loss_workspace_bytes(args->T), "workspace too small");
  float* const terms = static_cast<float*>(workspace);
  float* const stats = terms + args->T;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (args->dtype == kF32) return run_fwd_bwd<float>(*args, grad_scale, loss, logp, dlogits, stats, terms, s);
  if (args->dtype == kBF16) return run_fwd_bwd<__bf16>(*args, grad_scale, loss, logp, dlogits, stats, terms, s);
  return run_fwd_bwd<_Float16>(*args, grad_scale, loss, logp, dlogits, stats, terms, s);
}
