// Clipped policy loss with a KL term, from the logits, and its gradient.
//
//   lp = z_a - log sum_v exp z_v;  r = exp(lp - old);  q = exp(ref - lp)
//   L  = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (q - 1 - log q)
//   c  = dL / dlp = -A r [r A <= clip(r) A] + beta (1 - q)
//   dz_v = w c / D ([v = a] - exp(z_v) / sum)
//
// A workgroup takes a row: one pass with a running largest logit and a sum of
// exponentials below it, a second one for the gradient.  Rows of weight 0,
// and rows whose c is 0 (a clipped token without a KL term), are not read
// again: their gradient is zeros.
#include "mhc_device.hpp"
#include "mhc_host.hpp"

namespace mhc {
namespace {

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / kWave;
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

// one result for the workgroup, in every thread, joined in a fixed order
MHC_DEV Running join_workgroup(Running r, float (&lds)[2 * kRowWaves]) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) join(r, __shfl_xor(r.top, d), __shfl_xor(r.sum, d));
  const int wave = threadIdx.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) {
    lds[wave] = r.top;
    lds[kRowWaves + wave] = r.sum;
  }
  __syncthreads();
  Running all;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) join(all, lds[w], lds[kRowWaves + w]);
  return all;
}

MHC_DEV float weight_of(const mhc_policy_args& a, int64_t t) {
  if (a.weights == nullptr) return 1.f;
  return a.weights_dtype == MHC_DTYPE_U8 ? (static_cast<const uint8_t*>(a.weights)[t] != 0 ? 1.f : 0.f)
                                         : static_cast<const float*>(a.weights)[t];
}

struct Token {
  float loss, logp, coef;  // without the weight
};

template <typename T>
MHC_DEV Token token_of(const mhc_policy_args& a, int64_t t, const T* row, float top, float sum) {
  const int64_t at = a.actions[t];
  const float nan = __builtin_nanf("");
  const float z = at >= 0 && at < a.V ? load1(row + at) : nan;
  const float lp = (z - top) - logf(sum);
  const float ratio = expf(lp - a.old_logp[t]), adv = a.advantages[t];
  // (a NaN ratio stays one: fminf and fmaxf would drop it)
  const float held_ratio = ratio < 1.f - a.clip_low ? 1.f - a.clip_low : ratio > 1.f + a.clip_high ? 1.f + a.clip_high : ratio;
  const float free = ratio * adv, held = held_ratio * adv;
  Token r;
  r.logp = lp;
  r.loss = -(free <= held ? free : held);
  r.coef = free <= held ? -free : 0.f;
  if (!(free == free)) r.loss = r.coef = nan;
  if (a.ref_logp != nullptr) {
    const float gap = a.ref_logp[t] - lp, over = expm1f(gap);  // q - 1 without cancellation near q = 1
    r.loss += a.kl_coef * (over - gap);
    r.coef -= a.kl_coef * over;
  }
  return r;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void policy_rows_kernel(const mhc_policy_args a, float* logp, float* stats,
                                                                  float* terms) {
  __shared__ float lds[2 * kRowWaves];
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
    for (int v = threadIdx.x; v < at.vecs; v += kRowThreads) {
      Vec<T, R::kE> q;
      q.template load<false>(row + at.head + v * R::kE);
      float x[R::kE];
#pragma unroll
      for (int k = 0; k < R::kE; ++k) x[k] = q.get(k);
      take(r, x);
    }
    if ((int)threadIdx.x < at.head + at.tail) {
      const int v = (int)threadIdx.x < at.head ? (int)threadIdx.x : (int)(a.V - at.tail) + ((int)threadIdx.x - at.head);
      const float x[1] = {load1(row + v)};
      take(r, x);
    }
    r = join_workgroup(r, lds);
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

// a sum over the workgroup's threads, in every thread, in a fixed order
MHC_DEV float sum_workgroup(float s, float (&lds)[2 * kRowWaves]) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) all += lds[w];
  return all;
}

// loss = sum of the terms / D, and 1 / D for the backward: one workgroup, a fixed order
__global__ __launch_bounds__(kRowThreads) void policy_loss_kernel(const mhc_policy_args a, const float* terms, float* loss,
                                                                  float* inv) {
  __shared__ float lds[2 * kRowWaves];
  float s = 0.f, d = 0.f;
  for (int64_t t = threadIdx.x; t < a.T; t += kRowThreads) {
    s += terms[t];
    d += weight_of(a, t);
  }
  s = sum_workgroup(s, lds);
  d = sum_workgroup(d, lds);
  if (threadIdx.x == 0) {
    const float den = a.denominator > 0.f ? a.denominator : d != 0.f ? d : 1.f;
    loss[0] = s / den;
    inv[0] = 1.f / den;
  }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void policy_grad_kernel(const mhc_policy_args a, const float* stats,
                                                                  const float* dloss, float scale, T* dlogits) {
  using R = Row<T>;
  const float unit = (dloss != nullptr ? dloss[0] : scale) * stats[3 * a.T];
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* const row = static_cast<const T*>(a.logits) + t * a.row_stride;
    T* const out = dlogits + t * a.V;
    const float top = stats[3 * t], coef = stats[3 * t + 2] * unit, each = -coef * stats[3 * t + 1];
    const int action = (int)a.actions[t];
    const R at(out, (int)a.V);
    const bool along = ((uintptr_t)(row + at.head) & 15) == 0;  // the logits' vectors line up with the gradient's
    if (stats[3 * t + 2] == 0.f) {
      for (int v = threadIdx.x; v < at.vecs; v += kRowThreads)
        *reinterpret_cast<u32x4*>(out + at.head + v * R::kE) = u32x4{0, 0, 0, 0};
    } else {
      for (int v = threadIdx.x; v < at.vecs; v += kRowThreads) {
        const int first = at.head + v * R::kE;
        Vec<T, R::kE> q;
        if (along) {
          q.template load<false>(row + first);
        } else {
          __builtin_memcpy(q.w, row + first, 16);
        }
        float x[R::kE];
#pragma unroll
        for (int k = 0; k < R::kE; ++k) x[k] = each * exp_below(q.get(k), top) + (first + k == action ? coef : 0.f);
        u32x4 o;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) o[k] = __builtin_bit_cast(uint32_t, x[k]);
          else o[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
        }
        *reinterpret_cast<u32x4*>(out + first) = o;
      }
    }
    if ((int)threadIdx.x < at.head + at.tail) {
      const int v = (int)threadIdx.x < at.head ? (int)threadIdx.x : (int)(a.V - at.tail) + ((int)threadIdx.x - at.head);
      const float g = stats[3 * t + 2] == 0.f ? 0.f : each * exp_below(load1(row + v), top) + (v == action ? coef : 0.f);
      store1(out + v, g);
    }
  }
}

unsigned grid_of(int64_t T) { return (unsigned)std::min<int64_t>(T, kMaxRows); }

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

template <typename T>
int run_fwd(const mhc_policy_args& a, float* loss, float* logp, float* stats, float* terms, hipStream_t s) {
  if (a.T > 0) {
    hipLaunchKernelGGL((policy_rows_kernel<T>), dim3(grid_of(a.T)), dim3(kRowThreads), 0, s, a, logp, stats, terms);
    MHC_CHECK_LAUNCH("policy_rows_kernel");
  }
  hipLaunchKernelGGL(policy_loss_kernel, dim3(1), dim3(kRowThreads), 0, s, a, (const float*)terms, loss, stats + 3 * a.T);
  MHC_CHECK_LAUNCH("policy_loss_kernel");
  return MHC_OK;
}

template <typename T>
int run_bwd(const mhc_policy_args& a, const float* stats, const float* dloss, float scale, void* dlogits, hipStream_t s) {
  hipLaunchKernelGGL((policy_grad_kernel<T>), dim3(grid_of(a.T)), dim3(kRowThreads), 0, s, a, stats, dloss, scale,
                     static_cast<T*>(dlogits));
  MHC_CHECK_LAUNCH("policy_grad_kernel");
  return MHC_OK;
}

int fwd(const mhc_policy_args& a, float* loss, float* logp, float* stats, float* terms, hipStream_t s) {
  if (a.dtype == kF32) return run_fwd<float>(a, loss, logp, stats, terms, s);
  if (a.dtype == kBF16) return run_fwd<__bf16>(a, loss, logp, stats, terms, s);
  return run_fwd<_Float16>(a, loss, logp, stats, terms, s);
}

int bwd(const mhc_policy_args& a, const float* stats, const float* dloss, float scale, void* dlogits, hipStream_t s) {
  if (a.dtype == kF32) return run_bwd<float>(a, stats, dloss, scale, dlogits, s);
  if (a.dtype == kBF16) return run_bwd<__bf16>(a, stats, dloss, scale, dlogits, s);
  return run_bwd<_Float16>(a, stats, dloss, scale, dlogits, s);
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
  return fwd(*args, loss, logp, stats, static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
}

extern "C" int mhc_policy_loss_bwd(const mhc_policy_args* args, const float* stats, const float* dloss, void* dlogits,
                                   void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_args(args)) return rc;
  if (args->T == 0) return MHC_OK;
  MHC_CHECK_ARG(stats != nullptr && dlogits != nullptr, "null pointer");
  return bwd(*args, stats, dloss, 1.f, dlogits, static_cast<hipStream_t>(stream));
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
  if (const int rc = fwd(*args, loss, logp, stats, terms, s)) return rc;
  return args->T == 0 ? MHC_OK : bwd(*args, stats, nullptr, grad_scale, dlogits, s);
}
