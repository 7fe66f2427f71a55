// One AdamW step over a list of tensors, with first and second moments in 32
// or in 8 bits.
//
//   p <- p (1 - lr wd)
//   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g g
//   p <- p - (m / (sqrt(v) / sqrt(1 - b2^t) + eps)) (lr / (1 - b1^t))
//
// Every operation is rounded to fp32 by itself (no contraction): the result
// does not depend on how a tensor is cut into vectors and workgroups, and is
// that of the same formula in elementary tensor operations.
//
// A model around mHC layers has hundreds of tensors of 4 to 4096 floats next
// to a few of millions.  As many of them go into one launch as the kernel
// arguments hold (100 in fp32, 84 with master copies, 72 with both and states
// in 8 bits): their pointers travel there (no table in device memory that a
// captured graph or a later step could find changed), and a workgroup finds
// its tensor with one or two loads of the chunk counts, a lane each, and
// votes.  Large tensors are bound by memory (16 of 4096 x 4096 bf16 with
// masters: 28 bytes an element at 5.2 TB/s; in 8 bits the same), lists of
// small ones by the host.
#include <cmath>

#include "mhc_device.hpp"
#include "mhc_host.hpp"

namespace mhc {
namespace {

constexpr int kThreads = 256;
constexpr int kQuant = 256;       // elements that share a scale: one wave, four elements a lane
constexpr int kPass = kThreads * 4;  // elements that a workgroup has at a time
constexpr int kChunk = 4 * kPass; // elements of one workgroup (kPass in a call too small to fill the card: four passes take 5 us)
constexpr int64_t kMaxChunks = 1 << 23;  // workgroups of a launch: its threads stay below 2^31
constexpr float kCodeMax = 448.f; // largest e4m3 value
constexpr float kMinTop = 0x1p-100f;  // least largest value of a block: its scale's inverse stays finite

struct Hyper {
  float decay, b1, c1, b2, c2, inv_bc2, eps, rate, gscale;
  const float* gscale_ptr;  // a factor of the gradients in device memory, or NULL
};

template <bool MASTER, bool Q8>
struct Table {
  static constexpr int kPointers = 4 + MASTER + Q8;
  static constexpr int kMax = (4096 - (int)sizeof(Hyper) - 16) / (8 * kPointers + 8);
  void* p[kMax][kPointers];  // param, grad, exp_avg, exp_avg_sq, master, scales
  int32_t end[kMax];         // chunks of the tensors up to and with this one
  int32_t last[kMax];        // elements of the tensor's last chunk
  int32_t count, chunk;      // elements of a chunk
  Hyper h;
};
static_assert(sizeof(Table<false, false>) <= 4096 && sizeof(Table<true, false>) <= 4096 && sizeof(Table<true, true>) <= 4096,
              "kernel arguments");

struct Quad {
  float v[4];
};

// four elements at p: as one vector, or one by one below `left` of them
template <typename T>
MHC_DEV Quad load4(const T* p, bool vec, int left) {
  Quad q;
  if (vec && left >= 4) {
    Vec<T, 4> r;
    r.load(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = r.get(k);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = k < left ? load1(p + k) : 0.f;
  }
  return q;
}

template <typename T>
MHC_DEV void store4(T* p, const Quad& q, bool vec, int left) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>(p) = f32x4{q.v[0], q.v[1], q.v[2], q.v[3]};
    } else {
      *reinterpret_cast<u32x2*>(p) = u32x2{pack2<T>(q.v[0], q.v[1]), pack2<T>(q.v[2], q.v[3])};
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) store1(p + k, q.v[k]);
  }
}

MHC_DEV uint32_t load_codes(const uint8_t* p, bool vec, int left) {
  if (vec && left >= 4) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) w |= (uint32_t)p[k] << (8 * k);
  return w;
}

MHC_DEV void store_codes(uint8_t* p, uint32_t w, bool vec, int left) {
  if (vec && left >= 4) {
    *reinterpret_cast<uint32_t*>(p) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = (uint8_t)(w >> (8 * k));
  }
}

MHC_DEV Quad decode(uint32_t w, float scale) {
#pragma clang fp contract(off)
  return Quad{{__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale,
               __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale}};
}

// The largest magnitude of a wave's elements.  Magnitudes are compared as
// integers, which orders them as the values and puts NaN on top, so that a
// NaN reaches the block's scale instead of being lost.
MHC_DEV float wave_top(const Quad& q) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = max(top, __builtin_bit_cast(uint32_t, q.v[k]) & 0x7fffffffu);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  return __builtin_bit_cast(float, max(top, __builtin_bit_cast(uint32_t, kMinTop)));
}

MHC_DEV uint32_t encode(const Quad& q, float top) {
#pragma clang fp contract(off)
  const float inv = (1.f / top) * kCodeMax;  // (the plain form's order)
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q.v[0] * inv, q.v[1] * inv, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q.v[2] * inv, q.v[3] * inv, w, true);
  return (uint32_t)w;
}

MHC_DEV bool lines_up(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

template <typename P, bool MASTER, bool Q8>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Table<MASTER, Q8> tab) {
#pragma clang fp contract(off)
  constexpr int kMax = Table<MASTER, Q8>::kMax;
  static_assert(kMax > kWave && kMax <= 2 * kWave, "two tensors for each lane");
  const int chunk = (int)blockIdx.x, lane = (int)threadIdx.x % kWave;
  int lo;
  const uint64_t past = __ballot(lane < tab.count && tab.end[lane] > chunk);
  if (past != 0) {
    lo = __builtin_ctzll(past);
  } else {
    const int at = kWave + lane;
    lo = kWave + __builtin_ctzll(__ballot(at < tab.count && tab.end[min(at, kMax - 1)] > chunk));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  void* const* const t = tab.p[lo];
  const int64_t first = (int64_t)(chunk - (lo > 0 ? tab.end[lo - 1] : 0)) * tab.chunk;
  const int64_t end = first + (chunk + 1 == tab.end[lo] ? tab.last[lo] : tab.chunk);
  P* const p = static_cast<P*>(t[0]);
  const P* const g = static_cast<const P*>(t[1]);
  float* const master = MASTER ? static_cast<float*>(t[3 + MASTER]) : nullptr;
  float* const scales = Q8 ? static_cast<float*>(t[3 + MASTER + Q8]) : nullptr;
  const Hyper& h = tab.h;
  const float gs = h.gscale_ptr != nullptr ? h.gscale * *h.gscale_ptr : h.gscale;
  // four elements at a multiple of four from an aligned start are one vector
  const bool pvec = lines_up(p, 4 * sizeof(P)) && lines_up(g, 4 * sizeof(P));
  const bool svec = Q8 ? lines_up(t[2], 4) && lines_up(t[3], 4) : lines_up(t[2], 16) && lines_up(t[3], 16);
  const bool mvec = !MASTER || lines_up(master, 16);

  for (int64_t i = first + threadIdx.x * 4; ; i += kPass) {
    // a wave's 256 elements are one block of an 8-bit state; its lanes past the end take part with zeros
    const int left = (int)min((int64_t)4, end - i);
    if (i - lane * 4 >= end) break;
    Quad gq = load4(g + i, pvec, left), pq;
    if constexpr (MASTER) pq = load4(master + i, mvec, left);
    else pq = load4(p + i, pvec, left);
    Quad mq, vq;
    const int64_t b = i / kQuant;
    if constexpr (Q8) {
      mq = decode(load_codes(static_cast<const uint8_t*>(t[2]) + i, svec, left), scales[2 * b]);
      vq = decode(load_codes(static_cast<const uint8_t*>(t[3]) + i, svec, left), scales[2 * b + 1]);
#pragma unroll
      for (int k = 0; k < 4; ++k) vq.v[k] = vq.v[k] * vq.v[k];
    } else {
      mq = load4(static_cast<const float*>(t[2]) + i, svec, left);
      vq = load4(static_cast<const float*>(t[3]) + i, svec, left);
    }
    Quad rq;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gk = gq.v[k] * gs;
      mq.v[k] = mq.v[k] * h.b1 + gk * h.c1;
      vq.v[k] = vq.v[k] * h.b2 + (gk * gk) * h.c2;
      rq.v[k] = sqrtf(vq.v[k]);
      const float step = mq.v[k] / (rq.v[k] * h.inv_bc2 + h.eps);
      pq.v[k] = pq.v[k] * h.decay - step * h.rate;
    }
    if constexpr (Q8) {
      // the second moment is held as its root: half the exponents, so 8 bits cover 2^35 of v below a block's largest
      const float mt = wave_top(mq), rt = wave_top(rq);
      store_codes(static_cast<uint8_t*>(t[2]) + i, encode(mq, mt), svec, left);
      store_codes(static_cast<uint8_t*>(t[3]) + i, encode(rq, rt), svec, left);
      if (threadIdx.x % kWave == 0) {
        scales[2 * b] = mt * (1.f / kCodeMax);
        scales[2 * b + 1] = rt * (1.f / kCodeMax);
      }
    } else {
      store4(static_cast<float*>(t[2]) + i, mq, svec, left);
      store4(static_cast<float*>(t[3]) + i, vq, svec, left);
    }
    if constexpr (MASTER) store4(master + i, pq, mvec, left);
    store4(p + i, pq, pvec, left);
  }
}

template <typename P, bool MASTER, bool Q8>
int launch(const mhc_adamw_tensor* tensors, int64_t count, const Hyper& h, hipStream_t s) {
  Table<MASTER, Q8> tab;
  const auto run = [&] {
    hipLaunchKernelGGL((adamw_kernel<P, MASTER, Q8>), dim3((unsigned)tab.end[tab.count - 1]), dim3(kThreads), 0, s, tab);
    MHC_CHECK_LAUNCH("adamw_kernel");
    return MHC_OK;
  };
  tab.h = h;
  tab.count = 0;
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += tensors[i].numel;
  tab.chunk = total < (int64_t)device_cu_count() * 8 * kChunk ? kPass : kChunk;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const mhc_adamw_tensor& t = tensors[i];
    if (t.numel == 0) continue;
    const int64_t mine = ceil_div(t.numel, tab.chunk);
    if (tab.count == Table<MASTER, Q8>::kMax || (tab.count > 0 && chunks + mine > kMaxChunks)) {
      if (const int rc = run()) return rc;
      tab.count = 0;
      chunks = 0;
    }
    chunks += mine;
    void** const p = tab.p[tab.count];
    p[0] = t.param, p[1] = const_cast<void*>(t.grad), p[2] = t.exp_avg, p[3] = t.exp_avg_sq;
    if constexpr (MASTER) p[4] = t.master;
    if constexpr (Q8) p[4 + MASTER] = t.scales;
    tab.end[tab.count] = (int32_t)chunks;
    tab.last[tab.count] = (int32_t)(t.numel - (mine - 1) * tab.chunk);
    ++tab.count;
  }
  return tab.count > 0 ? run() : MHC_OK;
}

template <typename P>
int launch_for(const mhc_adamw_tensor* tensors, int64_t count, const Hyper& h, bool master, bool q8, hipStream_t s) {
  if constexpr (sizeof(P) == 2) {
    if (master) return q8 ? launch<P, true, true>(tensors, count, h, s) : launch<P, true, false>(tensors, count, h, s);
  }
  return q8 ? launch<P, false, true>(tensors, count, h, s) : launch<P, false, false>(tensors, count, h, s);
}

}  // namespace
}  // namespace mhc

extern "C" int mhc_adamw_step(const mhc_adamw_tensor* tensors, int64_t count, int dtype, int state_bits, double lr,
                              double beta1, double beta2, double eps, double weight_decay, int64_t step,
                              double grad_scale, const float* grad_scale_ptr, void* stream) {
  using namespace mhc;
  clear_error();
  MHC_CHECK_ARG(count >= 0, "count must be >= 0 (got %lld)", (long long)count);
  MHC_CHECK_ARG(dtype == kF32 || dtype == kBF16 || dtype == kF16, "unsupported dtype %d", dtype);
  MHC_CHECK_ARG(state_bits == 32 || state_bits == 8, "state_bits must be 32 or 8 (got %d)", state_bits);
  MHC_CHECK_ARG(lr >= 0 && eps >= 0 && weight_decay >= 0, "lr, eps and weight_decay must be >= 0");
  MHC_CHECK_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas must be in [0, 1) (got %g, %g)", beta1,
                beta2);
  MHC_CHECK_ARG(step >= 1, "step must be >= 1 (got %lld)", (long long)step);
  if (count == 0) return MHC_OK;
  MHC_CHECK_ARG(tensors != nullptr, "null pointer: tensors");
  int64_t any = 0;  // a tensor with elements (one without has no addresses)
  while (any + 1 < count && tensors[any].numel == 0) ++any;
  const bool q8 = state_bits == 8, master = tensors[any].master != nullptr;
  MHC_CHECK_ARG(!master || dtype != kF32, "a master copy is for 16-bit parameters");
  for (int64_t i = 0; i < count; ++i) {
    const mhc_adamw_tensor& t = tensors[i];
    MHC_CHECK_ARG(t.numel >= 0, "tensor %lld: numel must be >= 0", (long long)i);
    MHC_CHECK_ARG((t.master != nullptr) == master || t.numel == 0, "tensor %lld: all tensors of a call have a master copy, or none",
                  (long long)i);
    if (t.numel == 0) continue;
    MHC_CHECK_ARG(t.param != nullptr && t.grad != nullptr && t.exp_avg != nullptr && t.exp_avg_sq != nullptr &&
                      (!q8 || t.scales != nullptr),
                  "tensor %lld: null pointer", (long long)i);
    MHC_CHECK_ARG(t.numel <= kMaxChunks * kChunk, "tensor %lld: numel %lld is too large", (long long)i,
                  (long long)t.numel);
  }
  const double bc1 = 1.0 - std::pow(beta1, (double)step), bc2 = 1.0 - std::pow(beta2, (double)step);
  const Hyper h = {(float)(1.0 - lr * weight_decay), (float)beta1, (float)(1.0 - beta1), (float)beta2,
                   (float)(1.0 - beta2),             (float)(1.0 / std::sqrt(bc2)), (float)eps, (float)(lr / bc1),
                   (float)grad_scale,                grad_scale_ptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kF32) return launch_for<float>(tensors, count, h, master, q8, s);
  if (dtype == kBF16) return launch_for<__bf16>(tensors, count, h, master, q8, s);
  return launch_for<_Float16>(tensors, count, h, master, q8, s);
}
