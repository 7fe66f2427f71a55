// linear_cross_entropy's gradients of up to 16 tokens (8 of 16-bit rows), from
// logits that were kept:
//
//   dx[t] = sum_v dz[t, v] W[v];  dW[v] = sum_t dz[t, v] x[t]
//
// One pass over W and dW by the vector unit, with dz in fp32 (rounded to 16
// bits, the few elements at the targets would be most of dW's error).  A wave
// has four columns a lane: x's values there and dx's sums in registers, dz from
// scalar loads, a row of W and of dW at a time.  Bound by memory (2 x 72999 x 2624
// fp32: 1.53 GB in 289 us, 5.3 TB/s; 4 x 32000 x 4096 bf16 524 MB in 135, 3.9).
#include "mhc_ce.hpp"
#include "mhc_plan.hpp"

namespace mhc {
namespace ce {
namespace {

constexpr int kWaves = 4, kVec = 4;  // of a workgroup, which shares its columns; columns of a lane

template <int TP> constexpr int kAhead = TP > 8 ? 4 : 8;  // rows of a wave under way

struct Few {
  const void *x, *w;
  int64_t ldx, ldw, V;
  const float* dz;   // [V, TP]
  void* dw;          // or NULL
  float* part;       // dx's sums, [parts, TP, pitch], or NULL
  int C;
  int64_t pitch;
  ScaledBy by;
};

// dz [V, TP], zeros for tokens that are not there
template <int TP>
__global__ __launch_bounds__(256) void few_dz_kernel(const Gradient g, const Kept kept, float* dz, int64_t V, const int* live) {
  const int n = *live;
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= V) return;
  float d[TP];
#pragma unroll
  for (int t = 0; t < TP; ++t) {
    const int m = max(min(t, n - 1), 0);  // (a load under a condition would wait for itself)
    const Gradient::Row r = g.row(m);
    d[t] = r.each * gemm::exp_of<false>(kept.z[m * kept.pitch + v] - r.t) - (r.to == v ? r.c : 0.f);
    d[t] = t < n ? d[t] : 0.f;
  }
#pragma unroll
  for (int t = 0; t < TP; ++t) dz[v * TP + t] = d[t];
}

// four elements, past the caches: dW is not read soon (2 x 72999 x 2624 fp32 327 us, through the caches 390)
template <typename T>
MHC_DEV void store_past(T* p, const float (&v)[kVec]) {
  typedef uint32_t words __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
  words w;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < kVec; ++k) w[k] = __builtin_bit_cast(uint32_t, v[k]);
  } else {
    w[0] = pack2<T>(v[0], v[1]);
    w[1] = pack2<T>(v[2], v[3]);
  }
  __builtin_nontemporal_store(w, reinterpret_cast<words*>(p));
}

template <typename T, int TP>
__global__ __launch_bounds__(64 * kWaves) void few_kernel(const Few a, const int* live, const int* index) {
  constexpr int V = kVec, A = kAhead<TP>;
  __shared__ float lds[kWaves - 1][kWave * V];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = (blockIdx.x * kWave + lane) * V, left = min(V, a.C - c);
  const int n = __builtin_amdgcn_readfirstlane(*live);
  const auto take = [&](const T* p, float(&z)[V]) {
    if (left < V) {
      gemm::take<false>(p, z, max(left, 0));
    } else if constexpr (V * sizeof(T) == 8) {
      Vec<T, V> r;
      __builtin_memcpy(r.w, p, 8);
#pragma unroll
      for (int k = 0; k < V; ++k) z[k] = r.get(k);
    } else {
      gemm::take<true>(p, z, V);
    }
  };
  float x[TP][V], sum[TP][V] = {};
#pragma unroll
  for (int t = 0; t < TP; ++t) {
#pragma unroll
    for (int k = 0; k < V; ++k) x[t][k] = 0.f;
    if (t < n) take(static_cast<const T*>(a.x) + index[t] * a.ldx + c, x[t]);
  }
  const float scale = a.by.a[0] * (a.by.b != nullptr ? a.by.b[0] : 1.f) * a.by.c;
  // rows of the workgroup, its waves one after the other
  const int64_t v0 = a.V * blockIdx.y / gridDim.y, v1 = a.V * (blockIdx.y + 1) / gridDim.y;
  const auto* const dz = (const __attribute__((address_space(4))) float*)(uintptr_t)a.dz;
  for (int64_t v = v0 + wave; v < v1; v += kWaves * A) {
    float w[A][V] = {}, d[A][TP];
#pragma unroll
    for (int q = 0; q < A; ++q) {  // (rows past the last one read it once more)
      const int64_t row = min(v + q * kWaves, v1 - 1);
      if (a.part != nullptr) take(static_cast<const T*>(a.w) + row * a.ldw + c, w[q]);
#pragma unroll
      for (int t = 0; t < TP; ++t) d[q][t] = dz[row * TP + t];
    }
#pragma unroll
    for (int q = 0; q < A; ++q) {
      const int64_t row = v + q * kWaves;
      if (row >= v1) break;
      float out[V] = {};
#pragma unroll
      for (int t = 0; t < TP; ++t)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          sum[t][k] = fmaf(d[q][t], w[q][k], sum[t][k]);
          out[k] = fmaf(d[q][t], x[t][k], out[k]);
        }
      if (a.dw != nullptr) {
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] *= scale;
        T* const to = static_cast<T*>(a.dw) + row * a.C + c;
        if (left == V) store_past(to, out);
        else if (left > 0) gemm::put<false>(to, out, left);
      }
    }
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int t = 0; t < TP; ++t) {
    __syncthreads();
    if (wave > 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) lds[wave - 1][k * kWave + lane] = sum[t][k];
    }
    __syncthreads();
    if (wave > 0) continue;
#pragma unroll
    for (int q = 0; q < kWaves - 1; ++q)
#pragma unroll
      for (int k = 0; k < V; ++k) sum[t][k] += lds[q][k * kWave + lane];
    float* const to = a.part + ((int64_t)blockIdx.y * TP + t) * a.pitch + c;
    if (c < a.pitch) *reinterpret_cast<f32x4*>(to) = f32x4{sum[t][0], sum[t][1], sum[t][2], sum[t][3]};
  }
}

// dx of every token from the parts' sums: 64 columns a workgroup, 16 groups of threads with every 16th part
template <typename T>
__global__ __launch_bounds__(256) void few_join_kernel(const float* part, int parts, int tp, int64_t pitch, const State s, const ScaledBy by, T* dx, int C) {
  __shared__ f32x4 lds[16][16];
  const int lane = threadIdx.x % 16, q = threadIdx.x / 16, t = blockIdx.y, c = (blockIdx.x * 16 + lane) * 4;
  const int pos = s.pos[t];
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (pos >= 0 && c < pitch) {
#pragma unroll 4
    for (int k = q; k < parts; k += 16) sum += *reinterpret_cast<const f32x4*>(part + ((int64_t)k * tp + pos) * pitch + c);
  }
  lds[q][lane] = sum;
  __syncthreads();
  if (q != 0) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) sum += lds[k][lane];
  const float scale = by.a[0] * (by.b != nullptr ? by.b[0] : 1.f) * by.c;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c + k < C) store1(dx + (int64_t)t * C + c + k, pos >= 0 ? sum[k] * scale : 0.f);
}

int padded_tokens(int64_t T) { return T <= 2 ? 2 : T <= 4 ? 4 : T <= 8 ? 8 : 16; }

struct Grid {
  int64_t columns, parts, pitch;
};

// Some 2048 workgroups, each with 64 rows at least.
Grid grid_of(const mhc_linear_ce_args& a) {
  const int64_t columns = ceil_div(a.C, kWave * kVec);
  return {columns, std::max<int64_t>(1, std::min(ceil_div(a.V, 64), (int64_t)device_cu_count() * 8 / columns)), ceil_div(a.C, 4) * 4};
}

template <typename T, int TP>
int run(const mhc_linear_ce_args& a, const State& st, const ScaledBy& by, void* dx, void* dw, char* ws, hipStream_t s) {
  const Grid grid = grid_of(a);
  float* const dz = reinterpret_cast<float*>(ws);
  float* const part = dz + (a.V * TP + 63) / 64 * 64;
  const Gradient g = {st.target, st.coef, st.top, st.inv, 0, 1.f};
  hipLaunchKernelGGL((few_dz_kernel<TP>), dim3((unsigned)ceil_div(a.V, 256)), dim3(256), 0, s, g, Kept{a.logits, kept_pitch(a.V)}, dz, a.V, (const int*)st.head);
  MHC_CHECK_LAUNCH("few_dz_kernel");
  const Few f = {a.x, a.w, a.ldx, a.ldw, a.V, dz, dw, dx != nullptr ? part : nullptr, (int)a.C, grid.pitch, by};
  hipLaunchKernelGGL((few_kernel<T, TP>), dim3((unsigned)grid.columns, (unsigned)grid.parts), dim3(64 * kWaves), 0, s, f, (const int*)st.head,
                     (const int*)st.index);
  MHC_CHECK_LAUNCH("few_kernel");
  if (dx == nullptr) return MHC_OK;
  hipLaunchKernelGGL((few_join_kernel<T>), dim3((unsigned)ceil_div(a.C, 64), (unsigned)a.T), dim3(256), 0, s, (const float*)part, (int)grid.parts, TP,
                     grid.pitch, st, by, static_cast<T*>(dx), (int)a.C);
  MHC_CHECK_LAUNCH("few_join_kernel");
  return MHC_OK;
}

template <typename T>
int run(const mhc_linear_ce_args& a, const State& st, const ScaledBy& by, void* dx, void* dw, char* ws, hipStream_t s) {
  switch (padded_tokens(a.T)) {
    case 2: return run<T, 2>(a, st, by, dx, dw, ws, s);
    case 4: return run<T, 4>(a, st, by, dx, dw, ws, s);
    case 8: return run<T, 8>(a, st, by, dx, dw, ws, s);
  }
  if constexpr (sizeof(T) == 4) return run<T, 16>(a, st, by, dx, dw, ws, s);
  return MHC_OK;  // (not reached: few_tokens())
}

}  // namespace

size_t few_bytes(const mhc_linear_ce_args& a) {
  const int64_t tp = padded_tokens(a.T);
  const Grid grid = grid_of(a);
  return (size_t)((a.V * tp + 63) / 64 * 64 + grid.parts * tp * grid.pitch) * sizeof(float);
}

int run_few(const mhc_linear_ce_args& a, const State& st, const float* dloss, float grad_scale, void* dx, void* dw, char* ws, hipStream_t s) {
  const ScaledBy by = {reinterpret_cast<const float*>(st.head) + 1, dloss, grad_scale};
  if (a.dtype == kF32) return run<float>(a, st, by, dx, dw, ws, s);
  if (a.dtype == kBF16) return run<__bf16>(a, st, by, dx, dw, ws, s);
  return run<_Float16>(a, st, by, dx, dw, ws, s);
}

}  // namespace ce
}  // namespace mhc
