// RMS norm with the residual's addition, its int8 form, and its gradients.
//
//   h = x + r, rounded to their type: what the next block adds to is what is normed
//   s = 1 / sqrt(mean h^2 + eps);  y = h s w
//   int8: a = max |h w|;  code = rint(127 h w / a);  scale = a s / 127
//   g = dy w;  n = h s;  dx = dr = s (g - n mean(g n)) + dh;  dw = sum_t dy n
//
// s cancels in the codes, so that they need only a row's largest product: of
// 16-bit values and weights the products are exact in fp32, and so is the code,
// ties included (see Coder).
//
// Bound by memory: a row is read once and written once, held in registers
// between (8192 x 4096 bf16, with a residual: forward 45 us for 268 MB, 6.0 TB/s;
// backward, from the gradients of both outputs, 50 us for 268 MB and 7 for the
// last sums of dw; int8 16 us for 2048 x 4096).  A copy gives 5.2 TB/s.
#include "mhc_gemm.hpp"
#include "mhc_plan.hpp"

namespace mhc {
namespace {

constexpr int kLongThreads = 1024;  // of the kernels for rows of any length
constexpr int kMaxRows = 1 << 20;   // workgroups of a launch; further rows go round again

struct NormArgs {
  const void* x;
  const void* r;   // or NULL
  const void* w;   // or NULL: ones
  int64_t ldx, ldr;
  void* h;         // [T, C], written if there is an r
  void* y;         // [T, C], or int8 codes
  float* scales;   // [T] of the codes
  float* rstd;     // [T], or NULL
  int64_t T;
  int C;
  float eps;
};

enum Mode { kPlain, kCodes, kCodesOnly };  // kCodesOnly: of x itself, without a norm

template <typename T> constexpr int kV = 16 / (int)sizeof(T);  // elements of a vector

// a value over all of a workgroup's threads, in every thread, in a fixed order
template <int THREADS, typename Op>
MHC_DEV float join_threads(float v, Op op, float* lds) {
  v = group_reduce<kWave>(v, op);
  if constexpr (THREADS == kWave) return v;
  const int wave = threadIdx.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[wave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int k = 1; k < THREADS / kWave; ++k) v = op(v, lds[k]);
  return v;
}

// The larger of two magnitudes, as bit patterns: NaN is larger than infinity, and that than any number.
struct LargerOp {
  MHC_DEV float operator()(float a, float b) const {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)));
  }
};

// Codes of values p from the largest magnitude of their row.  Both are scaled
// by a power of two first, so that 127 p and the quotient stay in range; the
// quotient is corrected by its remainder, which makes it the nearest number to
// 127 p / top.  A row of zeros has codes of 0 and the scale 0, one with an
// infinity or NaN codes of 0 and the scale NaN.
//
// 127 p is exact for a p of up to 17 bits (bf16 times bf16 has 16), and no such
// quotient that is not a tie rounds to one.  A product of two fp16 numbers has 22
// bits, of which 127 p may lose up to five, and quotients lie as near as 2^-31
// to a tie: codes whose quotient is within its error of one (one in 2^15) are put
// right by their distance from 127 p, which is a number, and by what was lost
// (2048 x 4096 fp16 13.3 to 14.1 us, all codes put right so 15.5).
struct Coder {
  float up, top, inv;
  bool some;

  MHC_DEV explicit Coder(float t) {
    const uint32_t e = min(max(__builtin_bit_cast(uint32_t, t) >> 23, 1u), 253u);
    up = __builtin_bit_cast(float, (254u - e) << 23);
    some = t > 0.f && t < __builtin_inff();
    top = some ? t * up : 1.f;
    inv = 1.f / top;
  }
  MHC_DEV float quotient(float p) const {
    const float a = 127.f * (p * up), q = a * inv;
    return fmaf(fmaf(-q, top, a), inv, q);
  }
  MHC_DEV int code(float p) const { return some ? (int)rintf(quotient(p)) : 0; }
  // the same, and how far a quotient is from its code at most: of a long product the code may not be the nearest if that is near 1/2
  static constexpr float kUnsure = 0.5f - 0x1p-16f;
  MHC_DEV int code(float p, float& far) const {
    const float q = quotient(p), c = rintf(q);
    far = fmaxf(far, fabsf(q - c));
    return some ? (int)c : 0;
  }
  MHC_DEV int sure_code(float p) const {
    const float u = p * up, a = 127.f * u, lost = fmaf(127.f, u, -a);
    float c = rintf(quotient(p));
    const float d = fmaf(-c, top, a), past = (fabsf(d) - 0.5f * top) + (d < 0.f ? -lost : lost);  // the middle between c and its neighbour
    if (past > 0.f || (past == 0.f && ((int)c & 1) != 0)) c += d < 0.f ? -1.f : 1.f;
    return some ? (int)c : 0;
  }
  static MHC_DEV float scale(float t, float s) { return t < __builtin_inff() ? t * s / 127.f : __builtin_nanf(""); }
};

// whether rows of T in this mode are such products
template <typename T, int MODE> constexpr bool kLong = MODE == kCodes && __is_same(T, _Float16);

template <bool WHOLE, bool LONG, int V>
MHC_DEV void put_codes(int8_t* p, const Coder& c, const float (&v)[V], int left) {
  uint32_t w[V / 4];
  const auto each = [&](auto code) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k)
      w[k] = (uint32_t)(code(v[4 * k]) & 255) | (uint32_t)(code(v[4 * k + 1]) & 255) << 8 | (uint32_t)(code(v[4 * k + 2]) & 255) << 16 |
             (uint32_t)code(v[4 * k + 3]) << 24;
  };
  if constexpr (LONG) {
    float far = 0.f;
    each([&](float z) { return c.code(z, far); });
    if (far > Coder::kUnsure) [[unlikely]] each([&](float z) { return c.sure_code(z); });
  } else {
    each([&](float z) { return c.code(z); });
  }
  if constexpr (WHOLE) {
    __builtin_memcpy(p, w, V);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) p[k] = (int8_t)(w[k / 4] >> (8 * (k % 4)));
  }
}

// the weights of a vector's elements
template <bool WHOLE, typename T, int V>
MHC_DEV void weights_of(const void* w, bool f32, int64_t n, int left, float (&v)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 1.f;
  } else if (f32) {
    gemm::take<WHOLE>(static_cast<const float*>(w) + n, v, left);
  } else if constexpr (sizeof(T) == 2) {
    gemm::take<WHOLE>(static_cast<const T*>(w) + n, v, left);
  }
}

// s of a row from its sum of squares, over `by`, which is 1.  Squares past fp32's
// range are summed once more, of values times a power of two that brings the
// row's largest to 1, and that is `by` (sum(k) gives the sum for values times k,
// largest() their largest magnitude).
template <typename Sum, typename Largest>
MHC_DEV float factor_of(float squares, int C, float eps, float& by, Sum sum, Largest largest) {
  by = 1.f;
  if (squares < __builtin_inff()) return 1.f / sqrtf(squares / (float)C + eps);
  const float top = largest();
  if (!(top < __builtin_inff())) return top == __builtin_inff() ? 0.f : top;
  by = __builtin_bit_cast(float, (254u - min(__builtin_bit_cast(uint32_t, top) >> 23, 253u)) << 23);
  return 1.f / sqrtf(sum(by) / (float)C + eps * by * by);
}

// --------------------------------------------------------------------------
// Rows that registers hold
// --------------------------------------------------------------------------

// A row in the registers of THREADS threads (a wave, and then four rows a
// workgroup, or a workgroup): NV vectors each, and the C % V elements after the
// last whole vector one for each of the first threads.  Threads past the last
// vector read it once more (a load under a condition would wait for itself) and
// count it as zeros.
template <typename T, int THREADS, int NV>
struct Held {
  static constexpr int V = kV<T>, kRows = THREADS == kWave ? 4 : 1, kBlock = THREADS * kRows;
  int tid, vecs, tail, C;
  bool on_tail;

  MHC_DEV explicit Held(int C_) : C(C_) {
    tid = threadIdx.x % THREADS;
    vecs = C / V;
    tail = vecs * V + tid;
    on_tail = tail < C;
  }
  MHC_DEV int vec(int i) const { return i * THREADS + tid; }
  MHC_DEV bool has(int i) const { return vec(i) < vecs; }

  template <typename S>
  MHC_DEV void load(const S* p, float (&z)[NV][V], float& last) const {
    if (vecs > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) gemm::take<true>(p + min(vec(i), vecs - 1) * V, z[i], V);
    }
    last = on_tail ? load1(p + tail) : 0.f;
  }
  template <typename S>
  MHC_DEV void store(S* p, const float (&z)[NV][V], float last) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (has(i)) gemm::put<true>(p + vec(i) * V, z[i], V);
    if (on_tail) store1(p + tail, last);
  }
  // zeros in the place of vectors that are not there
  MHC_DEV void clear(float (&z)[NV][V]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) z[i][k] = has(i) ? z[i][k] : 0.f;
  }
  MHC_DEV void load_weights(const void* w, bool f32, float (&z)[NV][V], float& last) const {
    if (w == nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) z[i][k] = 1.f;
      last = 1.f;
    } else if (f32) {
      load_cached(static_cast<const float*>(w), z, last);
    } else if constexpr (sizeof(T) == 2) {
      load_cached(static_cast<const T*>(w), z, last);
    }
  }
  // (every row reads the weights)
  template <typename S>
  MHC_DEV void load_cached(const S* p, float (&z)[NV][V], float& last) const {
    if (vecs > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Vec<S, V> r;
        __builtin_memcpy(r.w, p + min(vec(i), vecs - 1) * V, sizeof(r.w));
#pragma unroll
        for (int k = 0; k < V; ++k) z[i][k] = r.get(k);
      }
    }
    last = on_tail ? load1(p + tail) : 0.f;
  }
};

template <typename T, int MODE, int THREADS, int NV>
__global__ __launch_bounds__((Held<T, THREADS, NV>::kBlock)) void norm_held_kernel(const NormArgs a, int w_f32) {
  using H = Held<T, THREADS, NV>;
  constexpr int V = H::V;
  __shared__ float lds[2][16];
  const H at(a.C);
  const int64_t t = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * H::kRows + (H::kRows > 1 ? threadIdx.x / THREADS : 0);
  if (t >= a.T) return;  // (a wave with its row)
  float z[NV][V] = {}, w[NV][V] = {}, z1, w1;
  at.load(static_cast<const T*>(a.x) + t * a.ldx, z, z1);
  if (a.r != nullptr) {
    float r[NV][V] = {}, r1;
    at.load(static_cast<const T*>(a.r) + t * a.ldr, r, r1);
    if constexpr (MODE != kCodesOnly) at.load_weights(a.w, w_f32, w, w1);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        z[i][k] += r[i][k];
        if constexpr (sizeof(T) == 2) z[i][k] = from16<T>(bits16<T>(z[i][k]));
      }
    z1 += r1;
    if constexpr (sizeof(T) == 2) z1 = from16<T>(bits16<T>(z1));
    at.store(static_cast<T*>(a.h) + t * a.C, z, z1);
  } else if constexpr (MODE != kCodesOnly) {
    at.load_weights(a.w, w_f32, w, w1);
  }
  at.clear(z);
  float s = 1.f, top = 0.f;
  if constexpr (MODE != kCodesOnly) {
    const auto squares = [&](float by) {
      float q = z1 * by * (z1 * by);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) q = fmaf(z[i][k] * by, z[i][k] * by, q);
      return join_threads<THREADS>(q, SumOp{}, lds[0]);
    };
    float by;
    s = factor_of(squares(1.f), a.C, a.eps, by, squares, [&] {
      float m = fabsf(z1);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) m = LargerOp{}(m, fabsf(z[i][k]));
      return join_threads<THREADS>(m, LargerOp{}, lds[1]);
    });
    if constexpr (MODE == kPlain) {
      s *= by;
    } else if (by != 1.f) {  // (products with the weights may be past the range, too)
      z1 *= by;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) z[i][k] *= by;
    }
  }
  if constexpr (MODE == kPlain) {
    if (at.tid == 0 && a.rstd != nullptr) a.rstd[t] = s;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) z[i][k] = z[i][k] * s * w[i][k];
    at.store(static_cast<T*>(a.y) + t * a.C, z, z1 * s * w1);
  } else {
    if constexpr (MODE == kCodes) {
      z1 = at.on_tail ? z1 * w1 : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) z[i][k] = at.has(i) ? z[i][k] * w[i][k] : 0.f;  // (0 times a weight that is not finite)
    }
    top = fabsf(z1);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) top = LargerOp{}(top, fabsf(z[i][k]));
    top = join_threads<THREADS>(top, LargerOp{}, lds[1]);
    if (at.tid == 0) a.scales[t] = Coder::scale(top, s);
    const Coder coder(top);
    int8_t* const codes = static_cast<int8_t*>(a.y) + t * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at.has(i)) put_codes<true, kLong<T, MODE>>(codes + at.vec(i) * V, coder, z[i], V);
    if (at.on_tail) codes[at.tail] = (int8_t)(kLong<T, MODE> ? coder.sure_code(z1) : coder.code(z1));
  }
}

// --------------------------------------------------------------------------
// Rows of any length: a workgroup goes over a row twice
// --------------------------------------------------------------------------

template <typename T, int MODE>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(const NormArgs a, int w_f32) {
  constexpr int V = kV<T>;
  __shared__ float lds[kLongThreads / kWave];
  const int C = a.C, vecs = (C + V - 1) / V;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* row = static_cast<const T*>(a.x) + t * a.ldx;
    const auto each = [&](const T* from, auto&& use) {
      for (int v = threadIdx.x; v < vecs; v += kLongThreads) {
        const int left = min(V, C - v * V);
        float z[V];
        if (left == V) {
          gemm::take<true>(from + v * V, z, V);
          use(v * V, left, z, std::true_type{});
        } else {
          gemm::take<false>(from + v * V, z, left);
          use(v * V, left, z, std::false_type{});
        }
      }
    };
    float squares = 0.f, top = 0.f;
    T* const h = static_cast<T*>(a.h) + t * C;
    each(row, [&](int n, int left, float(&z)[V], auto whole) {
      constexpr bool W = decltype(whole)::value;
      if (a.r != nullptr) {
        float r[V];
        gemm::take<W>(static_cast<const T*>(a.r) + t * a.ldr + n, r, left);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          z[k] += r[k];
          if constexpr (sizeof(T) == 2) z[k] = from16<T>(bits16<T>(z[k]));
        }
        gemm::put<W>(h + n, z, left);
      }
      float w[V];
      if (MODE != kPlain) weights_of<W, T>(a.w, w_f32, n, left, w);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        squares = fmaf(z[k], z[k], squares);
        if (MODE != kPlain) top = LargerOp{}(top, fabsf(z[k] * w[k]));
      }
    });
    if (a.r != nullptr) row = h;  // (each thread reads what it wrote)
    float s = 1.f, by = 1.f;
    if constexpr (MODE != kCodesOnly) {
      squares = join_threads<kLongThreads>(squares, SumOp{}, lds);
      s = factor_of(
          squares, C, a.eps, by,
          [&](float by) {
            float q = 0.f;
            each(row, [&](int, int, float(&z)[V], auto) {
#pragma unroll
              for (int k = 0; k < V; ++k) q = fmaf(z[k] * by, z[k] * by, q);
            });
            return join_threads<kLongThreads>(q, SumOp{}, lds);
          },
          [&] {
            float m = 0.f;
            each(row, [&](int, int, float(&z)[V], auto) {
#pragma unroll
              for (int k = 0; k < V; ++k) m = LargerOp{}(m, fabsf(z[k]));
            });
            return join_threads<kLongThreads>(m, LargerOp{}, lds);
          });
      if constexpr (MODE == kPlain) {
        s *= by;
      } else if (by != 1.f) {  // (products with the weights may be past the range, too)
        top = 0.f;
        each(row, [&](int n, int left, float(&z)[V], auto whole) {
          float w[V];
          weights_of<decltype(whole)::value, T>(a.w, w_f32, n, left, w);
#pragma unroll
          for (int k = 0; k < V; ++k) top = LargerOp{}(top, fabsf(z[k] * by * w[k]));
        });
      }
    }
    if constexpr (MODE != kPlain) top = join_threads<kLongThreads>(top, LargerOp{}, lds);
    if (threadIdx.x == 0) {
      if (MODE == kPlain && a.rstd != nullptr) a.rstd[t] = s;
      if (MODE != kPlain) a.scales[t] = Coder::scale(top, s);
    }
    const Coder coder(top);
    each(row, [&](int n, int left, float(&z)[V], auto whole) {
      constexpr bool W = decltype(whole)::value;
      float w[V];
      weights_of<W, T>(a.w, w_f32, n, left, w);
      if constexpr (MODE == kPlain) {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] = z[k] * s * w[k];
        gemm::put<W>(static_cast<T*>(a.y) + t * C + n, z, left);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] = z[k] * by * w[k];
        put_codes<W, kLong<T, MODE>>(static_cast<int8_t*>(a.y) + t * C + n, coder, z, left);
      }
    });
  }
}

// --------------------------------------------------------------------------
// Gradients
// --------------------------------------------------------------------------

struct NormBwdArgs {
  const void* dy;
  const void* dh;  // or NULL
  const void* h;
  const float* rstd;
  const void* w;   // or NULL
  int64_t lddy, lddh, ldh;
  void* dx;        // [T, C], or NULL
  float* part;     // sums of dw, [workgroups, part_pitch], or NULL
  int64_t T;
  int C;
};

// A row of the sums of dw: C, and up to three more, so that every row is in whole vectors.
__host__ __device__ inline int64_t part_pitch(int64_t C) { return (C + 3) / 4 * 4; }

template <typename T>
__global__ __launch_bounds__(kLongThreads) void norm_bwd_long_kernel(const NormBwdArgs a, int w_f32) {
  constexpr int V = kV<T>;
  __shared__ float lds[kLongThreads / kWave];
  const int C = a.C, vecs = (C + V - 1) / V;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const float s = a.rstd[t];
    // g and n of a vector
    const auto each = [&](auto&& use) {
      for (int v = threadIdx.x; v < vecs; v += kLongThreads) {
        const int n = v * V, left = min(V, C - n);
        const auto one = [&](auto whole) {
          constexpr bool W = decltype(whole)::value;
          float g[V], h[V], w[V];
          gemm::take<W>(static_cast<const T*>(a.dy) + t * a.lddy + n, g, left);
          gemm::take<W>(static_cast<const T*>(a.h) + t * a.ldh + n, h, left);
          weights_of<W, T>(a.w, w_f32, n, left, w);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            g[k] *= w[k];
            h[k] *= s;
          }
          use(n, left, g, h, whole);
        };
        if (left == V) one(std::true_type{});
        else one(std::false_type{});
      }
    };
    float along = 0.f;
    each([&](int, int, float(&g)[V], float(&h)[V], auto) {
#pragma unroll
      for (int k = 0; k < V; ++k) along = fmaf(g[k], h[k], along);
    });
    along = join_threads<kLongThreads>(along, SumOp{}, lds) / (float)C;
    each([&](int n, int left, float(&g)[V], float(&h)[V], auto whole) {
      constexpr bool W = decltype(whole)::value;
      float d[V] = {};
      if (a.dh != nullptr) gemm::take<W>(static_cast<const T*>(a.dh) + t * a.lddh + n, d, left);
#pragma unroll
      for (int k = 0; k < V; ++k) d[k] = fmaf(s, g[k] - h[k] * along, d[k]);
      gemm::put<W>(static_cast<T*>(a.dx) + t * C + n, d, left);
    });
  }
}

// Rows that registers hold: dx, and this workgroup's sums of dw, to
// part[workgroup].  A workgroup takes rows in turn and keeps the weights and
// the sums in registers.
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__((Held<T, THREADS, NV>::kBlock)) void norm_bwd_held_kernel(const NormBwdArgs a, int w_f32) {
  using H = Held<T, THREADS, NV>;
  constexpr int V = H::V, kRows = H::kRows;
  __shared__ float lds[16];
  const H at(a.C);
  const int row = kRows > 1 ? threadIdx.x / THREADS : 0;
  float w[NV][V] = {}, w1 = 0.f, sum[NV][V] = {}, sum1 = 0.f;
  at.load_weights(a.w, w_f32, w, w1);
  for (int64_t t = (int64_t)blockIdx.x * kRows + row; t < a.T; t += (int64_t)gridDim.x * kRows) {
    float g[NV][V] = {}, n[NV][V] = {}, d[NV][V] = {}, g1, n1, d1 = 0.f;
    at.load(static_cast<const T*>(a.dy) + t * a.lddy, g, g1);
    at.load(static_cast<const T*>(a.h) + t * a.ldh, n, n1);
    if (a.dh != nullptr && a.dx != nullptr) at.load(static_cast<const T*>(a.dh) + t * a.lddh, d, d1);
    const float s = a.rstd[t];
    float along = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        n[i][k] *= s;
        const float dn = at.has(i) ? g[i][k] * n[i][k] : 0.f;  // dy n, of which dw is the sum over rows and along over columns, times w
        sum[i][k] += dn;
        along = at.has(i) ? fmaf(dn, w[i][k], along) : along;
        g[i][k] *= w[i][k];
      }
    n1 *= s;
    sum1 = fmaf(g1, n1, sum1);
    g1 *= w1;
    if (at.on_tail) along = fmaf(g1, n1, along);
    if (a.dx == nullptr) continue;
    along = join_threads<THREADS>(along, SumOp{}, lds) / (float)a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) d[i][k] = fmaf(s, g[i][k] - n[i][k] * along, d[i][k]);
    at.store(static_cast<T*>(a.dx) + t * a.C, d, fmaf(s, g1 - n1 * along, d1));
  }
  if (a.part == nullptr) return;
  float* const part = a.part + blockIdx.x * part_pitch(a.C);
  if constexpr (kRows == 1) {
    at.store(part, sum, sum1);
  } else {
    __shared__ float sums[kRows][THREADS * NV * V + THREADS];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) sums[row][(i * V + k) * THREADS + at.tid] = sum[i][k];
    sums[row][NV * V * THREADS + at.tid] = sum1;
    __syncthreads();
    if (row != 0) return;
#pragma unroll
    for (int q = 1; q < kRows; ++q) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) sum[i][k] += sums[q][(i * V + k) * THREADS + at.tid];
      sum1 += sums[q][NV * V * THREADS + at.tid];
    }
    at.store(part, sum, sum1);
  }
}

constexpr int kDwCols = 64 * 8;  // columns of a workgroup of norm_dw_kernel

int dw_rows(int64_t T, int C) { return (int)std::max<int64_t>(16, ceil_div(T * ceil_div(C, kDwCols), 4 * device_cu_count())); }

// sums of dy n over a workgroup's rows, to part[block of rows][C]: for rows too long to be held by norm_bwd_kernel
template <typename T>
__global__ __launch_bounds__(256) void norm_dw_kernel(const NormBwdArgs a, int rows, uint32_t wide) {
  __shared__ float lds[4][kDwCols];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t block = blockIdx.x / wide;
  const int n0 = (int)(blockIdx.x % wide) * kDwCols, n = n0 + lane * 8, left = min(8, a.C - n);
  const int64_t t0 = (int64_t)block * rows, t1 = min(t0 + rows, a.T);
  float sum[8] = {};
  if (left > 0) {
    for (int64_t t = t0 + wave; t < t1; t += 4) {
      float g[8], h[8];
      if (left == 8) {
        gemm::take<true>(static_cast<const T*>(a.dy) + t * a.lddy + n, g, 8);
        gemm::take<true>(static_cast<const T*>(a.h) + t * a.ldh + n, h, 8);
      } else {
        gemm::take<false>(static_cast<const T*>(a.dy) + t * a.lddy + n, g, left);
        gemm::take<false>(static_cast<const T*>(a.h) + t * a.ldh + n, h, left);
      }
      const float s = a.rstd[t];
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] = fmaf(g[k], h[k] * s, sum[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) lds[wave][lane * 8 + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < kDwCols; c += 256)
    if (n0 + c < a.C) a.part[block * part_pitch(a.C) + n0 + c] = (lds[0][c] + lds[1][c]) + (lds[2][c] + lds[3][c]);
}

// dw from the rows of its sums: sixteen columns a workgroup, each of 64 groups
// of threads with every 64th row, eight of them under way, joined in order.
constexpr int kJoinCols = 4, kJoinParts = 64;

template <typename W>
__global__ __launch_bounds__(kJoinCols* kJoinParts) void norm_dw_join_kernel(const float* part, W* dw, int rows, int C) {
  __shared__ f32x4 lds[kJoinParts][kJoinCols];
  const int col = threadIdx.x % kJoinCols, q = threadIdx.x / kJoinCols;
  const int64_t pitch = part_pitch(C);
  const int c = (blockIdx.x * kJoinCols + col) * 4;
  const float* const p = part + min((int64_t)c, pitch - 4);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int r = q; r < rows; r += 8 * kJoinParts) {
    f32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const f32x4*>(p + min(r + k * kJoinParts, rows - 1) * pitch);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (r + k * kJoinParts < rows) s += v[k];
  }
  lds[q][col] = s;
  __syncthreads();
  if (threadIdx.x >= kJoinCols * 4) return;  // a thread for each column
  const float* const mine = reinterpret_cast<const float*>(lds) + threadIdx.x;
  const int n = blockIdx.x * kJoinCols * 4 + threadIdx.x;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kJoinParts; ++k) sum += mine[k * kJoinCols * 4];
  if (n < C) store1(dw + n, sum);
}

// codes times their row's scale, eight a thread
template <typename O, bool WHOLE>
MHC_DEV void values_of(const int8_t* codes, float scale, O* out, int left) {
  float v[8];
  if constexpr (WHOLE) {
    int8_t c[8];
    __builtin_memcpy(c, codes, 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)c[k] * scale;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? (float)codes[k] * scale : 0.f;
  }
  gemm::put<WHOLE>(out, v, left);
}

template <typename O>
__global__ __launch_bounds__(256) void values_kernel(const int8_t* codes, int64_t ld, const float* scales, O* out, int64_t T, int C, uint32_t groups) {
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < T * groups; at += (int64_t)gridDim.x * 256) {
    const int64_t t = at / groups;
    const int n = (int)(at % groups) * 8, left = min(8, C - n);
    if (left == 8) values_of<O, true>(codes + t * ld + n, scales[t], out + t * C + n, 8);
    else values_of<O, false>(codes + t * ld + n, scales[t], out + t * C + n, left);
  }
}

template <typename O>
int run_values(const int8_t* codes, int64_t ld, const float* scales, void* out, int64_t T, int C, hipStream_t s) {
  const uint32_t groups = (uint32_t)ceil_div(C, 8);
  const dim3 grid((unsigned)std::min(ceil_div(T * groups, 256), (int64_t)device_cu_count() * 32));
  hipLaunchKernelGGL((values_kernel<O>), grid, dim3(256), 0, s, codes, ld, scales, static_cast<O*>(out), T, C, groups);
  MHC_CHECK_LAUNCH("values_kernel");
  return MHC_OK;
}

unsigned grid_of(int64_t T) { return (unsigned)std::min<int64_t>(T, kMaxRows); }

// How a row of C elements is held: by how many threads, and how many vectors
// each; none: it is not.
struct Hold {
  int threads, vecs;
};

// A wave for a row as long as it has two vectors a lane (67 MB of rows and
// residuals of bf16: 512 wide 44.5 us, with 256 threads 93; 1024 wide 44 and 57;
// but 2048 wide 47.5 with four vectors a lane, and 44), then a workgroup (4096
// wide 44, in two passes 102; 32768 wide 53 and 82).
Hold hold_of(int C, int dtype) {
  const int vecs = std::max(1, C * gemm::elem_bytes(dtype) / 16);
  if (vecs <= 64) return {64, 1};
  if (vecs <= 128) return {64, 2};
  if (vecs <= 256) return {256, 1};
  if (vecs <= 512) return {256, 2};
  if (vecs <= 1024) return {256, 4};
  if (vecs <= 2048) return {1024, 2};
  if (vecs <= 4096) return {1024, 4};
  return {0, 0};
}

// The same in the backward, which has five vectors of numbers for each of a
// row's, and a row of sums of dw for each workgroup (three times as many bytes
// read, and dw: 2048 wide 56 us, with 256 threads 62; 8192 wide 57, with 256
// threads 63, in two passes 115; 16384 wide 65, with 1024 threads 67).
Hold bwd_hold_of(int C, int dtype) {
  const int vecs = std::max(1, C * gemm::elem_bytes(dtype) / 16);
  if (vecs <= 64) return {64, 1};
  if (vecs <= 128) return {64, 2};
  if (vecs <= 256) return {64, 4};
  if (vecs <= 512) return {256, 2};
  if (vecs <= 1024) return {512, 2};
  if (vecs <= 2048) return {512, 4};
  return {0, 0};
}

template <int THREADS, int VECS>
struct HoldOf {
  static constexpr int kThreads = THREADS, kVecs = VECS;
  static bool is(const Hold& h) { return h.threads == THREADS && h.vecs == VECS; }
};

// f(HoldOf<...>{}) for the one of the list that h is
template <typename F>
int with_hold(const Hold&, F) { return MHC_OK; }
template <typename H, typename... Hs, typename F>
int with_hold(const Hold& h, F f) {
  if (H::is(h)) return f(H{});
  return with_hold<Hs...>(h, f);
}

template <typename T, int MODE>
int run_norm(const NormArgs& a, int w_f32, hipStream_t s) {
  const Hold hold = hold_of(a.C, dtype_code<T>());
  if (hold.threads > 0) {
    return with_hold<HoldOf<64, 1>, HoldOf<64, 2>, HoldOf<256, 1>, HoldOf<256, 2>, HoldOf<256, 4>, HoldOf<1024, 2>, HoldOf<1024, 4>>(
        hold, [&](auto of) {
          using O = decltype(of);
          using H = Held<T, O::kThreads, O::kVecs>;
          const int64_t groups = ceil_div(a.T, H::kRows);  // (in two dimensions: a launch has fewer than 2^32 threads in one)
          hipLaunchKernelGGL((norm_held_kernel<T, MODE, O::kThreads, O::kVecs>), dim3(grid_of(groups), (unsigned)ceil_div(groups, kMaxRows)), dim3(H::kBlock), 0, s, a, w_f32);
          MHC_CHECK_LAUNCH("norm_held_kernel");
          return (int)MHC_OK;
        });
  }
  hipLaunchKernelGGL((norm_long_kernel<T, MODE>), dim3(grid_of(a.T)), dim3(kLongThreads), 0, s, a, w_f32);
  MHC_CHECK_LAUNCH("norm_long_kernel");
  return MHC_OK;
}

template <int MODE>
int run_norm(const NormArgs& a, int dtype, int w_f32, hipStream_t s) {
  if (dtype == kF32) return run_norm<float, MODE>(a, w_f32, s);
  if (dtype == kBF16) return run_norm<__bf16, MODE>(a, w_f32, s);
  return run_norm<_Float16, MODE>(a, w_f32, s);
}

template <typename F>
int with_bwd_hold(const Hold& h, F f) {
  return with_hold<HoldOf<64, 1>, HoldOf<64, 2>, HoldOf<64, 4>, HoldOf<256, 2>, HoldOf<512, 2>, HoldOf<512, 4>>(h, f);
}

// Workgroups of norm_bwd_held_kernel: up to four of a CU, as many as it has room
// for (more would start when the others are done: 4096 wide 66 us for 58), with
// four rows each if there are so many.
template <typename T>
int64_t bwd_blocks(const Hold& h, int64_t rows_) {
  const int fit = with_bwd_hold(h, [](auto of) {
    using O = decltype(of);
    return occupancy_blocks(reinterpret_cast<const void*>(norm_bwd_held_kernel<T, O::kThreads, O::kVecs>), Held<T, O::kThreads, O::kVecs>::kBlock, 0);
  });
  const int64_t cus = device_cu_count(), most = cus * std::min(4, std::max(1, fit)), rows = h.threads == 64 ? ceil_div(rows_, 4) : rows_;
  return std::min(std::min(rows, most), std::max(cus, ceil_div(rows, 4)));
}

int64_t bwd_blocks(const Hold& h, int64_t T, int dtype) {
  return dtype == kF32 ? bwd_blocks<float>(h, T) : dtype == kBF16 ? bwd_blocks<__bf16>(h, T) : bwd_blocks<_Float16>(h, T);
}

// rows of the sums of dw
int64_t part_rows(int64_t T, int C, int dtype) {
  const Hold hold = bwd_hold_of(C, dtype);
  return hold.threads > 0 ? bwd_blocks(hold, T, dtype) : ceil_div(T, dw_rows(T, C));
}

template <typename T>
int run_dw_join(const float* part, void* dw, int w_f32, int64_t rows, int64_t C, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(C, kJoinCols * 4)), block(kJoinCols * kJoinParts);
  if (w_f32) hipLaunchKernelGGL((norm_dw_join_kernel<float>), grid, block, 0, s, part, static_cast<float*>(dw), (int)rows, (int)C);
  else hipLaunchKernelGGL((norm_dw_join_kernel<T>), grid, block, 0, s, part, static_cast<T*>(dw), (int)rows, (int)C);
  MHC_CHECK_LAUNCH("norm_dw_join_kernel");
  return MHC_OK;
}

template <typename T>
int run_bwd(NormBwdArgs a, int w_f32, void* dw, hipStream_t s) {
  if (dw == nullptr) a.part = nullptr;
  const Hold hold = bwd_hold_of(a.C, dtype_code<T>());
  const int64_t blocks = part_rows(a.T, a.C, dtype_code<T>());
  if (hold.threads > 0) {
    const int rc = with_bwd_hold(hold, [&](auto of) {
      using O = decltype(of);
      using H = Held<T, O::kThreads, O::kVecs>;
      hipLaunchKernelGGL((norm_bwd_held_kernel<T, O::kThreads, O::kVecs>), dim3((unsigned)blocks), dim3(H::kBlock), 0, s, a, w_f32);
      MHC_CHECK_LAUNCH("norm_bwd_held_kernel");
      return (int)MHC_OK;
    });
    return rc != MHC_OK || dw == nullptr ? rc : run_dw_join<T>(a.part, dw, w_f32, blocks, a.C, s);
  }
  if (a.dx != nullptr) {
    hipLaunchKernelGGL((norm_bwd_long_kernel<T>), dim3(grid_of(a.T)), dim3(kLongThreads), 0, s, a, w_f32);
    MHC_CHECK_LAUNCH("norm_bwd_long_kernel");
  }
  if (dw == nullptr) return MHC_OK;
  const uint32_t wide = (uint32_t)ceil_div(a.C, kDwCols);
  hipLaunchKernelGGL((norm_dw_kernel<T>), dim3(wide * (uint32_t)blocks), dim3(256), 0, s, a, dw_rows(a.T, a.C), wide);
  MHC_CHECK_LAUNCH("norm_dw_kernel");
  return run_dw_join<T>(a.part, dw, w_f32, blocks, a.C, s);
}

int check_shape(int64_t T, int64_t C, int dtype) {
  MHC_CHECK_ARG(T >= 0 && C >= 1, "T must be >= 0 and C >= 1 (got %lld, %lld)", (long long)T, (long long)C);
  MHC_CHECK_ARG(C < ((int64_t)1 << 24), "C must be below 2^24 (got %lld)", (long long)C);  // (vectors of a row are counted in 32 bits)
  MHC_CHECK_ARG(dtype == kF32 || dtype == kBF16 || dtype == kF16, "unsupported dtype %d", dtype);
  return MHC_OK;
}

int check_norm(const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w, int w_dtype, const void* h, int64_t T, int64_t C,
               int dtype, float eps) {
  if (const int rc = check_shape(T, C, dtype)) return rc;
  MHC_CHECK_ARG(w == nullptr || w_dtype == dtype || w_dtype == kF32, "w_dtype must be the rows' or fp32 (got %d)", w_dtype);
  MHC_CHECK_ARG(eps > 0.f && eps < __builtin_inff(), "eps must be positive (got %g)", (double)eps);
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(x != nullptr && (r == nullptr || h != nullptr), "null pointer");
  MHC_CHECK_ARG((ldx >= C || T == 1) && (r == nullptr || ldr >= C || T == 1), "ldx and ldr must be at least C");
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

extern "C" int mhc_add_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, void* h,
                                    void* y, float* rstd, int64_t T, int64_t C, int dtype, float eps, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_norm(x, ldx, residual, ldr, w, w_dtype, h, T, C, dtype, eps)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(y != nullptr, "null pointer");
  const NormArgs a = {x, residual, w, ldx, ldr, h, y, nullptr, rstd, T, (int)C, eps};
  return run_norm<kPlain>(a, dtype, w_dtype == kF32, static_cast<hipStream_t>(stream));
}

extern "C" int mhc_add_rms_norm_int8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, void* h,
                                     int8_t* codes, float* scales, int64_t T, int64_t C, int dtype, float eps, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_norm(x, ldx, residual, ldr, w, w_dtype, h, T, C, dtype, eps)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(codes != nullptr && scales != nullptr, "null pointer");
  const NormArgs a = {x, residual, w, ldx, ldr, h, codes, scales, nullptr, T, (int)C, eps};
  return run_norm<kCodes>(a, dtype, w_dtype == kF32, static_cast<hipStream_t>(stream));
}

extern "C" int mhc_quantize_int8(const void* x, int64_t ldx, int8_t* codes, float* scales, int64_t T, int64_t C, int dtype, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(T, C, dtype)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(x != nullptr && codes != nullptr && scales != nullptr, "null pointer");
  MHC_CHECK_ARG(ldx >= C || T == 1, "ldx must be at least C");
  const NormArgs a = {x, nullptr, nullptr, ldx, 0, nullptr, codes, scales, nullptr, T, (int)C, 1.f};
  return run_norm<kCodesOnly>(a, dtype, 0, static_cast<hipStream_t>(stream));
}

extern "C" int mhc_dequantize_int8(const int8_t* codes, int64_t ld, const float* scales, void* out, int out_dtype, int64_t T, int64_t C,
                                   void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(T, C, out_dtype)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(codes != nullptr && scales != nullptr && out != nullptr, "null pointer");
  MHC_CHECK_ARG(ld >= C || T == 1, "ld must be at least C");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (out_dtype == kF32) return run_values<float>(codes, ld, scales, out, T, (int)C, s);
  if (out_dtype == kBF16) return run_values<__bf16>(codes, ld, scales, out, T, (int)C, s);
  return run_values<_Float16>(codes, ld, scales, out, T, (int)C, s);
}

extern "C" size_t mhc_add_rms_norm_bwd_workspace_bytes(int64_t T, int64_t C, int dtype) {
  if (T <= 0 || C <= 0 || C >= ((int64_t)1 << 24)) return 0;
  return (size_t)(mhc::part_rows(T, (int)C, dtype) * mhc::part_pitch(C)) * sizeof(float);
}

extern "C" int mhc_add_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh, const float* rstd,
                                    const void* w, int w_dtype, void* dx, void* dw, int64_t T, int64_t C, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(T, C, dtype)) return rc;
  MHC_CHECK_ARG(T > 0, "T must be > 0");
  MHC_CHECK_ARG((w == nullptr && dw == nullptr) || w_dtype == dtype || w_dtype == kF32, "w_dtype must be the rows' or fp32 (got %d)", w_dtype);
  MHC_CHECK_ARG(dy != nullptr && h != nullptr && rstd != nullptr, "null pointer");
  MHC_CHECK_ARG((lddy >= C && ldh >= C && (dh == nullptr || lddh >= C)) || T == 1, "rows must be at least C apart");
  MHC_CHECK_ARG(dw == nullptr || (workspace != nullptr && workspace_bytes >= mhc_add_rms_norm_bwd_workspace_bytes(T, C, dtype)),
                "workspace too small");
  MHC_CHECK_ARG(aligned(workspace, 16), "workspace must be 16-byte aligned");
  if (dx == nullptr && dw == nullptr) return MHC_OK;
  const NormBwdArgs a = {dy, dh, h, rstd, w, lddy, lddh, ldh, dx, static_cast<float*>(workspace), T, (int)C};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kF32) return run_bwd<float>(a, 1, dw, s);
  if (dtype == kBF16) return run_bwd<__bf16>(a, w_dtype == kF32, dw, s);
  return run_bwd<_Float16>(a, w_dtype == kF32, dw, s);
}
