// Matrix products out[m, n] = sum_k A(m, k) B(n, k) on MFMA with a fused
// epilogue (gfx950), for fp32, bf16 and fp16 operands.
//
// Each operand is either "k-major" (its k are contiguous: x and W of x W^T)
// or not (its rows are k: W of dz W, and both operands of dz^T x).
#pragma once

#include <cmath>
#include <type_traits>

#include "mhc_device.hpp"
#include "mhc_host.hpp"

namespace mhc {
namespace gemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // sixteen bytes that start at any element

// --------------------------------------------------------------------------
// Epilogue: out = act(sum + bias) + residual, and act' for a backward
// --------------------------------------------------------------------------

struct Epilogue {
  const void* bias;      // [N] of the operands' type, or NULL
  const void* residual;  // [M, N] of the output's type, or NULL
  void* out;             // [M, N]
  void* dact;            // [M, N] as DactOf has it, or NULL; act is not none then
  int act;               // MHC_ACT_*
  int out_f32;           // out and residual are fp32, else of the operands' type
};

struct Act {
  float y, d;
};

// FAST (16-bit operands): the hardware's exponential and reciprocal, which are
// good to 2^-22 of the value; else the library's exponential and a division.
template <bool FAST>
MHC_DEV float exp_of(float x) {
  return FAST ? __builtin_amdgcn_exp2f(x * 1.44269504f) : expf(x);
}
template <bool FAST>
MHC_DEV float sigmoid(float x) {
  const float d = 1.f + exp_of<FAST>(-x);
  return FAST ? __builtin_amdgcn_rcpf(d) : 1.f / d;
}

// Phi(z), with e = exp(-z^2 / 2), which the derivative needs too: Phi(-|z|) is e
// times a polynomial in t = 1 / (1 + 0.26 |z|), so that gelu keeps its value far
// below zero, where (1 + erf) / 2 loses it.  The nine coefficients are those of
// the least largest error of the value over |z| <= 14, 1.7e-8 of it (a linear
// program over a grid of z); their sum in fp32 is off by some 3e-7.
template <bool FAST>
MHC_DEV float normal_cdf(float z, float e) {
  constexpr float kC[] = {0.103756599f, 0.10306108f, 0.102696232f, 0.0524016619f, 0.157570824f, -0.14586091f, 0.246889755f, -0.150537908f, 0.0300226714f};
  const float u = 1.f + 0.26f * fabsf(z), t = FAST ? __builtin_amdgcn_rcpf(u) : 1.f / u;
  float r = kC[8];
#pragma unroll
  for (int k = 7; k >= 0; --k) r = fmaf(r, t, kC[k]);
  const float tail = e * t * r;
  return z < 0.f ? tail : 1.f - tail;
}

// act(z) and act'(z).  NaN goes through each of them, but for relu', which is 0
// wherever z is not above 0.
template <bool FAST, int ACT>
MHC_DEV Act activate(float z) {
  if constexpr (ACT == MHC_ACT_RELU) {
    return {z < 0.f ? 0.f : z, z > 0.f ? 1.f : 0.f};
  } else if constexpr (ACT == MHC_ACT_GELU) {
    const float e = exp_of<FAST>(-0.5f * z * z), p = normal_cdf<FAST>(z, e);
    return {z * p, p + z * e * 0.39894228f};
  } else if constexpr (ACT == MHC_ACT_GELU_TANH) {  // (1 + tanh u) / 2 is sigmoid(2 u)
    const float p = sigmoid<FAST>(1.59576912f * (z + 0.044715f * z * z * z));
    return {z * p, p + z * p * (1.f - p) * 1.59576912f * (1.f + 0.134145f * z * z)};
  } else {
    const float p = sigmoid<FAST>(z);
    return {z * p, p * (1.f + z * (1.f - p))};
  }
}

template <bool FAST, int ACT, int R, int V>
MHC_DEV void activate_each(float (&z)[R][V], float (&d)[R][V]) {
#pragma unroll
  for (int b = 0; b < R; ++b)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const Act a = activate<FAST, ACT>(z[b][k]);
      z[b][k] = a.y;
      d[b][k] = a.d;
    }
}

template <bool FAST, int R, int V>
MHC_DEV void activate_all(int act, float (&z)[R][V], float (&d)[R][V]) {
  switch (act) {
    case MHC_ACT_RELU: return activate_each<FAST, MHC_ACT_RELU>(z, d);
    case MHC_ACT_GELU: return activate_each<FAST, MHC_ACT_GELU>(z, d);
    case MHC_ACT_GELU_TANH: return activate_each<FAST, MHC_ACT_GELU_TANH>(z, d);
    case MHC_ACT_SILU: return activate_each<FAST, MHC_ACT_SILU>(z, d);
    default: return;
  }
}

// act'(z) as a backward reads it: fp32 for fp32 operands, else 16 bits.  All of
// the derivatives lie in [-0.13, 1.13], and most of fp16's codes are for numbers
// that they never are: with 2^-11 of the value, fp16 would add to the one
// rounding of dz.  From 1/32 on the code is fixed point in steps of 2^-15, below
// it has nine bits after the leading one, down to 2^-29 and evenly from there:
// the error is at most 2^-16, and 2^-10 of the value (a unit far below zero has
// a derivative of 1e-5 and less, and still its gradient), 0 and 1 are exact.
// Codes rise with the value from 16384 for 0; the largest is NaN.
template <typename T> struct DactOf { using Type = uint16_t; };
template <> struct DactOf<float> { using Type = float; };

constexpr uint32_t kDactZero = 16384, kDactNan = 0xffff;
constexpr uint32_t kDactEven = 25 << 9;     // code of 1/32: 24 powers of two of 512 codes, and what is below them
constexpr float kDactLeast = 0x1p-97f;      // 2^-29, the least with nine bits of its own, to the least normal number
constexpr uint32_t kDactFixed = kDactEven - 1024;  // fixed point counts 1/32 as 1024

MHC_DEV uint32_t dact_code(float d) {
  const float a = fabsf(d);
  const uint32_t low = (__builtin_bit_cast(uint32_t, a * kDactLeast) + 0x2000u) >> 14;  // (of NaN: far above the codes)
  const uint32_t high = (uint32_t)fmaf(a, 32768.f, (float)kDactFixed + 0.5f);
  const uint32_t c = !(a >= 0x1p-5f) ? low : high, sign = (uint32_t)(__builtin_bit_cast(int32_t, d) >> 31);
  return min((c ^ sign) + (kDactZero - sign), kDactNan);
}
MHC_DEV float dact_value(uint16_t q) {
  const int32_t c = (int32_t)q - (int32_t)kDactZero;
  const uint32_t a = (uint32_t)max(c, -c);
  const float low = __builtin_bit_cast(float, a << 14) * (1.f / kDactLeast);
  const float high = fmaf((float)a, 0x1p-15f, -(float)kDactFixed * 0x1p-15f);
  const float v = __builtin_copysignf(a < kDactEven ? low : high, __builtin_bit_cast(float, c));
  return q == kDactNan ? __builtin_nanf("") : v;
}
MHC_DEV float dact_value(float d) { return d; }

// Eight values to or from p, which starts anywhere, as 16-byte vectors (the
// hardware takes them at any element), or (not WHOLE) those before `left` one
// by one; or one value.  Callers branch on WHOLE around all of their loads:
// a load under a condition of its own would be waited for there.
template <bool WHOLE, typename O, int V>
MHC_DEV void put(O* p, const float (&z)[V], int left) {
  if constexpr (V == 1) {
    if constexpr (__is_same(O, uint16_t)) *p = (uint16_t)dact_code(z[0]);
    else store1(p, z[0]);
  } else {
    uint32_t w[V * sizeof(O) / 4];
#pragma unroll
    for (int k = 0; k < (int)(V * sizeof(O) / 4); ++k) {
      if constexpr (sizeof(O) == 4) w[k] = __builtin_bit_cast(uint32_t, (float)z[k]);
      else if constexpr (__is_same(O, uint16_t)) w[k] = dact_code(z[2 * k]) | dact_code(z[2 * k + 1]) << 16;
      else w[k] = pack2<O>(z[2 * k], z[2 * k + 1]);
    }
    if constexpr (WHOLE) {
      __builtin_memcpy(p, w, V * sizeof(O));
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (k >= left) break;
        if constexpr (sizeof(O) == 4) p[k] = __builtin_bit_cast(O, w[k]);
        else p[k] = __builtin_bit_cast(O, (uint16_t)(w[k / 2] >> (16 * (k % 2))));
      }
    }
  }
}

template <bool WHOLE, typename O, int V>
MHC_DEV void take(const O* p, float (&z)[V], int left) {
  if constexpr (V == 1) {
    z[0] = load1(p);
  } else {
    Vec<O, V> r;
    if constexpr (WHOLE) {
#pragma unroll
      for (int k = 0; k < (int)(V * sizeof(O) / 16); ++k) {
        const u32x4 u = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p) + k);
        r.w[4 * k] = u.x, r.w[4 * k + 1] = u.y, r.w[4 * k + 2] = u.z, r.w[4 * k + 3] = u.w;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) z[k] = r.get(k);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) z[k] = k < left ? load1(p + k) : 0.f;
    }
  }
}

// act' as put() stored it
template <bool WHOLE, typename D, int V>
MHC_DEV void take_dact(const D* p, float (&z)[V], int left) {
  if constexpr (sizeof(D) == 4) {
    take<WHOLE>(p, z, left);
  } else if constexpr (WHOLE) {
    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = dact_value((uint16_t)(w[k / 2] >> (16 * (k % 2))));
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = k < left ? dact_value(p[k]) : 0.f;
  }
}

// The residuals of V outputs from column n on (those before `left`), of R rows
// `step` apart from row m on (of the last row past the end; zeros without a
// residual): all of them loaded before the first is used.
template <typename T, bool WHOLE, int V, int R>
MHC_DEV void residual_of(const Epilogue& e, int64_t m, int step, int64_t M, int64_t n, int64_t N, int left, float (&r)[R][V]) {
  if (e.residual == nullptr) {
#pragma unroll
    for (int b = 0; b < R; ++b)
#pragma unroll
      for (int k = 0; k < V; ++k) r[b][k] = 0.f;
  } else if (e.out_f32) {
#pragma unroll
    for (int b = 0; b < R; ++b) take<WHOLE>(static_cast<const float*>(e.residual) + min(m + b * step, M - 1) * N + n, r[b], left);
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int b = 0; b < R; ++b) take<WHOLE>(static_cast<const T*>(e.residual) + min(m + b * step, M - 1) * N + n, r[b], left);
  }
}

template <typename T, int V>
MHC_DEV void bias_of(const Epilogue& e, int64_t n, int left, float (&b)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) b[k] = e.bias != nullptr && k < left ? load1(static_cast<const T*>(e.bias) + n + k) : 0.f;
}

// The outputs of R rows `step` apart from row m on, V from column n on (those
// before `left`), from their sums.
template <typename T, bool WHOLE, int V, int R>
MHC_DEV void finish(const Epilogue& e, int64_t m, int step, int64_t M, int64_t n, int64_t N, int left, float (&z)[R][V],
                    const float (&bias)[V], const float (&residual)[R][V]) {
  float d[R][V];
#pragma unroll
  for (int b = 0; b < R; ++b)
#pragma unroll
    for (int k = 0; k < V; ++k) z[b][k] += bias[k];
  activate_all<sizeof(T) == 2>(e.act, z, d);
#pragma unroll
  for (int b = 0; b < R; ++b) {
    if (m + b * step >= M) break;
    const int64_t at = (m + b * step) * N + n;
    if (e.dact != nullptr) put<WHOLE>(static_cast<typename DactOf<T>::Type*>(e.dact) + at, d[b], left);
#pragma unroll
    for (int k = 0; k < V; ++k) z[b][k] += residual[b][k];
    if (e.out_f32) put<WHOLE>(static_cast<float*>(e.out) + at, z[b], left);
    else if constexpr (sizeof(T) == 2) put<WHOLE>(static_cast<T*>(e.out) + at, z[b], left);
  }
}

// --------------------------------------------------------------------------
// MFMA
// --------------------------------------------------------------------------

// Sixteen bytes of one row's k a lane: lane l has row l % 16 and the group
// l / 16 of the step's k.  Which k a place holds does not matter as long as
// both operands agree.
template <typename T>
MHC_DEV f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
    // (the vectors are cast whole: a bit cast of one element of a vector takes its first)
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[k], bf[k], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// --------------------------------------------------------------------------
// The tile kernel: BM x BN outputs a workgroup, WM x WN waves
// --------------------------------------------------------------------------

// An operand as it is stored: rows of `width` elements, `ld` elements apart.
// Rows start on four bytes, as the loads to LDS ask, and are a multiple of
// four bytes long, so that the end of the last one is the end of a word.
struct Operand {
  const void* p;
  int64_t ld, width;
};

// Offsets inside a tile, of up to 256 rows, stay below 2^31: rows are at most
// this far apart, or the tile has half as many of them (most_rows).
constexpr int64_t kMaxRowBytes = 1 << 23;

// Whether rows of `width` elements, `ld` apart, can be an Operand as they are.
inline bool in_words(const void* p, int64_t ld, int64_t width, int bytes) {
  return aligned(p, 4) && ld * bytes % 4 == 0 && width * bytes % 4 == 0 && ld * bytes <= kMaxRowBytes;
}

struct Product {
  Operand a, b;
  int64_t M, N, K;
  Epilogue e;
  int splits;   // of the reduction, each of kper k; more than one: `out` of the epilogue holds the sums of each
  int kper;     // a multiple of a stage
};

// LDS holds an operand's tile of a stage, 128 bytes of k for each index, in
// 16-byte chunks that the wave's loads put there directly.
//
// k-major: a row for each index, with eight chunks of k.  Chunk c of row r is
// at c ^ (r % 8), so that lanes that read the same chunk of 16 rows meet
// different banks.
//
// Otherwise: a row for each k, with chunks of the index.  16-bit operands are
// read with a transposing load (four k of one index a lane): its 16 lanes
// take 32 bytes of each of four rows, and chunk c of row k is at
// c ^ (2 (k % 4) + k & 8), which spreads the eight rows of half a wave over
// all banks (tiles of 64 have rows of half as many banks, two to a line:
// c ^ 2 (k % 4) ^ k & 8 / 4).  fp32 operands are read one by one, four groups of lanes from
// rows four apart: chunk c of row k is at c ^ 4 (k / 4 % 4).
template <typename T>
struct Stage {
  static constexpr int kE = 16 / (int)sizeof(T);  // elements of a chunk
  static constexpr int kK = 8 * kE;               // k of a stage
};

template <typename T, int R>
MHC_DEV int row_key(int k) {
  static_assert(R >= 64, "a row has more chunks than a key has values");
  if constexpr (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
  else return R >= 128 ? ((k & 3) << 1) | (k & 8) : ((k & 3) << 1) ^ ((k & 8) >> 2);
}

// Sixteen bytes a lane from memory to LDS, in the order of the lanes, without
// passing through registers; past the end of `rs` zeros are stored.  In
// assembly, since the compiler would wait for it before every LDS read.  The
// caller waits (wait_loads) before the barrier that hands the stage over.
MHC_DEV void load_to_lds(u32x4 rs, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "s"(lds));
}

// until at most N of the wave's loads are under way
template <int N>
MHC_DEV void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

MHC_DEV uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// One operand's side of a workgroup's tile: R indices from i0.
template <typename T, bool KM, int R, int WAVES>
struct Loader {
  using S = Stage<T>;
  static constexpr int kLoads = R * 128 / 1024 / WAVES;  // of a wave, each 64 chunks
  uint64_t base;
  int64_t left;       // bytes from base to the operand's end
  int64_t step;       // bytes of base from stage to stage
  uint32_t off[kLoads];
  uint32_t lds;       // of the wave's first chunk in a stage

  MHC_DEV void init(const Operand& o, int64_t i0, int64_t count, int64_t k0, int64_t k1, int wave, int lane, uint32_t lds0) {
    const int64_t ld = o.ld * (int64_t)sizeof(T);
    if constexpr (KM) {
      base = reinterpret_cast<uint64_t>(o.p) + (uint64_t)(i0 * ld + k0 * (int64_t)sizeof(T));
      left = (count - i0 - 1) * ld + (o.width - k0) * (int64_t)sizeof(T);
      step = 128;
    } else {
      base = reinterpret_cast<uint64_t>(o.p) + (uint64_t)(k0 * ld + i0 * (int64_t)sizeof(T));
      left = (k1 - k0 - 1) * ld + (o.width - i0) * (int64_t)sizeof(T);
      step = S::kK * ld;
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = (wave * kLoads + i) * 64 + lane;
      if constexpr (KM) {
        const int row = at >> 3;
        off[i] = (uint32_t)(row * ld) + (((at & 7) ^ (row & 7)) << 4);
      } else {
        constexpr int kC = R / S::kE;  // chunks of a row
        const int k = at / kC;
        off[i] = (uint32_t)(k * ld) + (((at % kC) ^ row_key<T, R>(k)) << 4);
      }
    }
    lds = lds0 + wave * kLoads * 1024;
  }

  // the stage at base; kleft: k from it to the end
  MHC_DEV void load(uint32_t stage, int kleft, int lane) const {
    // (offsets of the tile stay below 2^31, see kMaxRowBytes and most_rows)
    const uint32_t n = left <= 0 ? 0u : left > 0x80000000ll ? 0x80000000u : (uint32_t)left;
    const u32x4 rs = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, n, 0x00020000u};
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t v = off[i];
      if constexpr (KM) {  // in the last stage, chunks past the end of a row are the next row's
        if (kleft < S::kK && ((lane & 7) ^ (lane >> 3)) * S::kE >= kleft) v = 0xfffffff0u;
      }
      load_to_lds(rs, v, lds + stage + i * 1024);
    }
  }

  MHC_DEV void next() {
    base += (uint64_t)step;
    left -= step;
  }

  // Zeros after the last of the `kleft` k that a stage has, in the chunk that
  // they end in: what follows them in memory is the next row.  (Whole chunks
  // past the end were not loaded; for rows of k, whole rows.)
  static MHC_DEV void clear_end(char* stage, int kleft, int thread, int threads) {
    if constexpr (KM) {
      const int c = kleft / S::kE;
      for (int row = thread; row < R; row += threads) {
        T* const p = reinterpret_cast<T*>(stage + row * 128 + ((c ^ (row & 7)) << 4));
        for (int j = kleft % S::kE; j < S::kE; ++j) p[j] = (T)0;
      }
    }
  }
};

// A wave's fragments of one operand: J times 16 indices from w0 of a tile
// R indices wide.  Lane l has index l % 16 and the k of group l / 16.
template <typename T, bool KM, int R, int J>
struct Reader {
  using S = Stage<T>;
  int at[KM ? 2 : J];

  MHC_DEV void init(int w0, int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (KM) {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (w0 + r) * 128 + (((s * 4 + g) ^ (r & 7)) << 4);
    } else if constexpr (sizeof(T) == 2) {
      const int k = g * 8 + (r >> 2);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int col = w0 + j * 16 + (r & 3) * 4;
        at[j] = k * R * 2 + (((col >> 3) ^ row_key<T, R>(k)) << 4) + (col & 7) * 2;
      }
    } else {
      const int k = g * 4;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int col = w0 + j * 16 + r;
        at[j] = k * R * 4 + (((col >> 2) ^ row_key<T, R>(k)) << 4) + (col & 3) * 4;
      }
    }
  }

  // the fragment of step s (half a stage) and tile j
  MHC_DEV u32x4 get(const char* stage, int s, int j) const {
    if constexpr (KM) {
      return *reinterpret_cast<const u32x4*>(stage + at[s] + j * 2048);
    } else if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const char* const p = stage + at[j] + s * 32 * R * 2;
      // (32 k and 4 k further the key is the same)
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * R * 2));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      return u32x4{a.x, a.y, b.x, b.y};
    } else {
      u32x4 v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const uint32_t*>(stage + at[j] + (s * 16 + k) * R * 4);
      return v;
    }
  }
};

// A wave's fragments of half a stage, and their products.
template <int JM, int JN>
struct Fragments {
  u32x4 a[JM], b[JN];

  template <typename RA, typename RB>
  MHC_DEV void read(const RA& ra, const RB& rb, const char* sa, const char* sb, int s) {
#pragma unroll
    for (int j = 0; j < JN; ++j) b[j] = rb.get(sb, s, j);
#pragma unroll
    for (int j = 0; j < JM; ++j) a[j] = ra.get(sa, s, j);
  }

  template <typename T>
  MHC_DEV void multiply(f32x4 (&acc)[JN][JM]) const {
#pragma unroll
    for (int j = 0; j < JM; ++j)
#pragma unroll
      for (int i = 0; i < JN; ++i) acc[i][j] = mfma16<T>(b[i], a[j], acc[i][j]);
  }
};

// Spreads READS LDS reads evenly over PRODUCTS matrix instructions.
template <int READS, int PRODUCTS>
MHC_DEV void interleave() {
#pragma unroll
  for (int r = 0; r < READS; ++r) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    constexpr int kEach = PRODUCTS / READS > 0 ? PRODUCTS / READS : 1;
    __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
  }
}

// ROWS rows of 64 sums in LDS, as tile_kernel puts them there, to the outputs
// from (m0, n0) on: eight columns a lane, of two rows at a time.
template <typename T, int ROWS, bool WHOLE>
MHC_DEV void store_columns(const Epilogue& e, const char* sums, int lane, int64_t m0, int64_t M, int64_t n0, int64_t N, int left) {
  const int c = lane % 8 * 8;
  float bias[8];
  bias_of<T>(e, n0 + c, left, bias);
  for (int r0 = lane / 8; r0 < ROWS && m0 + r0 < M; r0 += 16) {
    float z[2][8], res[2][8];
    residual_of<T, WHOLE>(e, m0 + r0, 8, M, n0 + c, N, left, res);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = r0 + b * 8;
        const f32x4 u = *reinterpret_cast<const f32x4*>(sums + r * 256 + (((c / 4 + k) ^ (r % 16)) << 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) z[b][4 * k + j] = u[j];
      }
    finish<T, WHOLE>(e, m0 + r0, 8, M, n0 + c, N, left, z, bias, res);
  }
}

template <typename T, int ROWS>
MHC_DEV void store_rows(const Epilogue& e, const char* sums, int lane, int64_t m0, int64_t M, int64_t n0, int64_t N) {
  const int left = (int)max((int64_t)0, min((int64_t)8, N - n0 - lane % 8 * 8));
  if (left == 8) store_columns<T, ROWS, true>(e, sums, lane, m0, M, n0, N, left);
  else if (left > 0) store_columns<T, ROWS, false>(e, sums, lane, m0, M, n0, N, left);
}

// The same for those of the sums that are not kKeep, one by one: rarely used, so it is short.
constexpr uint32_t kKeep = 0x7fc5a5a5u;  // (a NaN: a sum that comes to it by itself is NaN in the outputs already)

template <typename T, int ROWS>
MHC_DEV void store_some(const Epilogue& e, const char* sums, int lane, int64_t m0, int64_t M, int64_t n0, int64_t N) {
  if (n0 + lane >= N) return;
  float bias[1];
  bias_of<T>(e, n0 + lane, 1, bias);
  for (int r = 0; r < ROWS && m0 + r < M; ++r) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(sums + r * 256 + (((lane / 4) ^ (r % 16)) << 4) + lane % 4 * 4);
    if (u == kKeep) continue;
    float z[1][1] = {{__builtin_bit_cast(float, u)}}, residual[1][1];
    residual_of<T, true>(e, m0 + r, 0, M, n0 + lane, N, 1, residual);
    finish<T, true>(e, m0 + r, 0, M, n0 + lane, N, 1, z, bias, residual);
  }
}

// A wave's JM x JN sums of 16 x 16, in registers, to the outputs from (m0, n0)
// on, through the workgroup's LDS (BYTES of it, free).  SOME: those that are not kKeep.
template <typename T, int JM, int JN, int WAVES, int BYTES, bool SOME = false>
MHC_DEV void store_tile(const Epilogue& e, char* smem, const f32x4 (&acc)[JN][JM], int64_t m0, int64_t M, int64_t n0, int64_t N, int wave,
                        int lane) {
  // The sums go through LDS, where each wave has room for up to 64 rows
  // of 64 columns, so that rows of the outputs are written as whole vectors of
  // consecutive lanes.  The 16-byte chunk c of row r is at c ^ (r % 16).
  constexpr int kFit = BYTES / (WAVES * 4096);  // sets of 16 rows that every wave has room for
  constexpr int kRound = JM >= 4 && kFit >= 4 ? 4 : JM >= 2 && kFit >= 2 ? 2 : 1, kRows = kRound * 16;
  static_assert(JN == 4 && JM % kRound == 0 && kFit >= 1, "64 columns a wave");
  char* const mine = smem + wave * kRows * 256;
  // (a round's sums have constant indices, and those of the first are gone before the second)
  int at = lane;
  asm volatile("" : "+v"(at));  // (or addresses of the outputs would be formed before the loop and held through it)
  const auto round = [&](auto first) {
    constexpr int h = decltype(first)::value;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRound; ++j)
#pragma unroll
      for (int i = 0; i < JN; ++i)
        *reinterpret_cast<f32x4*>(mine + (j * 16 + at % 16) * 256 + (((i * 4 + at / 16) ^ (at % 16)) << 4)) = acc[i][h + j];
    __syncthreads();
    const int64_t mh = m0 + h * 16;
    if constexpr (SOME) store_some<T, kRows>(e, mine, at, mh, M, n0, N);
    else store_rows<T, kRows>(e, mine, at, mh, M, n0, N);
  };
  static_assert(JM / kRound <= 2, "two rounds");
  round(std::integral_constant<int, 0>{});
  if constexpr (JM > kRound) round(std::integral_constant<int, kRound>{});
}

// The tile of a workgroup.  Workgroups go round the eight XCDs, each with an
// L2 of its own: one XCD takes a run of consecutive tiles, in bands of eight
// rows of tiles, so that its tiles share rows of A and B.
MHC_DEV void tile_of(uint32_t id, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  const uint32_t total = tm * tn, per = total / 8, more = total % 8, xcd = id % 8;
  const uint32_t t = xcd * per + min(xcd, more) + id / 8;
  const uint32_t band = t / (8 * tn), first = band * 8, rows = min(8u, tm - first);
  m = first + (t % (8 * tn)) % rows;
  n = (t % (8 * tn)) / rows;
}

// A workgroup's place: its tile, its part of the reduction, and its wave's corner of the tile.
template <int BM, int BN, int WM, int WN>
struct Place {
  int64_t m0, n0;
  int wm, wn, k0, k1, wave, lane;

  MHC_DEV Place(const Product& p, uint32_t tile, int split) {
    lane = threadIdx.x % kWave;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    uint32_t tm, tn;
    tile_of(tile, (uint32_t)ceil_div(p.M, BM), (uint32_t)ceil_div(p.N, BN), tm, tn);
    m0 = (int64_t)tm * BM;
    n0 = (int64_t)tn * BN;
    wm = wave / WN * (BM / WM);
    wn = wave % WN * (BN / WN);
    k0 = split * p.kper;
    k1 = min((int)p.K, k0 + p.kper);
  }
};

// The sums of a workgroup's tile.  (The first operand's index, n, runs over a
// lane's four values.)  Bound by the matrix instructions and, beside them, the
// LDS reads of the fragments: a wave of a 256 x 256 tile reads 24 KB for 64
// products of 16 x 16 x 32, 70 % of what LDS gives in their time (bf16 8192 x
// 4096 x 4096: x W^T 206 to 219 us from box to box, 1.25 to 1.33 PFLOP/s; a
// library's 178).  Smaller tiles read more for each product and serve where
// large ones would leave CUs idle; their stages are as long as their chain of
// wait, barrier, reads and products, which more stages under way don't shorten.
template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, int NS>
MHC_DEV void sum_tile(const Product& p, const Place<BM, BN, WM, WN>& at, char* smem, f32x4 (&acc)[BN / WN / 16][BM / WM / 16]) {
  using S = Stage<T>;
  constexpr int kWaves = WM * WN, JM = BM / WM / 16, JN = BN / WN / 16;
  constexpr int kA = BM * 128, kStage = kA + BN * 128;
  const int lane = at.lane;
  Loader<T, AK, BM, kWaves> la;
  Loader<T, BK, BN, kWaves> lb;
  constexpr int kLoads = decltype(la)::kLoads + decltype(lb)::kLoads;
  const uint32_t lds = lds_address(smem);
  la.init(p.a, at.m0, p.M, at.k0, at.k1, at.wave, lane, lds);
  lb.init(p.b, at.n0, p.N, at.k0, at.k1, at.wave, lane, lds + kA);
  Reader<T, AK, BM, JM> ra;
  Reader<T, BK, BN, JN> rb;
  ra.init(at.wm, lane);
  rb.init(at.wn, lane);
  // The fragments of half a stage are read while the products of the half
  // before are formed; in the middle of a stage its last reads are done, so
  // that the barrier there frees its place and hands over the next one.
  // NS stages are under way.  (Those past the end read nothing: every pass
  // issues the same number of loads.)
  int kleft = at.k1 - at.k0;
#pragma unroll
  for (int q = 0; q < NS; ++q) {
    la.load(q * kStage, kleft - q * S::kK, lane);
    lb.load(q * kStage, kleft - q * S::kK, lane);
    la.next();
    lb.next();
  }
  wait_loads<(NS - 1) * kLoads>();
  __syncthreads();
  const auto clear_end = [&](int stage, int left) {
    if (left <= 0 || left >= S::kK || left % S::kE == 0) return;
    la.clear_end(smem + stage, left, threadIdx.x, 64 * kWaves);
    lb.clear_end(smem + stage + kA, left, threadIdx.x, 64 * kWaves);
    __syncthreads();
  };
  int cur = 0;
  clear_end(cur, kleft);
  Fragments<JM, JN> f0, f1;
  f0.read(ra, rb, smem, smem + kA, 0);
  for (; kleft > 0; kleft -= S::kK) {
    f1.read(ra, rb, smem + cur, smem + cur + kA, 1);
    f0.template multiply<T>(acc);
    interleave<(JM * (AK ? 1 : S::kE / 4) + JN * (BK ? 1 : S::kE / 4)), JM * JN * (sizeof(T) == 4 ? 4 : 1)>();
    wait_loads<(NS - 2) * kLoads>();
    __syncthreads();
    la.load(cur, kleft - NS * S::kK, lane);
    lb.load(cur, kleft - NS * S::kK, lane);
    la.next();
    lb.next();
    cur = cur == (NS - 1) * kStage ? 0 : cur + kStage;
    clear_end(cur, kleft - S::kK);
    f0.read(ra, rb, smem + cur, smem + cur + kA, 0);
    f1.template multiply<T>(acc);
    interleave<(JM * (AK ? 1 : S::kE / 4) + JN * (BK ? 1 : S::kE / 4)), JM * JN * (sizeof(T) == 4 ? 4 : 1)>();
  }
  wait_loads<0>();  // (the last ones store zeros)
}

// --------------------------------------------------------------------------
// fp32 operands on the bf16 matrix instructions
// --------------------------------------------------------------------------

// Eight fp32 values, times kLift, as three bf16 values each: the leading eight
// bits of the value, of what is left and of what is left then.  Cut off and not
// rounded, they add up to the value exactly: the last bit of an fp32 value is
// 2^-149 or more, and of a bf16 one 2^-133 or more, which is why values are
// lifted (unlifted, a value around 2^-120 would keep 2^-13 of itself too
// little).  Lifted values past the range are infinite, and the second part of
// an infinity is NaN.
constexpr float kLift = 0x1p16f;

MHC_DEV void split8(const u32x4& lo, const u32x4& hi, u32x4 (&part)[3]) {
  const f32x4 flo = __builtin_bit_cast(f32x4, lo), fhi = __builtin_bit_cast(f32x4, hi);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t x[2], y[2], z[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float v = kLift * (w < 2 ? flo[2 * w + k] : fhi[2 * w - 4 + k]);
      x[k] = __builtin_bit_cast(uint32_t, v);
      const float r = v - __builtin_bit_cast(float, x[k] & 0xffff0000u);
      y[k] = __builtin_bit_cast(uint32_t, r);
      z[k] = __builtin_bit_cast(uint32_t, r - __builtin_bit_cast(float, y[k] & 0xffff0000u));
    }
    part[0][w] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302);
    part[1][w] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302);
    part[2][w] = __builtin_amdgcn_perm(z[1], z[0], 0x07060302);
  }
}

// sum_tile for fp32 with each product of two values as six of their parts.
// The three that are left out are below 2^-21 of it, and 2^-24 on average, so
// that the sums are as good as fp32's own (2048 x 2048 x 2048: 7.0e-7 of the
// result off float64, 8.1e-7 with fp32 instructions).  Six bf16 products take
// 3/8 of the time of one in fp32; the splits, on the vector unit, go on beside
// them in another wave (the lift is one of their 6.5 instructions for a value,
// and 5 % of the time).
template <bool AK, bool BK, int BM, int BN, int WM, int WN, int NS>
MHC_DEV void sum_tile_split(const Product& p, const Place<BM, BN, WM, WN>& at, char* smem, f32x4 (&acc)[BN / WN / 16][BM / WM / 16]) {
  using S = Stage<float>;
  constexpr int kWaves = WM * WN, JM = BM / WM / 16, JN = BN / WN / 16;
  constexpr int kA = BM * 128, kStage = kA + BN * 128;
  const int lane = at.lane;
  Loader<float, AK, BM, kWaves> la;
  Loader<float, BK, BN, kWaves> lb;
  constexpr int kLoads = decltype(la)::kLoads + decltype(lb)::kLoads;
  const uint32_t lds = lds_address(smem);
  la.init(p.a, at.m0, p.M, at.k0, at.k1, at.wave, lane, lds);
  lb.init(p.b, at.n0, p.N, at.k0, at.k1, at.wave, lane, lds + kA);
  Reader<float, AK, BM, JM> ra;
  Reader<float, BK, BN, JN> rb;
  ra.init(at.wm, lane);
  rb.init(at.wn, lane);
  int kleft = at.k1 - at.k0;
#pragma unroll
  for (int q = 0; q < NS - 1; ++q) {
    la.load(q * kStage, kleft - q * S::kK, lane);
    lb.load(q * kStage, kleft - q * S::kK, lane);
    la.next();
    lb.next();
  }
  int cur = 0, ahead = (NS - 1) * kStage;
  for (; kleft > 0; kleft -= S::kK) {
    wait_loads<(NS - 2) * kLoads>();
    __syncthreads();  // this stage is there, and nobody reads the one before any more
    la.load(ahead, kleft - (NS - 1) * S::kK, lane);
    lb.load(ahead, kleft - (NS - 1) * S::kK, lane);
    la.next();
    lb.next();
    char* const sa = smem + cur;
    char* const sb = sa + kA;
    if (kleft < S::kK && kleft % S::kE != 0) {
      la.clear_end(sa, kleft, threadIdx.x, 64 * kWaves);
      lb.clear_end(sb, kleft, threadIdx.x, 64 * kWaves);
      __syncthreads();
    }
    u32x4 b[JN][3];
#pragma unroll
    for (int i = 0; i < JN; ++i) split8(rb.get(sb, 0, i), rb.get(sb, 1, i), b[i]);
#pragma unroll
    for (int j = 0; j < JM; ++j) {
      u32x4 a[3];
      split8(ra.get(sa, 0, j), ra.get(sa, 1, j), a);
#pragma unroll
      for (int q = 0; q < 6; ++q) {  // the small ones first
        constexpr int kB[6] = {2, 0, 1, 1, 0, 0}, kAt[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int i = 0; i < JN; ++i) acc[i][j] = mfma16<__bf16>(b[i][kB[q]], a[kAt[q]], acc[i][j]);
      }
    }
    cur = cur == (NS - 1) * kStage ? 0 : cur + kStage;
    ahead = ahead == (NS - 1) * kStage ? 0 : ahead + kStage;
  }
  wait_loads<0>();
#pragma unroll
  for (int i = 0; i < JN; ++i)
#pragma unroll
    for (int j = 0; j < JM; ++j) acc[i][j] *= 1.f / (kLift * kLift);
}

// --------------------------------------------------------------------------
// The kernels of tiles
// --------------------------------------------------------------------------

// fp32 tiles of at least 64 x 128 are summed on the bf16 instructions (us in
// fp32, and so: 8192 x 4096 x 4096 in 256 x 256 1950 and 1370, 2048 x 2048 x 2048
// in 64 x 128 136 and 119, its backward in 128 x 128 268 and 200; a library's
// fp32 product takes 1800 for the first.  64 x 64 have too few products for each
// value that is split: 512 x 2048 x 2048 43 and 56).
template <typename T, int BN>
constexpr bool kSplit = sizeof(T) == 4 && BN > 64;

// LDS of a workgroup: its stages and, for sums on split values, a bit for each
// sum of a thread, in words, and one word for each wave.
template <typename T, int BM, int BN, int WM, int WN, int NS>
struct TileBytes {
  static constexpr int kStages = NS * (BM + BN) * 128, kThreads = 64 * WM * WN, kWords = BM * BN / kThreads / 32;
  static constexpr int kAll = kStages + (kSplit<T, BN> ? (kWords * kThreads + WM * WN) * 4 : 0);
};

// A tile of outputs, or (split) of one part of the reduction's sums.  Sums on
// split values that come out infinite or as NaN are formed once more with fp32
// instructions: their values or lifted sums were past the range (2^111, 2^95),
// or had an infinity, whose parts make NaN of everything.  The other sums of the tile stay as they are, so that a row's
// outputs do not depend on what other rows hold.
template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, int NS>
MHC_DEV void run_tile(const Product& p, char* smem, uint32_t tile, int split) {
  using B = TileBytes<T, BM, BN, WM, WN, NS>;
  constexpr int kWaves = WM * WN, JM = BM / WM / 16, JN = BN / WN / 16;
  const Place<BM, BN, WM, WN> at(p, tile, split);
  const int64_t m0 = at.m0 + at.wm, n0 = at.n0 + at.wn;
  Epilogue e = p.e;
  if (p.splits > 1) e.out = static_cast<float*>(e.out) + (int64_t)split * p.M * p.N;
  f32x4 acc[JN][JM] = {};
  if constexpr (!kSplit<T, BN>) {
    sum_tile<T, AK, BK, BM, BN, WM, WN, NS>(p, at, smem, acc);
    store_tile<T, JM, JN, kWaves, B::kStages>(e, smem, acc, m0, p.M, n0, p.N, at.wave, at.lane);
  } else {
    static_assert(B::kWords * 32 == JM * JN * 4);
    sum_tile_split<AK, BK, BM, BN, WM, WN, NS>(p, at, smem, acc);
    uint32_t* const marks = reinterpret_cast<uint32_t*>(smem + B::kStages);
    uint32_t* const found = marks + B::kWords * B::kThreads;
    const auto past = [](float v) { return !(fabsf(v) < __builtin_inff()); };
    bool one = false;
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int j = 0; j < JM; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) one |= past(acc[i][j][k]);
    int mine = 0;
    if (__ballot(one) != 0) {  // those of outputs that are there
      // bit 4 (i JM + j) + k of a thread is for acc[i][j][k], row j 16 + lane % 16, column i 16 + lane / 16 4 + k
      uint32_t mark[B::kWords] = {}, any = 0;
      const int rows = (int)min((int64_t)(JM * 16), p.M - m0) - at.lane % 16, cols = (int)min((int64_t)(JN * 16), p.N - n0) - at.lane / 16 * 4;
#pragma unroll
      for (int i = 0; i < JN; ++i)
#pragma unroll
        for (int j = 0; j < JM; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int bit = 4 * (i * JM + j) + k;
            if (past(acc[i][j][k]) && j * 16 < rows && i * 16 + k < cols) mark[bit / 32] |= 1u << bit % 32;
          }
#pragma unroll
      for (int w = 0; w < B::kWords; ++w) {
        marks[w * B::kThreads + threadIdx.x] = mark[w];
        any |= mark[w];
      }
      mine = __ballot(any != 0) != 0;
    }
    if (at.lane == 0) found[at.wave] = mine;
    __syncthreads();
    uint32_t again = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) again |= found[w];
    again = __builtin_amdgcn_readfirstlane(again);
    store_tile<T, JM, JN, kWaves, B::kStages>(e, smem, acc, m0, p.M, n0, p.N, at.wave, at.lane);
    if (!again) return;
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int j = 0; j < JM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();  // nobody reads the sums in LDS any more
    Place<BM, BN, WM, WN> once_more = at;
    asm volatile("" : "+v"(once_more.lane), "+s"(once_more.wave));  // (or registers would hold places from the first sums to these)
    sum_tile<T, AK, BK, BM, BN, WM, WN, NS>(p, once_more, smem, acc);  // (it waits for the wave's stores, too)
    uint32_t mark[B::kWords] = {};
    if (mine) {
#pragma unroll
      for (int w = 0; w < B::kWords; ++w) mark[w] = marks[w * B::kThreads + threadIdx.x];
    }
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int j = 0; j < JM; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int bit = 4 * (i * JM + j) + k;
          if (!(mark[bit / 32] >> bit % 32 & 1)) acc[i][j][k] = __builtin_bit_cast(float, kKeep);
        }
    store_tile<T, JM, JN, kWaves, B::kStages, true>(e, smem, acc, m0, p.M, n0, p.N, at.wave, at.lane);
  }
}

template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(const Product p) {
  __shared__ __attribute__((aligned(1024))) char smem[TileBytes<T, BM, BN, WM, WN, NS>::kAll];
  run_tile<T, AK, BK, BM, BN, WM, WN, NS>(p, smem, blockIdx.x, (int)blockIdx.y);
}

// Column sums of fp32 rows: 32 columns a workgroup, each column in eight parts
// (sixteen with 512 threads) that are joined in order.
constexpr int kSumCols = 32;

template <int THREADS, typename T>
MHC_DEV void sum_columns(float (*lds)[kSumCols], const float* part, T* db, int64_t rows, int64_t N, uint32_t block) {
  constexpr int kParts = THREADS / kSumCols;
  const int c = threadIdx.x % kSumCols, q = threadIdx.x / kSumCols;
  const int64_t n = (int64_t)block * kSumCols + c;
  float s = 0.f;
#pragma unroll 8
  for (int64_t b = q; b < rows; b += kParts) s += part[b * N + min(n, N - 1)];
  lds[q][c] = s;
  __syncthreads();
  if (q != 0 || n >= N) return;
#pragma unroll
  for (int k = 1; k < kParts; ++k) s += lds[k][c];
  store1(db + n, s);
}

// A backward's two products and the last sums of db, none of which needs
// another, as one launch: alone, neither product of a few hundred rows fills
// the card, and each launch is some 3 us of host time (backward of 1000 x 1100
// x 1536 fp32: 99 us in four launches, 65 in two; 64 x 1024 x 1024 bf16 19 and
// 14).  The longer reductions go first.
struct Pair {
  Product dx, dw;
  uint32_t dx0, dx_count, dw0, dw_count;  // the workgroups of each; those of db come last
  const float* part;
  void* db;
  int64_t part_rows, N;
};

template <typename T, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void pair_kernel(const Pair p) {
  __shared__ __attribute__((aligned(1024))) char smem[TileBytes<T, BM, BN, WM, WN, NS>::kAll];
  const uint32_t id = blockIdx.x;
  if (id - p.dx0 < p.dx_count) {
    const uint32_t at = id - p.dx0, tiles = p.dx_count / p.dx.splits;
    run_tile<T, true, false, BM, BN, WM, WN, NS>(p.dx, smem, at % tiles, (int)(at / tiles));
  } else if (id - p.dw0 < p.dw_count) {
    const uint32_t at = id - p.dw0, tiles = p.dw_count / p.dw.splits;
    run_tile<T, false, false, BM, BN, WM, WN, NS>(p.dw, smem, at % tiles, (int)(at / tiles));
  } else {
    sum_columns<64 * WM * WN>(reinterpret_cast<float(*)[kSumCols]>(smem), p.part, static_cast<T*>(p.db), p.part_rows, p.N,
                              id - p.dx_count - p.dw_count);
  }
}

// --------------------------------------------------------------------------
// Few rows: x W^T with M <= 64, bound by reading W
// --------------------------------------------------------------------------

// A workgroup has 16 NT rows of W and all of x, and its eight waves take
// stages of the k in turn: each wave has some of its own under way to LDS, so
// that memory is read in whole lines (fragments read straight from memory are
// half lines: 9.1 us for 16 rows of 4096 x 4096 bf16, 12.7 us for 32; so 6.0,
// 8.0).  No wave waits for another before the end, where their sums meet in
// LDS, in order.
constexpr int kFewWaves = 8;

// the waves' sums, in order, and the epilogue
template <typename T, int MT, int NT>
MHC_DEV void join_waves(const f32x4 (&acc)[NT][MT], float* sums, int M, int64_t n0, int64_t N, const Epilogue& e) {
  constexpr int kN = 16 * NT;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(sums + ((wave * MT + j) * 16 + lane % 16) * kN + i * 16 + lane / 16 * 4) = acc[i][j];
  __syncthreads();
  for (int at = threadIdx.x; at < MT * 16 * kN; at += 64 * kFewWaves) {
    const int m = at / kN, n = at % kN;
    float z[1][1] = {};
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) z[0][0] += sums[(v * MT * 16 + m) * kN + n];
    if (m < M && n0 + n < N) {
      float bias[1], residual[1][1];
      bias_of<T>(e, n0 + n, 1, bias);
      residual_of<T, true>(e, m, 0, M, n0 + n, N, 1, residual);
      finish<T, true>(e, m, 0, M, n0 + n, N, 1, z, bias, residual);
    }
  }
}

template <typename T, int MT, int NT, int NS>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(const Operand x, const Operand w, int M, int64_t N, int K, const Epilogue e) {
  using S = Stage<T>;
  constexpr int kW = 2048 * NT, kStage = 2048 * (NT + MT), kLoads = 2 * (NT + MT);
  __shared__ __attribute__((aligned(1024))) char smem[kFewWaves * NS * kStage];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
  char* const mine = smem + wave * NS * kStage;
  Loader<T, true, 16 * NT, 1> lw;
  Loader<T, true, 16 * MT, 1> lx;
  lw.init(w, n0, N, wave * S::kK, K, 0, lane, lds_address(mine));
  lx.init(x, 0, M, wave * S::kK, K, 0, lane, lds_address(mine) + kW);
  lw.step = lx.step = kFewWaves * 128;
  Reader<T, true, 16 * NT, NT> rw;
  Reader<T, true, 16 * MT, MT> rx;
  rw.init(0, lane);
  rx.init(0, lane);
  f32x4 acc[NT][MT] = {};
  int kleft = K - wave * S::kK;
#pragma unroll
  for (int q = 0; q < NS; ++q) {
    lw.load(q * kStage, kleft - q * kFewWaves * S::kK, lane);
    lx.load(q * kStage, kleft - q * kFewWaves * S::kK, lane);
    lw.next();
    lx.next();
  }
  int cur = 0;
  for (; kleft > 0; kleft -= kFewWaves * S::kK) {
    wait_loads<(NS - 1) * kLoads>();
    if (kleft < S::kK && kleft % S::kE != 0) {
      lw.clear_end(mine + cur, kleft, lane, kWave);
      lx.clear_end(mine + cur + kW, kleft, lane, kWave);
    }
    u32x4 fw[2][NT], fx[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < NT; ++i) fw[s][i] = rw.get(mine + cur, s, i);
#pragma unroll
      for (int j = 0; j < MT; ++j) fx[s][j] = rx.get(mine + cur + kW, s, j);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is read: its place can be loaded again
    lw.load(cur, kleft - NS * kFewWaves * S::kK, lane);
    lx.load(cur, kleft - NS * kFewWaves * S::kK, lane);
    lw.next();
    lx.next();
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma16<T>(fw[s][i], fx[s][j], acc[i][j]);
    cur = cur == (NS - 1) * kStage ? 0 : cur + kStage;
  }
  wait_loads<0>();
  __syncthreads();
  join_waves<T, MT, NT>(acc, reinterpret_cast<float*>(smem), M, n0, N, e);
}

// The same for rows that start anywhere: fragments straight from memory, with
// kDepth steps of loads under way.
template <typename T>
MHC_DEV u32x4 load_any(const T* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// a chunk of a row that ends before `left` elements, zeros after
template <typename T>
MHC_DEV u32x4 load_end(const T* p, int left) {
  constexpr int kE = 16 / (int)sizeof(T);
  T v[kE];
#pragma unroll
  for (int j = 0; j < kE; ++j) v[j] = j < left ? p[j] : (T)0;
  return __builtin_bit_cast(u32x4, v);
}

template <typename T, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_ragged_rows_kernel(const T* x, int64_t ldx, const T* w, int64_t ldw, int M,
                                                                         int64_t N, int K, const Epilogue e) {
  constexpr int kE = 16 / (int)sizeof(T), kStep = 4 * kE;  // k of a step: a chunk for each of four groups of lanes
  constexpr int kDepth = MT == 1 ? 8 : MT == 2 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) float sums[kFewWaves * MT * 256];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  // (lanes of rows that are not there read another one; their sums are not stored)
  const T* const wr = w + min(n0 + r, N - 1) * ldw + g * kE;
  const T* xr[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xr[j] = x + (int64_t)min(j * 16 + r, M - 1) * ldx + g * kE;
  f32x4 acc[1][MT] = {};
  const int whole = K / (kStep * kDepth) * (kStep * kDepth);
  for (int k = wave * kStep * kDepth; k < whole; k += kFewWaves * kStep * kDepth) {
    u32x4 fw[kDepth], fx[MT][kDepth];
#pragma unroll
    for (int q = 0; q < kDepth; ++q) {
      fw[q] = load_any(wr + k + q * kStep);
#pragma unroll
      for (int j = 0; j < MT; ++j) fx[j][q] = load_any(xr[j] + k + q * kStep);
    }
#pragma unroll
    for (int q = 0; q < kDepth; ++q)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[0][j] = mfma16<T>(fw[q], fx[j][q], acc[0][j]);
  }
  for (int k = whole + wave * kStep; k < K; k += kFewWaves * kStep) {
    const int left = K - k - g * kE;
    const bool full = left >= kE;
    const u32x4 fw = full ? load_any(wr + k) : load_end(wr + k, left);
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[0][j] = mfma16<T>(fw, full ? load_any(xr[j] + k) : load_end(xr[j] + k, left), acc[0][j]);
  }
  join_waves<T, MT, 1>(acc, sums, M, n0, N, e);
}

template <typename T, int MT, int NT, int NS>
int launch_few_rows(const Operand& x, const Operand& w, int64_t M, int64_t N, int64_t K, const Epilogue& e, hipStream_t s) {
  hipLaunchKernelGGL((few_rows_kernel<T, MT, NT, NS>), dim3((unsigned)ceil_div(N, 16 * NT)), dim3(64 * kFewWaves), 0, s, x, w, (int)M, N,
                     (int)K, e);
  MHC_CHECK_LAUNCH("few_rows_kernel");
  return MHC_OK;
}

template <typename T, int MT>
int launch_few(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(N, 16)), block(64 * kFewWaves);
  if (!in_words(x, ldx, K, sizeof(T)) || !in_words(w, ldw, K, sizeof(T))) {
    hipLaunchKernelGGL((few_ragged_rows_kernel<T, MT>), grid, block, 0, s, static_cast<const T*>(x), ldx, static_cast<const T*>(w), ldw,
                       (int)M, N, (int)K, e);
    MHC_CHECK_LAUNCH("few_ragged_rows_kernel");
    return MHC_OK;
  }
  const Operand ox = {x, ldx, K}, ow = {w, ldw, K};
  // Each workgroup reads all of x: between one and two of 16 columns a CU, one
  // of 32 columns reads it once (bf16, 8192 x 2048: 32 rows 11.6 for 10.0 us,
  // 64 rows 13.9 for 12.4; but 4096 x 4096 9.5 for 12.4, and 8200 x 1000
  // 7.5 for 8.4: some CUs have two; in fp32 17.0 for 20.0).
  if constexpr (MT >= 2 && sizeof(T) == 2) {
    const int64_t cus = device_cu_count();
    if (N > 16 * cus && N <= 32 * cus) return launch_few_rows<T, MT, 2, MT == 2 ? 2 : 1>(ox, ow, M, N, K, e, s);
  }
  // (more stages under way in fewer workgroups of a CU: 5.4 for 4.9 us at one row of 4096 x 4096, 10.1 for 8.6 at 32 of 8192 x 2048)
  return launch_few_rows<T, MT, 1, MT == 1 ? 2 : 1>(ox, ow, M, N, K, e, s);
}

template <typename T>
int run_few_rows(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e, hipStream_t s) {
  if (M <= 16) return launch_few<T, 1>(x, ldx, w, ldw, M, N, K, e, s);
  if (M <= 32) return launch_few<T, 2>(x, ldx, w, ldw, M, N, K, e, s);
  return launch_few<T, 4>(x, ldx, w, ldw, M, N, K, e, s);
}

// The sum over the splits, in order, and the epilogue: eight columns a thread
// (four of fp32 outputs, so that a wave reads and writes one piece).
template <typename T> constexpr int kJoin = sizeof(T) == 4 ? 4 : 8;

template <typename T, bool WHOLE>
MHC_DEV void join_columns(const float* part, int splits, int64_t m, int64_t M, int64_t n, int64_t N, int left, const Epilogue& e) {
  constexpr int V = kJoin<T>;
  float z[1][V] = {}, bias[V], residual[1][V];
  bias_of<T>(e, n, left, bias);
  residual_of<T, WHOLE>(e, m, 0, M, n, N, left, residual);
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    float v[V];
    take<WHOLE>(part + ((int64_t)k * M + m) * N + n, v, left);
#pragma unroll
    for (int j = 0; j < V; ++j) z[0][j] += v[j];
  }
  finish<T, WHOLE>(e, m, 0, M, n, N, left, z, bias, residual);
}

template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float* part, int splits, int64_t M, int64_t N, const Epilogue e) {
  constexpr int V = kJoin<T>;
  const uint32_t groups = (uint32_t)ceil_div(N, V);
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < M * groups; at += (int64_t)gridDim.x * 256) {
    const int64_t m = at / groups, n = at % groups * V;
    const int left = (int)min((int64_t)V, N - n);
    if (left == V) join_columns<T, true>(part, splits, m, M, n, N, left, e);
    else join_columns<T, false>(part, splits, m, M, n, N, left, e);
  }
}

template <typename T>
int launch_join(const Epilogue& e, const float* part, int splits, int64_t M, int64_t N, hipStream_t s) {
  const unsigned blocks = (unsigned)std::min(ceil_div(M * ceil_div(N, kJoin<T>), 256), (int64_t)device_cu_count() * 16);
  hipLaunchKernelGGL((join_kernel<T>), dim3(blocks), dim3(256), 0, s, part, splits, M, N, e);
  MHC_CHECK_LAUNCH("join_kernel");
  return MHC_OK;
}

// How a product is cut up: its tile, and into how many parts its reduction.
struct Cut {
  int tile, splits, kper;
  float us;  // estimated
};

// The tiles, and what they take in us on an MI355X: `ends` for the launch, the
// first loads and the outputs, and a stage `alone` with
// few workgroups on the card (its latencies), `busy` for each workgroup of a
// CU that has `fit` of them (its matrix instructions and LDS reads).  From
// x W^T over 16 to 512 stages: 256 x 256 16-bit at 1.12 alone, 1.6 with all
// CUs at it (1.3 PFLOP/s); a stage of fp32 has half the k (timed before values
// were lifted, which takes 5 % more of a stage from 64 x 128 on).
struct TileCost {
  int bm, bn, fit;
  float ends, alone16, busy16, alone32, busy32;
};
constexpr TileCost kTiles[] = {
    {256, 256, 1, 7.0f, 1.12f, 1.60f, 4.10f, 4.75f},   {128, 256, 1, 5.0f, 0.68f, 0.92f, 2.35f, 2.60f},
    {128, 128, 2, 5.0f, 0.48f, 0.53f, 1.67f, 1.28f},   {64, 128, 2, 4.5f, 0.35f, 0.335f, 1.03f, 0.78f},
    {64, 64, 3, 3.6f, 0.29f, 0.21f, 0.58f, 0.525f},
};

inline float stage_us(const TileCost& c, int dtype, float of_cu) {  // of_cu: workgroups of a CU
  const float alone = dtype == kF32 ? c.alone32 : c.alone16, busy = dtype == kF32 ? c.busy32 : c.busy16;
  const float q = ceilf(of_cu);
  return of_cu <= 1.f ? alone + std::max(0.f, busy - alone) * of_cu : std::max(alone * ceilf(q / c.fit), busy * q);
}

inline float join_us(int splits, int64_t M, int64_t N) {  // a launch, and 8 bytes of each sum at 4 TB/s
  return splits > 1 ? 4.f + 2.f * splits * (float)M * (float)N / 1e6f : 0.f;
}

// Rows that a tile may have of an operand.  A k-major one whose rows are longer
// than kMaxRowBytes has been copied to rows of whole chunks; they are at most
// 2^24 bytes long (K < 2^22), and 128 of them stay below 2^31.
inline int most_rows(bool k_major, int64_t K, int dtype) { return k_major && K * (dtype == kF32 ? 4 : 2) > kMaxRowBytes ? 128 : 256; }

// The cut with the least estimated time.  Large tiles read least, small ones
// give every CU work; a reduction is split where even those are too few,
// which costs a launch and its sums' way through memory.
inline Cut cut_of(int64_t M, int64_t N, int64_t K, int dtype, bool a_k, bool b_k) {
  const int kK = dtype == kF32 ? 32 : 64;
  const int stages = (int)ceil_div(K, kK);
  const float cus = (float)device_cu_count();
  Cut best = {0, 1, stages * kK, 0.f};
  for (int t = 0; t < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++t) {
    const TileCost& c = kTiles[t];
    if (c.bm > most_rows(a_k, K, dtype) || c.bn > most_rows(b_k, K, dtype)) continue;
    const float tiles = (float)ceil_div(M, c.bm) * (float)ceil_div(N, c.bn);
    for (int want = 1; want <= 16; ++want) {
      if (want > 1 && (tiles * (want - 1) > 4.f * cus || stages < 2 * want)) break;
      const int per = (stages + want - 1) / want, splits = (stages + per - 1) / per;
      if (splits < want) continue;
      const float us = c.ends + per * stage_us(c, dtype, tiles * splits / cus) + join_us(splits, M, N);
      if (best.us == 0.f || us < best.us) best = {t, splits, per * kK, us};
    }
  }
  return best;
}

// Both products of a backward, dx = dz W and dw = dz^T x, in one launch of the
// smaller tiles, or (together false) one after the other.
struct PairCut {
  bool together;
  Cut dx, dw;
};

inline PairCut pair_of(int64_t M, int64_t N, int64_t K, int dtype) {
  PairCut best = {false, cut_of(M, K, N, dtype, true, false), cut_of(N, K, M, dtype, false, false)};
  float least = best.dx.us + best.dw.us;
  const float cus = (float)device_cu_count();
  const int kK = dtype == kF32 ? 32 : 64;
  const int stages1 = (int)ceil_div(N, kK), stages2 = (int)ceil_div(M, kK);
  constexpr int kWant[] = {1, 2, 3, 4, 6, 8};
  for (int t = 2; t < 5; ++t) {  // (at most 128 rows: see most_rows)
    const TileCost& c = kTiles[t];
    const float tiles1 = (float)ceil_div(M, c.bm) * (float)ceil_div(K, c.bn), tiles2 = (float)ceil_div(N, c.bm) * (float)ceil_div(K, c.bn);
    if (tiles1 + tiles2 > 16.f * cus) continue;  // (each fills the card)
    for (int want1 : kWant) {
      if (want1 > 1 && (tiles1 * want1 + tiles2 > 4.f * cus || stages1 < 2 * want1)) break;
      const int per1 = (stages1 + want1 - 1) / want1, splits1 = (stages1 + per1 - 1) / per1;
      for (int want2 : kWant) {
        if (want2 > 1 && (tiles1 * want1 + tiles2 * want2 > 4.f * cus || stages2 < 2 * want2)) break;
        const int per2 = (stages2 + want2 - 1) / want2, splits2 = (stages2 + per2 - 1) / per2;
        const float n1 = tiles1 * splits1, n2 = tiles2 * splits2, of_cu = (n1 + n2) / cus;
        // more than one a CU: of all lengths
        const float per = of_cu <= 1.f ? (float)std::max(per1, per2) : (n1 * per1 + n2 * per2) / (n1 + n2);
        const float us = c.ends + std::max(per * stage_us(c, dtype, of_cu), (float)std::max(per1, per2) * stage_us(c, dtype, 0.f)) +
                         join_us(splits1, M, K) + join_us(splits2, N, K);
        if (us < least) {
          least = us;
          best = {true, {t, splits1, per1 * kK, us}, {t, splits2, per2 * kK, us}};
        }
      }
    }
  }
  return best;
}

// Whether x W^T goes to the kernels for few rows: up to 64 of them, unless a
// tile is estimated faster (33 to 64 rows of a W of over some 30 M elements,
// or with short rows: 8192 x 8192 bf16 35 us here, 27 in tiles; 16384 x 1024
// 14 and 8).  From one to four workgroups of a CU; per stage of a wave:
// 0.35, 0.65, 1.05 us for 16, 32, 64 rows (fp32: 0.8, 1.1, 1.5).
inline bool few_rows(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, int dtype) {
  if (M > 64) return false;
  const bool f32 = dtype == kF32;
  const int bytes = f32 ? 4 : 2;
  const bool words = in_words(x, ldx, K, bytes) && in_words(w, ldw, K, bytes);
  const float stage = f32 ? (M <= 16 ? 0.8f : M <= 32 ? 1.1f : 1.5f) : (M <= 16 ? 0.35f : M <= 32 ? 0.65f : 1.05f);
  const float of_cu = std::max(1.f, (float)N / 16.f / (float)device_cu_count());
  const float few = 3.f + of_cu * (float)ceil_div(K * bytes, 128 * kFewWaves) * stage * (words ? 1.f : 1.8f);
  // (tiles need copies of rows that are no whole words: two launches and the operands' way out and in)
  const float copies = words ? 0.f : 9.f + 2.f * (float)((M + N) * K * bytes) / 4e6f;
  return few <= cut_of(M, N, K, dtype, true, true).us + copies;
}

template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, int NS>
int launch(const Product& p, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(p.M, BM) * ceil_div(p.N, BN)), (unsigned)p.splits), block(64 * WM * WN);
  hipLaunchKernelGGL((tile_kernel<T, AK, BK, BM, BN, WM, WN, NS>), grid, block, 0, s, p);
  MHC_CHECK_LAUNCH("tile_kernel");
  return MHC_OK;
}

// Rows of waves of the middle tiles: two waves for each SIMD, so that one has
// products while the other waits for its fragments (bf16 2048 x 2048 x 2048 in
// 128 x 128 28 us with four waves, 24 with eight; 1000 x 1024 x 1024 in
// 64 x 128 11.2 and 9.8).  fp32, which has more products for each fragment,
// stays with four (2048 x 2048 x 2048 in two parts 104 and 111).
template <typename T>
constexpr int kRowWaves = sizeof(T) == 2 ? 4 : 2;

template <typename T, bool AK, bool BK>
int run_layout(const Product& p, int tile, hipStream_t s) {
  switch (tile) {
    case 0: return launch<T, AK, BK, 256, 256, 2, 4, 2>(p, s);
    case 1: return launch<T, AK, BK, 128, 256, 2, 4, 2>(p, s);
    case 2: return launch<T, AK, BK, 128, 128, kRowWaves<T>, 2, 2>(p, s);
    case 3: return launch<T, AK, BK, 64, 128, kRowWaves<T>, 2, 3>(p, s);
    default: return launch<T, AK, BK, 64, 64, 4, 1, 3>(p, s);
  }
}

template <typename T, int BM, int BN, int WM, int WN, int NS>
int launch_pair(Pair p, hipStream_t s) {
  p.dx_count = (uint32_t)(ceil_div(p.dx.M, BM) * ceil_div(p.dx.N, BN) * p.dx.splits);
  p.dw_count = (uint32_t)(ceil_div(p.dw.M, BM) * ceil_div(p.dw.N, BN) * p.dw.splits);
  const bool first = p.dx.kper >= p.dw.kper;
  p.dx0 = first ? 0 : p.dw_count;
  p.dw0 = first ? p.dx_count : 0;
  const unsigned sums = p.db != nullptr ? (unsigned)ceil_div(p.N, kSumCols) : 0;
  hipLaunchKernelGGL((pair_kernel<T, BM, BN, WM, WN, NS>), dim3(p.dx_count + p.dw_count + sums), dim3(64 * WM * WN), 0, s, p);
  MHC_CHECK_LAUNCH("pair_kernel");
  return MHC_OK;
}

// The products of a backward together.  part: the sums of dx's parts, if it is split, and then of dw's.
template <typename T>
int run_pair(Pair p, const PairCut& c, float* part, hipStream_t s) {
  const Epilogue dx = p.dx.e, dw = p.dw.e;
  float* const part2 = c.dx.splits > 1 ? part + c.dx.splits * p.dx.M * p.dx.N : part;
  p.dx.splits = c.dx.splits, p.dx.kper = c.dx.kper;
  p.dw.splits = c.dw.splits, p.dw.kper = c.dw.kper;
  if (c.dx.splits > 1) p.dx.e = Epilogue{nullptr, nullptr, part, nullptr, MHC_ACT_NONE, 1};
  if (c.dw.splits > 1) p.dw.e = Epilogue{nullptr, nullptr, part2, nullptr, MHC_ACT_NONE, 1};
  int rc = c.dx.tile == 2   ? launch_pair<T, 128, 128, kRowWaves<T>, 2, 2>(p, s)
           : c.dx.tile == 3 ? launch_pair<T, 64, 128, kRowWaves<T>, 2, 3>(p, s)
                            : launch_pair<T, 64, 64, 4, 1, 3>(p, s);
  if (rc == MHC_OK && c.dx.splits > 1) rc = launch_join<T>(dx, part, c.dx.splits, p.dx.M, p.dx.N, s);
  if (rc == MHC_OK && c.dw.splits > 1) rc = launch_join<T>(dw, part2, c.dw.splits, p.dw.M, p.dw.N, s);
  return rc;
}

// The product of one type; a_k / b_k: the operand's k are contiguous.  part: splits * M * N floats where it is split.
template <typename T>
int run_product(Product p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s) {
  const Epilogue e = p.e;
  p.splits = c.splits;
  p.kper = c.kper;
  if (c.splits > 1) p.e = Epilogue{nullptr, nullptr, part, nullptr, MHC_ACT_NONE, 1};
  const int rc = a_k && b_k ? run_layout<T, true, true>(p, c.tile, s)
                 : a_k      ? run_layout<T, true, false>(p, c.tile, s)
                            : run_layout<T, false, false>(p, c.tile, s);
  if (rc != MHC_OK || c.splits == 1) return rc;
  return launch_join<T>(e, part, c.splits, p.M, p.N, s);
}

int run_few_rows_f32(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e, hipStream_t s);
int run_few_rows_bf16(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e, hipStream_t s);
int run_few_rows_f16(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e, hipStream_t s);
int run_pair_f32(const Pair& p, const PairCut& c, float* part, hipStream_t s);
int run_pair_bf16(const Pair& p, const PairCut& c, float* part, hipStream_t s);
int run_pair_f16(const Pair& p, const PairCut& c, float* part, hipStream_t s);
int run_product_f32(const Product& p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s);
int run_product_bf16(const Product& p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s);
int run_product_f16(const Product& p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s);

}  // namespace gemm
}  // namespace mhc
