// Products of linear_cross_entropy, whose rows of tokens are counted on the
// device: logits' sums, their gradient, and that gradient's two products.
#pragma once

#include "mhc_gemm.hpp"

namespace mhc {
namespace ce {

using gemm::Cut;
using gemm::Epilogue;
using gemm::Operand;
using gemm::Product;

// What the forward leaves for the backward, in words: the tokens that count
// ("live"), in order, and what is known of each.
struct State {
  int* head;     // how many are live; as floats, the largest weight over D, and the largest weight; as a double from word 4 on, D
  int* index;    // [T] their tokens
  int* pos;      // [T] of each token: its place among them, or -1
  int* target;   // [T] by place: -1 where it is no column
  float* coef;   // [T] by place: weight / largest weight
  float* top;    // [T] by place: largest logit
  float* inv;    // [T] by place: 1 / sum of exp(logit - top)

  static constexpr int kHead = 16;
  static size_t bytes(int64_t T) { return (size_t)(kHead + 6 * T) * 4; }
  State(void* p, int64_t T) {
    head = static_cast<int*>(p);
    index = head + kHead;
    pos = index + T;
    target = pos + T;
    coef = reinterpret_cast<float*>(target + T);
    top = coef + T;
    inv = top + T;
  }
};

// dz in fp16 is held times 2^14: a probability below 2^-14 would lose bits
// there, and one of 2^-24 be 0.
template <typename T> inline constexpr float kDzUnit = 1.f;
template <> inline constexpr float kDzUnit<_Float16> = 0x1p14f;

// fp32 rows as pairs of fp16 parts: each row times a power of two that brings its
// largest value to 2^14, each value the sum of the nearest fp16 number and of
// the one nearest to what is left, which is the value to 2^-24 of itself (and to
// 2^-40 of the row's largest).  Of the products of two values three parts are
// formed (the fourth is below 2^-24): rows of [high, low, high] against rows of
// [high, high, low], 3 C long, half of what linear_act's fp32 tiles do.
//
// dz's two products are formed so, too, from logits that were kept.  Their k are
// tokens and columns, whose powers of two go to dz: dx's rows are sums of dz w[v]
// over the parts of W, each row of dz w lifted as one of x is, dW's of dz x[t]
// over the parts of x, each column lifted.
//
// Powers of two are put together as their exponents: the product of two of them
// may be past fp32's range where the value that they go to is 0, or brings it
// back into it, and so may the value times one of them.
MHC_DEV int power_of(float two) { return (int)(__builtin_bit_cast(uint32_t, two) >> 23) - 127; }
MHC_DEV float times_power(float v, int e) { return __builtin_ldexpf(v, e); }

struct Halves {
  const float *x, *w;  // of each row: what its parts are to be multiplied by

  template <int BM, int BN, int WM, int WN, int JM, int JN>
  MHC_DEV void scale(const Product& p, const gemm::Place<BM, BN, WM, WN>& at, f32x4 (&acc)[JN][JM]) const {
    const int64_t m0 = at.m0 + at.wm + at.lane % 16, n0 = at.n0 + at.wn + at.lane / 16 * 4;
    int row[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j) row[j] = power_of(x[min(m0 + j * 16, p.M - 1)]);
#pragma unroll
    for (int i = 0; i < JN; ++i) {
      int column[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) column[k] = power_of(w[min(n0 + i * 16 + k, p.N - 1)]);
#pragma unroll
      for (int j = 0; j < JM; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][j][k] = times_power(acc[i][j][k], row[j] + column[k]);
    }
  }
};

// The power of two, as its exponent's bits, that brings a row of the largest
// magnitude `top` to 2^14, if both are normal numbers (a row with an infinity or
// NaN: 1), and its reciprocal.
MHC_DEV uint32_t lift_of(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 127 : min(268u - max(e, 15u), 253u);
}
MHC_DEV float lift_by(uint32_t up) { return __builtin_bit_cast(float, up << 23); }
MHC_DEV float lower_by(uint32_t up) { return __builtin_bit_cast(float, (254u - up) << 23); }

// dz of a piece of the vocabulary as fp16 parts, in rows of `pitch`, for each of
// its products, and the largest magnitudes by which they are lifted, as bits.
struct Parts {
  _Float16 *x_high, *x_low;  // for dx
  _Float16 *w_high, *w_low;  // for dW
  uint32_t *row, *col;
  uint32_t *rows, *cols;     // of parts of each, see tops_kernel
  int64_t pitch;

  static constexpr int kRows = 64;  // of a part of a column
  static size_t top_words(int64_t T, int64_t N) { return T + N + T * ceil_div(N, 256) + ceil_div(T, kRows) * N; }
};

// The logits that a forward keeps: of each live token a row of `pitch`.
struct Kept {
  float* z;  // or NULL
  int64_t pitch;
};
inline int64_t kept_pitch(int64_t V) { return (V + 63) / 64 * 64; }

// Logits to dz = coef (softmax - [v = target]), zeros past the last column.
//
// dz of 16-bit operands is rounded to their type, since it is an operand of two
// products of that type: with the largest weight brought to 1 (and fp16's 2^14)
// an element is off by 2^-8 (2^-11) of itself at most, which a product's sums
// average out where many elements count; a row of dW that one token's element
// makes up is off by as much as its own rounding adds (8192 x 50257 x 4096 bf16:
// dx and dW 2.0e-3 off in the root mean square, 1.7e-3 from dz in fp32, which is
// the outputs' rounding alone).  Two parts of dz, as fp32's, would double both
// products (4.4 ms of 6.8).  The exponential is the hardware's: 2^-22 of itself, and
// 0 below 2^-126.
struct Gradient {
  const int* target;
  const float *coef, *top, *inv;
  int64_t v0;  // the vocabulary's index of the first column
  float unit;

  // a token's numbers
  struct Row {
    float c, t, each;
    int to;
  };
  MHC_DEV Row row(int64_t m) const {
    const int to = target[m];
    const float c = to < 0 ? __builtin_nanf("") : coef[m] * unit;
    return {c, top[m], c * inv[m], to};
  }

  template <bool FAST, typename P, int JM, int JN>
  MHC_DEV void apply(const Product& p, const P& at, f32x4 (&acc)[JN][JM]) const {
    const int64_t m0 = at.m0 + at.wm + at.lane % 16, n0 = at.n0 + at.wn + at.lane / 16 * 4;
#pragma unroll
    for (int j = 0; j < JM; ++j) {
      const Row r = row(min(m0 + j * 16, p.M - 1));
      const int64_t mine = r.to < 0 ? -1 : r.to - v0 - n0;  // the target's place among the lane's columns
#pragma unroll
      for (int i = 0; i < JN; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float d = r.each * gemm::exp_of<FAST>(acc[i][j][k] - r.t) - (mine == i * 16 + k ? r.c : 0.f);
          acc[i][j][k] = n0 + i * 16 + k < p.N ? d : 0.f;
        }
    }
  }
};

// The same from logits that were kept: ROWS rows of 256 columns, eight a lane,
// of dz [rows, width], of which N columns are there (6144 x 12800 bf16: 97 us
// for 472 MB, 4.9 TB/s).
template <typename T, int THREADS, int ROWS>
MHC_DEV void dz_of_kept(const Gradient& g, const Kept& kept, T* dz, int64_t width, int64_t N, int64_t rows, int64_t m0, int64_t n0) {
  constexpr int kEach = THREADS / 32, kAhead = 4;
  const int64_t n = n0 + threadIdx.x % 32 * 8;
  if (n >= width) return;
  const float* const from = kept.z + g.v0 + n;
  const int64_t m1 = min(m0 + ROWS, rows);
  for (int64_t m = m0 + threadIdx.x / 32; m < m1; m += kEach * kAhead) {
    f32x4 z[kAhead][2];
    Gradient::Row r[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {  // (rows past the last one read it once more: a load under a condition would wait for itself)
      const int64_t at = min(m + q * kEach, m1 - 1);
      const f32x4* const p = reinterpret_cast<const f32x4*>(from + at * kept.pitch);
      z[q][0] = __builtin_nontemporal_load(p);
      z[q][1] = __builtin_nontemporal_load(p + 1);
      r[q] = g.row(at);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (m + q * kEach >= m1) break;
      const int64_t mine = r[q].to < 0 ? -1 : r[q].to - g.v0 - n;
      float d[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        d[k] = r[q].each * gemm::exp_of<sizeof(T) == 2>(z[q][k / 4][k % 4] - r[q].t) - (mine == k ? r[q].c : 0.f);
        d[k] = n + k < N ? d[k] : 0.f;
      }
      gemm::put<true>(dz + (m + q * kEach) * width + n, d, 8);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const Gradient g, const Kept kept, T* dz, int64_t width, int64_t N, const int* live) {
  const uint32_t wide = (uint32_t)ceil_div(width, 256);
  dz_of_kept<T, 256, 32>(g, kept, dz, width, N, *live, (int64_t)(blockIdx.x / wide) * 32, (int64_t)(blockIdx.x % wide) * 256);
}

template <bool FAST>
struct GradientOf : Gradient {
  using Own = gemm::AsTheyAre::Own;
  template <typename P>
  MHC_DEV Own ahead(const Product&, const P&) const { return {}; }
  template <typename P, int JM, int JN>
  MHC_DEV void operator()(const Product& p, const P& at, int, char*, const Own&, f32x4 (&acc)[JN][JM]) const {
    this->template apply<FAST>(p, at, acc);
  }
};

// the same of logits that are products of halves
struct GradientOfHalves : Gradient {
  Halves halves;
  using Own = gemm::AsTheyAre::Own;
  template <typename P>
  MHC_DEV Own ahead(const Product&, const P&) const { return {}; }
  template <typename P, int JM, int JN>
  MHC_DEV void operator()(const Product& p, const P& at, int, char*, const Own&, f32x4 (&acc)[JN][JM]) const {
    halves.scale(p, at, acc);
    this->template apply<false>(p, at, acc);
  }
};

// sums times a * b * c, a and b in memory (b may be NULL)
struct ScaledBy {
  const float *a, *b;
  float c;
  using Own = gemm::AsTheyAre::Own;
  template <typename P>
  MHC_DEV Own ahead(const Product&, const P&) const { return {}; }
  template <typename P, int JM, int JN>
  MHC_DEV void operator()(const Product&, const P&, int, char*, const Own&, f32x4 (&acc)[JN][JM]) const {
    const float s = a[0] * (b != nullptr ? b[0] : 1.f) * c;
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int j = 0; j < JM; ++j) acc[i][j] *= s;
  }
};

// The product with as many rows of tokens as there are: they are rows of the
// outputs, or (AK false) what is summed over.  False: not this workgroup's.
template <bool AK, int BM, int BN>
MHC_DEV bool limit(Product& p, const int* live, uint32_t tile) {
  const int64_t n = __builtin_amdgcn_readfirstlane(*live);
  if constexpr (AK) {
    p.M = min(p.M, n);
    return tile < ceil_div(p.M, BM) * ceil_div(p.N, BN);
  } else {
    p.K = min(p.K, n);
    return true;
  }
}

// The epilogue's sums alone, known here, so that nothing else is compiled.
MHC_DEV void only_sums(Epilogue& e) {
  e.bias = nullptr;
  e.dact = nullptr;
  e.act = MHC_ACT_NONE;
}

// One part of a reduction whose parts have outputs of their own, one after the
// other, which sum up what the calls for pieces of it add.
MHC_DEV void move_to_part(Epilogue& e, int64_t at) {
  e.out = static_cast<float*>(e.out) + at;
  if (e.residual != nullptr) e.residual = static_cast<const float*>(e.residual) + at;
}

// (SUMS: the parts of a reduction add to sums of their own; O: of the outputs)
template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, int NS, bool SUMS, typename O, typename Then>
__global__ __launch_bounds__(64 * WM * WN) void live_tile_kernel(Product p, const int* live, int64_t width, const Then then) {
  __shared__ __attribute__((aligned(1024))) char smem[gemm::TileBytes<T, BM, BN, WM, WN, NS>::kAll];
  const int64_t part = p.M * p.N;
  if (!limit<AK, BM, BN>(p, live, blockIdx.x)) return;
  only_sums(p.e);
  if constexpr (SUMS) {
    move_to_part(p.e, blockIdx.y * part);
    p.splits = 1;
  }
  gemm::run_tile<T, AK, BK, BM, BN, WM, WN, NS, O>(p, smem, blockIdx.x, (int)blockIdx.y, part, width, then);
}

// dx and dW of one piece of the vocabulary and dz of the next, none of which
// needs another, as one launch, so that the card is full to its end: their
// tiles are few and long (6144 tokens, 50257 columns in four pieces, C = 4096:
// 384 of 196 stages on 256 CUs, 800 of 96 and 1200 of 64; 1.62 ms in one launch,
// 1.88 in three; the whole call, from logits that were kept, 6.8 ms and 7.6).
// The longest go first.  fp32 tiles gain nothing by it (1000
// tokens, 32768 columns, C = 1024: 0.79 ms for dx and dW, 0.74 apart).
struct Joint {
  Product dx, dw, dz;   // M = 0: not there
  int64_t part, width;  // of a part of dx's sums, and of dz's rows
  ScaledBy by;
  Gradient g;
  Kept kept;            // what dz is of, if there is any
};

// A kernel's first argument where it lies, to be read when it is needed: those
// of all three products at once are more than there are scalar registers.
template <typename A>
MHC_DEV const A& first_argument() {
  auto* p = (const __attribute__((address_space(4))) A*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const A*)p;
}

template <typename T, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void joint_kernel(const Joint, const int* live) {
  __shared__ __attribute__((aligned(1024))) char smem[gemm::TileBytes<T, BM, BN, WM, WN, NS>::kAll];
  const int64_t n = __builtin_amdgcn_readfirstlane(*live);
  const auto tiles = [](int64_t M, int64_t N) { return (uint32_t)(ceil_div(M, BM) * ceil_div(N, BN)); };
  const Joint& j = first_argument<Joint>();
  uint32_t id = blockIdx.x;
  const uint32_t of_dx = tiles(min(j.dx.M, n), j.dx.N), all_dx = of_dx * j.dx.splits, of_dw = tiles(j.dw.M, j.dw.N);
  if (id < all_dx) {
    const Joint& k = first_argument<Joint>();
    Product p = k.dx;
    only_sums(p.e);
    p.M = min(p.M, n);
    p.splits = 1;
    move_to_part(p.e, id / of_dx * k.part);
    gemm::run_tile<T, true, false, BM, BN, WM, WN, NS, T>(p, smem, id % of_dx, (int)(id / of_dx), 0, p.N);
  } else if (id - all_dx < of_dw) {
    const Joint& k = first_argument<Joint>();
    Product p = k.dw;
    only_sums(p.e);
    p.K = min(p.K, n);
    gemm::run_tile<T, false, false, BM, BN, WM, WN, NS, T>(p, smem, id - all_dx, 0, 0, p.N, ScaledBy(k.by));
  } else {
    const Joint& k = first_argument<Joint>();
    Product p = k.dz;
    only_sums(p.e);
    p.M = min(p.M, n);
    id -= all_dx + of_dw;
    if (id >= tiles(p.M, p.N)) return;
    if (k.kept.z != nullptr) {
      const uint32_t wide = (uint32_t)ceil_div(p.N, BN);
      dz_of_kept<T, 64 * WM * WN, BM>(Gradient(k.g), Kept(k.kept), static_cast<T*>(p.e.out), k.width, p.N, p.M, (int64_t)(id / wide) * BM,
                                      (int64_t)(id % wide) * BN);
      return;
    }
    gemm::run_tile<T, true, true, BM, BN, WM, WN, NS, T>(p, smem, id, 0, 0, k.width, GradientOf<sizeof(T) == 2>{k.g});
  }
}

template <typename T>
int run_joint(const Joint& j, const int* live, hipStream_t s) {
  constexpr int kB = 256;
  const auto tiles = [](int64_t M, int64_t N) { return ceil_div(M, kB) * ceil_div(N, kB); };
  const int64_t grid = tiles(j.dx.M, j.dx.N) * j.dx.splits + tiles(j.dw.M, j.dw.N) + tiles(j.dz.M, j.dz.N);
  hipLaunchKernelGGL((joint_kernel<T, kB, kB, 2, 4, 2>), dim3((unsigned)grid), dim3(512), 0, s, j, live);
  MHC_CHECK_LAUNCH("joint_kernel");
  return MHC_OK;
}

// exp(x - top) below `top`; a part of a row that is -inf alone has no top, and -inf - -inf would be NaN
MHC_DEV float base_of(float top) { return top == -__builtin_inff() ? 0.f : top; }

// The live tokens' rows: where they lie in x, or one after the other.
struct RowsOf {
  const int* index;  // or NULL
  int64_t rows;
  template <typename L, typename P>
  MHC_DEV void init(L& l, const Product& p, const P& at, uint32_t lds) const {
    l.init(p.a, index != nullptr ? 0 : at.m0, index != nullptr ? rows : p.M, at.k0, at.k1, at.wave, at.lane, lds);
    if (index != nullptr) l.take_rows(p.a, index, at.m0, p.M, at.wave, at.lane);
  }
};

MHC_DEV float weight_of(const mhc_linear_ce_args& a, int64_t t) {
  if (a.weights == nullptr) return 1.f;
  return a.weights_dtype == MHC_DTYPE_U8 ? (static_cast<const uint8_t*>(a.weights)[t] != 0 ? 1.f : 0.f)
                                         : static_cast<const float*>(a.weights)[t];
}

// The numbers of all tokens: how many are live, their largest weight and D.
MHC_DEV void store_head(const mhc_linear_ce_args& a, const State& s, int live, double sum, float top) {
  const double d = a.denominator > 0.f ? (double)a.denominator : sum != 0 ? sum : 1.0;
  s.head[0] = live;
  reinterpret_cast<float*>(s.head)[1] = (float)((double)top / d);
  reinterpret_cast<float*>(s.head)[2] = top;
  *reinterpret_cast<double*>(s.head + 4) = d;
}

// Up to 64 tokens: which are live is found by every workgroup for itself, a
// token for each lane, and the first one writes down the state for the launches
// after it: one launch less, and some 4 us (64 x 32000 x 2048 bf16 45.6 to 41.3).
struct FewTokens {
  mhc_linear_ce_args a;
  State s;
  float* logp;

  // how many are live; their places' tokens and targets to `index` and `target` (LDS, the same by every wave)
  MHC_DEV int live(int* index, int* target) const {
    const int t = threadIdx.x % kWave;
    float w = t < a.T ? weight_of(a, t) : 0.f;
    const int64_t y = t < a.T ? a.targets[t] : a.ignore_index;
    if (y == a.ignore_index) w = 0.f;
    const uint64_t all = __ballot(w != 0.f);
    const int place = __popcll(all & (((uint64_t)1 << t) - 1)), to = y >= 0 && y < a.V ? (int)y : -1, count = __popcll(all);
    if (w != 0.f) {
      index[place] = t;
      target[place] = to;
    }
    if (blockIdx.x == 0 && threadIdx.x < kWave) {
      double sum = (double)w;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
      const float top = group_max<kWave>(fabsf(w));
      if (t < a.T) {
        s.pos[t] = w != 0.f ? place : -1;
        if (w == 0.f) logp[t] = 0.f;
      }
      if (w != 0.f) {
        s.index[place] = t;
        s.target[place] = to;
        s.coef[place] = w;
      }
      if (t == 0) store_head(a, s, count, sum, top);
    }
    return count;
  }
};

// A tile of logits, of which only each row's largest and the sum of
// exp(logit - largest) are kept, and the target's: to part[row][tile] and
// at_target[row]; and the logits themselves, if there is a place for them.  The
// tile is one of the vocabulary's from v0 on, of which a row has `tiles`.
struct SumsOf {
  const int* target;
  float2* part;
  float* at_target;
  int64_t tiles, v0;
  Kept kept;
};

// What becomes of a tile of logits; `rows`: a bit for each of the rows that it is for.
template <bool FAST, int BM, int BN, int WM, int WN, int JM, int JN>
MHC_DEV void store_sums(const Product& p, const gemm::Place<BM, BN, WM, WN>& at, const SumsOf& of, f32x4 (&acc)[JN][JM], const uint32_t* rows, char* smem) {
  constexpr int kThreads = 64 * WM * WN;
  const int64_t m0 = at.m0 + at.wm + at.lane % 16, n0 = at.n0 + at.wn + at.lane / 16 * 4;
  const auto is_for = [&](int r) { return rows == nullptr || (rows[r / 32] >> r % 32 & 1) != 0; };
  if (of.kept.z != nullptr) {
    float* const to = of.kept.z + of.v0 + n0;
#pragma unroll
    for (int j = 0; j < JM; ++j) {
      if (m0 + j * 16 >= p.M || !is_for(at.wm + at.lane % 16 + j * 16)) continue;
#pragma unroll
      for (int i = 0; i < JN; ++i)
        if (of.v0 + n0 + i * 16 < of.kept.pitch) *reinterpret_cast<f32x4*>(to + (m0 + j * 16) * of.kept.pitch + i * 16) = acc[i][j];
    }
  }
  if (at.n0 + BN > p.N) {
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int j = 0; j < JM; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n0 + i * 16 + k >= p.N) acc[i][j][k] = -__builtin_inff();
  }
  float2* const of_waves = reinterpret_cast<float2*>(smem);  // [columns of waves][BM]
#pragma unroll
  for (int j = 0; j < JM; ++j) {
    float top = acc[0][j][0];
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, acc[i][j][k]);
    top = xor_allreduce<16>(top, MaxOp{});
    top = xor_allreduce<32>(top, MaxOp{});
    const float base = base_of(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += gemm::exp_of<FAST>(acc[i][j][k] - base);
    sum = xor_allreduce<16>(sum, SumOp{});
    sum = xor_allreduce<32>(sum, SumOp{});
    if (at.lane < 16) of_waves[at.wave % WN * BM + at.wm + j * 16 + at.lane] = float2{top, sum};
    const int64_t m = m0 + j * 16;
    const int64_t mine = m < p.M && is_for(at.wm + at.lane % 16 + j * 16) ? of.target[m] - of.v0 - n0 : -1;
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (mine == i * 16 + k) of.at_target[m] = acc[i][j][k];
  }
  __syncthreads();
  for (int r = threadIdx.x; r < BM; r += kThreads) {
    if (at.m0 + r >= p.M) break;
    if (!is_for(r)) continue;
    float2 all = of_waves[r];
#pragma unroll
    for (int w = 1; w < WN; ++w) {
      const float2 one = of_waves[w * BM + r];
      const float top = fmaxf(all.x, one.x), base = base_of(top);
      all.y = all.y * gemm::exp_of<FAST>(all.x - base) + one.y * gemm::exp_of<FAST>(one.x - base);
      all.x = top;
    }
    of.part[(at.m0 + r) * of.tiles + (of.v0 + at.n0) / BN] = all;
  }
}

// (fp32: the rows of a tile that have a sum past the range of parts are formed
// once more with fp32 instructions, as run_tile does it for single sums.  Tiles
// for few tokens, which have few sums and time, set them aside every four
// stages: of 40 tokens, C = 2285, fp32 log probabilities are 5e-8 off, without
// 3.4e-7.)
template <typename T, bool HALVES, int BM, int BN, int WM, int WN, int NS>
MHC_DEV void sums_tile(const Product& p, const RowsOf& rows, const SumsOf& of, const Halves& halves, char* smem) {
  constexpr int JM = BM / WM / 16, JN = BN / WN / 16, kEvery = BM == 64 ? 4 : 0;
  constexpr bool kFast = sizeof(T) == 2 && !HALVES;
  const gemm::Place<BM, BN, WM, WN> at(p, blockIdx.x, 0);
  f32x4 acc[JN][JM] = {};
  if constexpr (!gemm::kSplit<T, BN>) {
    gemm::sum_tile<T, true, true, BM, BN, WM, WN, NS, RowsOf, kEvery>(p, at, smem, acc, rows);
    if constexpr (HALVES) halves.scale(p, at, acc);
    __syncthreads();  // nobody reads the stages any more
    store_sums<kFast>(p, at, of, acc, nullptr, smem);
  } else {
    __shared__ uint32_t past[BM / 32];
    if (threadIdx.x < BM / 32) past[threadIdx.x] = 0;
    gemm::sum_tile_split<true, true, BM, BN, WM, WN, NS, RowsOf, kEvery>(p, at, smem, acc, rows);
    const int n0 = (int)min(p.N - at.n0, (int64_t)BN) - at.wn - at.lane / 16 * 4;  // columns from the lane's first on
#pragma unroll
    for (int j = 0; j < JM; ++j) {
      bool one = false;
#pragma unroll
      for (int i = 0; i < JN; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) one |= !(fabsf(acc[i][j][k]) < __builtin_inff()) && i * 16 + k < n0;
      const int r = at.wm + j * 16 + at.lane % 16;
      if (one && at.m0 + r < p.M) atomicOr(past + r / 32, 1u << r % 32);
    }
    __syncthreads();  // nobody reads the stages any more
    uint32_t again = 0;
#pragma unroll
    for (int k = 0; k < BM / 32; ++k) again |= past[k];
    again = __builtin_amdgcn_readfirstlane(again);
    store_sums<kFast>(p, at, of, acc, nullptr, smem);
    if (!again) return;
#pragma unroll
    for (int i = 0; i < JN; ++i)
#pragma unroll
      for (int j = 0; j < JM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    gemm::Place<BM, BN, WM, WN> once_more = at;
    asm volatile("" : "+v"(once_more.lane), "+s"(once_more.wave));  // (or registers would hold places from the first sums to these)
    __syncthreads();  // nobody reads the rows' numbers in LDS any more
    gemm::sum_tile<T, true, true, BM, BN, WM, WN, NS, RowsOf, kEvery>(p, once_more, smem, acc, rows);
    __syncthreads();
    store_sums<kFast>(p, once_more, of, acc, past, smem);
  }
}

template <typename T, bool HALVES, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void sums_tile_kernel(Product p, const RowsOf rows, const int* live, const SumsOf of, const Halves halves) {
  __shared__ __attribute__((aligned(1024))) char smem[NS * (BM + BN) * 128];
  if (limit<true, BM, BN>(p, live, blockIdx.x)) sums_tile<T, HALVES, BM, BN, WM, WN, NS>(p, rows, of, halves, smem);
}

template <typename T, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void sums_few_kernel(Product p, SumsOf of, const FewTokens few) {
  __shared__ __attribute__((aligned(1024))) char smem[NS * (64 + BN) * 128];
  __shared__ int index[64], target[64];
  const int64_t rows = p.M;
  p.M = __builtin_amdgcn_readfirstlane(few.live(index, target));
  if (p.M == 0) return;
  __syncthreads();
  of.target = target;
  sums_tile<T, false, 64, BN, WM, WN, NS>(p, RowsOf{index, rows}, of, {}, smem);
}

inline constexpr int kFewRows = 16, kRowsColumns = 32;

// Up to 16 tokens: 32 columns a workgroup, whose waves split k as few_rows_kernel's
// do, so that a small vocabulary's products take no longer than their loads, and
// 16 rows are multiplied instead of 64 (12 x 9376 x 2285 fp32 62 to 29 us, 2 x 72999
// x 2624 251 to 143; bf16 2 x 4524 x 2240 21 to 10).  takes_rows says when.  All
// tokens' logits are formed, and those of the live ones looked at, 32 threads for
// each.
template <typename T, int NS>
__global__ __launch_bounds__(64 * gemm::kFewWaves) void sums_rows_kernel(const Product p, const SumsOf of, const FewTokens few) {
  constexpr int NT = kRowsColumns / 16, kN = kRowsColumns, kSums = gemm::kFewWaves * kFewRows * kN * 4;
  __shared__ __attribute__((aligned(1024))) char smem[std::max(gemm::kFewBytes<1, NT, NS>, kSums)];
  __shared__ int index[64], target[64];
  const int count = __builtin_amdgcn_readfirstlane(few.live(index, target));
  if (count == 0) return;
  const int64_t n0 = (int64_t)blockIdx.x * kN;
  f32x4 acc[NT][1] = {};
  gemm::sum_few_rows<T, 1, NT, NS>(p.a, p.b, (int)p.M, n0, p.N, (int)p.K, smem, acc);
  float* const sums = reinterpret_cast<float*>(smem);  // [waves][rows][columns]
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int i = 0; i < NT; ++i) *reinterpret_cast<f32x4*>(sums + (wave * kFewRows + lane % 16) * kN + i * 16 + lane / 16 * 4) = acc[i][0];
  __syncthreads();
  const int place = threadIdx.x / kN, col = threadIdx.x % kN;
  const bool mine = place < count;
  const int64_t n = n0 + col;
  const float* const from = sums + index[mine ? place : 0] * kN + col;
  float z = 0.f;
#pragma unroll
  for (int v = 0; v < gemm::kFewWaves; ++v) z += from[v * kFewRows * kN];
  if (mine && of.kept.z != nullptr && n < of.kept.pitch) of.kept.z[place * of.kept.pitch + n] = z;
  if (mine && n == target[place]) of.at_target[place] = z;
  if (n >= p.N) z = -__builtin_inff();
  const float top = group_max<32>(z), sum = group_sum<32>(gemm::exp_of<sizeof(T) == 2>(z - base_of(top)));
  if (mine && col == 0) of.part[place * of.tiles + blockIdx.x] = float2{top, sum};
}

template <typename T>
int run_sums_rows(const Product& p, const SumsOf& of, const FewTokens& few, hipStream_t s) {
  static_assert(kFewRows * kRowsColumns == 64 * gemm::kFewWaves, "a thread for each sum");
  hipLaunchKernelGGL((sums_rows_kernel<T, 1>), dim3((unsigned)ceil_div(p.N, kRowsColumns)), dim3(64 * gemm::kFewWaves), 0, s, p, of, few);
  MHC_CHECK_LAUNCH("sums_rows_kernel");
  return MHC_OK;
}

template <typename T, bool HALVES, int BM, int BN, int WM, int WN, int NS>
int launch_sums(const Product& p, const RowsOf& rows, const int* live, const SumsOf& of, const Halves& halves, hipStream_t s) {
  hipLaunchKernelGGL((sums_tile_kernel<T, HALVES, BM, BN, WM, WN, NS>), dim3((unsigned)(ceil_div(p.M, BM) * ceil_div(p.N, BN))), dim3(64 * WM * WN),
                     0, s, p, rows, live, of, halves);
  MHC_CHECK_LAUNCH("sums_tile_kernel");
  return MHC_OK;
}

template <typename T, bool HALVES = false>
int run_sums(Product p, const RowsOf& rows, const Cut& c, const int* live, const SumsOf& of, const Halves& halves, hipStream_t s) {
  using gemm::kRowWaves;
  p.splits = 1;
  p.kper = c.kper;
  switch (c.tile) {
    case 0: return launch_sums<T, HALVES, 256, 256, 2, 4, 2>(p, rows, live, of, halves, s);
    case 1: return launch_sums<T, HALVES, 128, 256, 2, 4, 2>(p, rows, live, of, halves, s);
    case 2: return launch_sums<T, HALVES, 128, 128, kRowWaves<T>, 2, 2>(p, rows, live, of, halves, s);
    case 3: return launch_sums<T, HALVES, 64, 128, kRowWaves<T>, 2, 3>(p, rows, live, of, halves, s);
    default: return launch_sums<T, HALVES, 64, 64, 4, 1, 3>(p, rows, live, of, halves, s);
  }
}

// Up to 64 tokens whose rows of x can be read where they lie; c.tile is one of 64 rows.
template <typename T>
int run_sums_few(Product p, const Cut& c, const SumsOf& of, const FewTokens& few, hipStream_t s) {
  using gemm::kRowWaves;
  p.splits = 1;
  p.kper = c.kper;
  if (c.tile == 3)
    hipLaunchKernelGGL((sums_few_kernel<T, 128, kRowWaves<T>, 2, 3>), dim3((unsigned)ceil_div(p.N, 128)), dim3(64 * kRowWaves<T> * 2), 0, s, p, of, few);
  else
    hipLaunchKernelGGL((sums_few_kernel<T, 64, 4, 1, 3>), dim3((unsigned)ceil_div(p.N, 64)), dim3(256), 0, s, p, of, few);
  MHC_CHECK_LAUNCH("sums_few_kernel");
  return MHC_OK;
}

template <typename T, bool AK, bool BK, bool SUMS, typename O, int BM, int BN, int WM, int WN, int NS, typename Then>
int launch_live(const Product& p, const int* live, int64_t width, const Then& then, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(p.M, BM) * ceil_div(p.N, BN)), (unsigned)p.splits), block(64 * WM * WN);
  hipLaunchKernelGGL((live_tile_kernel<T, AK, BK, BM, BN, WM, WN, NS, SUMS, O, Then>), grid, block, 0, s, p, live, width, then);
  MHC_CHECK_LAUNCH("live_tile_kernel");
  return MHC_OK;
}

// width: of the outputs' rows; part: the sums of a reduction's parts, if it is split (and not SUMS)
template <typename T, bool AK, bool BK, bool SUMS, typename O = T, typename Then>
int run_live(Product p, const Cut& c, const int* live, int64_t width, const Then& then, float* part, hipStream_t s) {
  using gemm::kRowWaves;
  const Epilogue e = p.e;
  p.splits = c.splits;
  p.kper = c.kper;
  if (c.splits > 1 && !SUMS) p.e = Epilogue{nullptr, nullptr, part, nullptr, MHC_ACT_NONE, 1};
  int rc;
  switch (c.tile) {
    case 0: rc = launch_live<T, AK, BK, SUMS, O, 256, 256, 2, 4, 2>(p, live, width, then, s); break;
    case 1: rc = launch_live<T, AK, BK, SUMS, O, 128, 256, 2, 4, 2>(p, live, width, then, s); break;
    case 2: rc = launch_live<T, AK, BK, SUMS, O, 128, 128, kRowWaves<T>, 2, 2>(p, live, width, then, s); break;
    case 3: rc = launch_live<T, AK, BK, SUMS, O, 64, 128, kRowWaves<T>, 2, 3>(p, live, width, then, s); break;
    default: rc = launch_live<T, AK, BK, SUMS, O, 64, 64, 4, 1, 3>(p, live, width, then, s); break;
  }
  if (rc != MHC_OK || c.splits == 1 || SUMS) return rc;
  return gemm::launch_join<T>(e, part, c.splits, p.M, p.N, s);
}

// The launches of one type, each compiled in a file of its own.
struct Runs {
  int (*sums)(Product p, const RowsOf& rows, const Cut& c, const int* live, const SumsOf& of, const Halves& halves, hipStream_t s);
  int (*sums_rows)(const Product& p, const SumsOf& of, const FewTokens& few, hipStream_t s);
  int (*sums_few)(Product p, const Cut& c, const SumsOf& of, const FewTokens& few, hipStream_t s);
  int (*dz)(const Product& p, const Cut& c, const int* live, int64_t width, const Gradient& g, hipStream_t s);
  int (*dz_of_kept)(const Gradient& g, const Kept& kept, void* dz, int64_t width, int64_t T, int64_t N, const int* live, hipStream_t s);
  int (*dx)(const Product& p, const Cut& c, const int* live, hipStream_t s);
  int (*dw)(const Product& p, const Cut& c, const int* live, const ScaledBy& by, float* part, hipStream_t s);
  int (*joint)(const Joint& j, const int* live, hipStream_t s);  // of 16-bit operands
};
const Runs& runs_f32();
const Runs& runs_bf16();
const Runs& runs_f16();

// dx and dW of up to few_tokens() tokens whose logits were kept by the vector unit
// (16 x 32000 x 4096 fp32 417 and 507 us, bf16 285 and 250, 8 tokens 209 and 238).
inline int few_tokens(int dtype) { return dtype == kF32 ? 16 : 8; }
size_t few_bytes(const mhc_linear_ce_args& a);
int run_few(const mhc_linear_ce_args& a, const State& st, const float* dloss, float grad_scale, void* dx, void* dw, char* ws, hipStream_t s);

// of rows of fp16 parts for fp32 logits
int run_sums_halves(const Product& p, const Cut& c, const int* live, const SumsOf& of, const Halves& halves, hipStream_t s);
int run_dz_halves(const Product& p, const Cut& c, const int* live, int64_t width, const Gradient& g, const Halves& halves, hipStream_t s);
// of logits that were kept: dz's parts of `rows` tokens and N columns, and its products, whose operands are the high parts
int run_parts(const Gradient& g, const Kept& kept, const Halves& halves, const Parts& parts, int64_t rows, int64_t N, const int* live, hipStream_t s);
int run_dx_halves(const Product& p, const void* a_low, const void* b_low, const uint32_t* tops, const Cut& c, const int* live, hipStream_t s);
int run_dw_halves(const Product& p, const void* a_low, const void* b_low, const uint32_t* tops, const Cut& c, const int* live, const ScaledBy& by,
                  float* part, hipStream_t s);

template <typename T>
int run_dz(const Product& p, const Cut& c, const int* live, int64_t width, const Gradient& g, hipStream_t s) {
  return run_live<T, true, true, false>(p, c, live, width, GradientOf<sizeof(T) == 2>{g}, nullptr, s);
}
template <typename T>
int run_dz_of_kept(const Gradient& g, const Kept& kept, void* dz, int64_t width, int64_t rows, int64_t N, const int* live, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(rows, 32) * ceil_div(width, 256)));
  hipLaunchKernelGGL((dz_kernel<T>), grid, dim3(256), 0, s, g, kept, static_cast<T*>(dz), width, N, live);
  MHC_CHECK_LAUNCH("dz_kernel");
  return MHC_OK;
}
template <typename T>
int run_dx(const Product& p, const Cut& c, const int* live, hipStream_t s) {
  return run_live<T, true, false, true>(p, c, live, p.N, gemm::AsTheyAre{}, nullptr, s);
}
template <typename T>
int run_dw(const Product& p, const Cut& c, const int* live, const ScaledBy& by, float* part, hipStream_t s) {
  return run_live<T, false, false, false>(p, c, live, p.N, by, part, s);
}

template <typename T>
const Runs& runs_of() {
  if constexpr (sizeof(T) == 2) {
    static const Runs r = {run_sums<T, false>, run_sums_rows<T>, run_sums_few<T>, run_dz<T>, run_dz_of_kept<T>, run_dx<T>, run_dw<T>, run_joint<T>};
    return r;
  } else {
    static const Runs r = {run_sums<T, false>, run_sums_rows<T>, run_sums_few<T>, run_dz<T>, run_dz_of_kept<T>, run_dx<T>, run_dw<T>, nullptr};
    return r;
  }
}

}  // namespace ce
}  // namespace mhc
