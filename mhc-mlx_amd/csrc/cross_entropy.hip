// Softmax cross entropy of logits z = x W^T, and its gradient.  Without gradients
// the logits are not stored; with them up to 2 GiB are, in fp32.
//
//   lp_t = z[t, y_t] - log sum_v exp z[t, v];  loss = -sum_t w_t lp_t / D
//   dz = w_t / D (softmax(z) - [v = y_t]);  dx = dz W;  dW = dz^T x
//
// Tokens that count for nothing (weight 0, or the ignored target) are left out
// at the start: the others' rows of x are brought together, and every product
// below takes as many rows as there are of them, which only the device knows
// (sums_rows_kernel multiplies all of up to 16 and takes the live ones' sums).
//
// Forward: the logits' product keeps of each tile a largest value and a sum of
// exponentials for each row, which are joined.  Backward: the vocabulary goes
// by in pieces; the logits of a piece are formed again and become its dz, of
// which dx (summed up in fp32 over the pieces) and the piece's rows of dW are
// products.  Where the logits are wide and few enough to be kept (keeps_logits),
// dz is read from them, which saves the fourth product.
#include "mhc_ce.hpp"
#include "mhc_operand.hpp"
#include "mhc_plan.hpp"

namespace mhc {
namespace {

using ce::Gradient;
using ce::ScaledBy;
using ce::State;
using gemm::Cut;
using gemm::Epilogue;
using gemm::Operand;
using gemm::Product;
using gemm::padded;
using gemm::up256;

// Threads of the kernels of one workgroup: few for few tokens.
constexpr int kFew = 256, kMany = 1024;

// dz of a piece of the vocabulary takes at most about this much: the two of
// them under way then stay near what the last-level cache holds, and few pieces
// read and write dx's sums (6144 of 8192 tokens, 50257 columns, C = 4096 bf16: 64
// MB a piece 9.44 ms, 128 8.27, 256 8.27, 512 8.64, 1024 9.39; three in four of 4096,
// 131072, 1024: 3.54, 3.39, 3.28, 3.35, 3.41; from logits that were kept, 6144
// tokens: 128 6.80, 256 6.91, 512 7.00, and 4096 x 100000 x 1024 3.17, 3.13, 3.11).
constexpr int64_t kPieceBytes = 256 << 20;

// The live tokens, in order, with their weights, and D: one workgroup, whose
// threads have kRun tokens each of a chunk.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void ce_live_kernel(const mhc_linear_ce_args a, float* logp, const State s) {
  constexpr int kRun = 8, kWaves = THREADS / kWave;
  __shared__ int counts[kWaves];
  __shared__ double sums[kWaves];
  __shared__ float tops[kWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int total = 0;  // of the chunks before
  double sum = 0;
  float top = 0.f;
  for (int64_t first = 0; first < a.T; first += THREADS * kRun) {
    const int64_t t0 = first + threadIdx.x * kRun;
    float w[kRun];
    int64_t y[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) {  // (tokens past the last one read it once more: a load under a condition would wait for itself)
      const int64_t t = min(t0 + k, a.T - 1);
      w[k] = ce::weight_of(a, t);
      y[k] = a.targets[t];
    }
    int count = 0;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (t0 + k >= a.T || y[k] == a.ignore_index) w[k] = 0.f;
      count += w[k] != 0.f;
      sum += (double)w[k];
      top = fmaxf(top, fabsf(w[k]));
    }
    int before = count;  // of the wave's lanes up to this one
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int up = __shfl_up(before, d);
      if (lane >= d) before += up;
    }
    __syncthreads();
    if (lane == kWave - 1) counts[wave] = before;
    __syncthreads();
    int place = total + before - count;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      if (v < wave) place += counts[v];
      total += counts[v];
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (t0 + k >= a.T) break;
      const bool live = w[k] != 0.f;
      s.pos[t0 + k] = live ? place : -1;
      if (!live) {
        logp[t0 + k] = 0.f;
        continue;
      }
      s.index[place] = (int)(t0 + k);
      s.target[place] = y[k] >= 0 && y[k] < a.V ? (int)y[k] : -1;
      s.coef[place] = w[k];
      ++place;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  top = group_max<kWave>(top);
  if (lane == 0) {
    sums[wave] = sum;
    tops[wave] = top;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int v = 1; v < kWaves; ++v) {
    sum += sums[v];
    top = fmaxf(top, tops[v]);
  }
  ce::store_head(a, s, total, sum, top);
}

// the live rows of x, one after the other, in whole chunks of 16 bytes with zeros after the last element
template <typename T>
__global__ __launch_bounds__(256) void ce_gather_kernel(const T* x, int64_t ld, T* to, const int* live, const int* index, int64_t C, uint32_t chunks) {
  constexpr int kE = 16 / (int)sizeof(T);
  const int64_t total = (int64_t)*live * chunks;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
    const int64_t row = at / chunks, k = at % chunks * kE;
    const T* const p = x + index[row] * ld + k;
    u32x4 v = {0, 0, 0, 0};
    if (k + kE <= C) {
      __builtin_memcpy(&v, p, 16);
    } else {
      T e[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j) e[j] = k + j < C ? p[j] : (T)0;
      __builtin_memcpy(&v, e, 16);
    }
    reinterpret_cast<u32x4*>(to)[at] = v;
  }
}

// four values of a row from element k on, zeros past its end
MHC_DEV f32x4 four_of(const float* row, int k, int C) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (k + 4 <= C) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k + j < C) v[j] = row[k + j];
  }
  return v;
}

// Rows of fp32 as rows of fp16 parts (see ce::Halves) in an order: of x or W for
// the logits, whose products of parts are one, or each part once; each in `wide`
// elements, zeros after the last.  The live rows of x (index given), or all of `rows`.  A wave for each
// row, of which it keeps HELD times 256 elements in registers and reads those
// beyond again (32768 x 1024: 335 MB in 51 us, 6.5 TB/s).
enum Order { kOfX, kOfW, kOnce };  // [high, low, high], [high, high, low], [high, low]

template <int ORDER, int HELD>
__global__ __launch_bounds__(256) void ce_halves_kernel(const float* x, int64_t ld, _Float16* to, float* scales, const int* live, const int* index,
                                                        int64_t rows, int C, int wide) {
  constexpr int kStep = 4 * kWave;
  const int k0 = threadIdx.x % kWave * 4;
  if (live != nullptr) rows = *live;
  for (int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave; r < rows; r += (int64_t)gridDim.x * 4) {
    const float* const row = x + (index != nullptr ? index[r] : r) * ld;
    f32x4 held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = four_of(row, k0 + i * kStep, C);
    float top = 0.f;
    const auto look = [&](const f32x4& v) {  // (as bit patterns, of which NaN's are the largest)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, top), __builtin_bit_cast(uint32_t, fabsf(v[j]))));
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) look(held[i]);
    for (int k = k0 + HELD * kStep; k < C; k += kStep) look(four_of(row, k, C));
    uint32_t bits = __builtin_bit_cast(uint32_t, top);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, d));
    const uint32_t up = ce::lift_of(bits);  // (the logits of a row with an infinity are NaN)
    const float by = ce::lift_by(up);
    if (k0 == 0) scales[r] = ce::lower_by(up);
    _Float16* const out = to + r * (ORDER == kOnce ? 2 : 3) * wide;
    const auto store = [&](int k, const f32x4& v) {
      f16x4 high, low;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        high[j] = (_Float16)(v[j] * by);
        low[j] = (_Float16)(v[j] * by - (float)high[j]);
      }
      *reinterpret_cast<f16x4*>(out + k) = high;  // (wide is a multiple of eight)
      *reinterpret_cast<f16x4*>(out + wide + k) = ORDER == kOfW ? high : low;
      if constexpr (ORDER != kOnce) *reinterpret_cast<f16x4*>(out + 2 * wide + k) = ORDER == kOfW ? low : high;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (k0 + i * kStep < wide) store(k0 + i * kStep, held[i]);
    for (int k = k0 + HELD * kStep; k < wide; k += kStep) store(k, four_of(row, k, C));
  }
}

// A row's parts to its sums, and its log probability, put together in fp64
// (log sum = e log 2 + log m with m around 1: the fp32 part stays below 0.35):
// WAVES for each row, more for a few rows of many parts.  (The weights become those over the largest one here.)
template <int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void ce_rows_kernel(const State s, const float2* part, const float* at_target, int64_t tiles,
                                                                                 float* logp, double* terms) {
  constexpr int kRows = WAVES == 1 ? 4 : 1, kThreads = WAVES * kWave;  // of a workgroup, and of a row
  __shared__ float lds[2][WAVES];
  const int at = threadIdx.x % kThreads, wave = at / kWave;
  const int64_t rows = *s.head;
  for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kThreads; r < rows; r += (int64_t)gridDim.x * kRows) {
    float top = -__builtin_inff();
#pragma unroll 4
    for (int64_t k = at; k < tiles; k += kThreads) top = fmaxf(top, part[r * tiles + k].x);
    top = group_max<kWave>(top);
    if constexpr (WAVES > 1) {
      lds[0][wave] = top;
      __syncthreads();
#pragma unroll
      for (int v = 0; v < WAVES; ++v) top = fmaxf(top, lds[0][v]);
    }
    const float base = ce::base_of(top);
    float sum = 0.f;
#pragma unroll 4
    for (int64_t k = at; k < tiles; k += kThreads) {
      const float2 one = part[r * tiles + k];
      sum += one.y * expf(one.x - base);
    }
    sum = wave_sum(sum);
    if constexpr (WAVES > 1) {
      lds[1][wave] = sum;
      __syncthreads();
      sum = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) sum += lds[1][v];
    }
    if (at != 0) continue;
    const float z = s.target[r] < 0 ? __builtin_nanf("") : at_target[r];
    int e;
    float m = frexpf(sum, &e);
    if (m < 0.70710678f) m *= 2.f, --e;
    const double lp = (double)z - (double)top - ((double)e * 0.6931471805599453 + (double)logf(m));
    s.top[r] = top;
    s.inv[r] = 1.f / sum;
    logp[s.index[r]] = (float)lp;
    const float coef = s.coef[r] / reinterpret_cast<const float*>(s.head)[2];
    s.coef[r] = coef;
    terms[r] = (double)coef * lp;
  }
}

// loss = -(largest weight / D) sum of the terms: one workgroup, a fixed order.
// (A launch of its own: counting the workgroups of the one before, so that its
// last one goes on, takes a fence of each, and 200 us for 8192 rows.)
template <int THREADS>
__global__ __launch_bounds__(THREADS) void ce_loss_kernel(const State s, const double* terms, float* loss) {
  __shared__ double lds[THREADS / kWave];
  const int rows = *s.head;
  double sum = 0;
#pragma unroll 8
  for (int r = threadIdx.x; r < rows; r += THREADS) sum += terms[r];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) sum += lds[w];
  loss[0] = rows == 0 ? 0.f : (float)(-sum * (double)reinterpret_cast<float*>(s.head)[2] / *reinterpret_cast<double*>(s.head + 4));
}

// dx of every token from the live ones' sums, of each part of the reduction, scaled: zeros for the others
template <typename T>
__global__ __launch_bounds__(256) void ce_scatter_kernel(const float* sums, int parts, const State s, const float* dloss, float scale, T* dx, int64_t tokens,
                                                         int64_t C, uint32_t groups) {
  constexpr int V = 8;
  const float by = reinterpret_cast<const float*>(s.head)[1] * (dloss != nullptr ? dloss[0] : 1.f) * scale;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < tokens * groups; at += (int64_t)gridDim.x * 256) {
    const int64_t t = at / groups, n = at % groups * V;
    const int left = (int)min((int64_t)V, C - n), pos = s.pos[t];
    float z[V] = {};
    if (pos >= 0) {
#pragma unroll 4
      for (int q = 0; q < parts; ++q) {
        const float* const p = sums + (q * tokens + pos) * C + n;
        float v[V];
        if (left == V) gemm::take<true>(p, v, V);
        else gemm::take<false>(p, v, left);
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] += v[k];
      }
#pragma unroll
      for (int k = 0; k < V; ++k) z[k] *= by;
    }
    if (left == V) gemm::put<true>(dx + t * C + n, z, V);
    else gemm::put<false>(dx + t * C + n, z, left);
  }
}

const ce::Runs& runs_of(int dtype) { return dtype == kF32 ? ce::runs_f32() : dtype == kBF16 ? ce::runs_bf16() : ce::runs_f16(); }

// columns of the vocabulary whose parts take at most kPieceBytes
int64_t halves_piece(const mhc_linear_ce_args& a) {
  const int64_t most = std::max<int64_t>(256, kPieceBytes / (6 * padded(a.C, kF16)) / 256 * 256);
  return std::min(a.V, ceil_div(ceil_div(a.V, ceil_div(a.V, most)), 256) * 256);
}

// Whether fp32 logits are formed of fp16 parts: where their products and the
// way of W into them (ten bytes for each of its elements at 4.5 TB/s) are
// estimated shorter than fp32 products (512 x 32768 x 1024 165 and 176 us, 4096 x
// 8000 x 2048 387 and 696; but 256 x 32768 x 1024 149 and 111).
bool in_halves(const mhc_linear_ce_args& a) {
  if (a.dtype != kF32 || a.T <= ce::kFewRows) return false;
  const int64_t piece = halves_piece(a), wide = padded(a.C, kF16);
  if (6 * wide > gemm::kMaxRowBytes) return false;
  const float pieces = (float)ceil_div(a.V, piece);
  const float halves = 4.f + pieces * (4.f + gemm::cut_of(a.T, piece, 3 * wide, kF16, true, true, 1).us) + (float)(a.V * wide) * 10e-6f / 4.5f;
  return halves < gemm::cut_of(a.T, a.V, a.C, kF32, true, true, 1).us;
}

// What `count` parts of each of x's rows and of a piece's rows of W take.
struct HalvesPlan {
  int64_t wide;  // elements of a part of a row
  size_t x, w;   // bytes, with the rows' scales
};

HalvesPlan plan_halves(const mhc_linear_ce_args& a, int64_t piece, int count) {
  const int64_t wide = padded(a.C, kF16);
  const auto bytes = [&](int64_t rows) { return up256((size_t)(rows * count * wide) * 2) + up256((size_t)rows * 4); };
  return {wide, bytes(a.T), bytes(piece)};
}

struct FwdPlan {
  Cut cut;
  int64_t tiles;
  int64_t piece;  // columns of the vocabulary at a time
  bool direct;    // the live rows of x are read where they lie
  bool few;       // and found by the products' launch
  bool rows;      // which is that for up to kFewRows tokens, else one of tiles
  size_t x, w, part, at_target, total;  // bytes; terms come last
};

// What reading `bytes` at a rate in GB/ms takes of `blocks` workgroups, of which
// `room` are on the card at once: a last round that is not full costs `share` of
// what it is not full by.
float reading_us(int64_t bytes, float rate, int64_t blocks, int64_t room, float share) {
  const float rounds = (float)blocks / (float)room, full = std::max(1.f, ceilf(rounds) / std::max(1.f, rounds));
  return (float)bytes / (rate * 1e6f) * (1.f + share * (full - 1.f));
}

// Whether up to kFewRows tokens go to sums_rows_kernel: all of fp32 rows, whose
// tiles are bound by their products (the call's kernels, 8 tokens: 32000 x 2048 56
// us, tiles 98), and 16-bit ones unless tiles of 64 rows, whose start is longer
// and of which fewer are on the card at once, are estimated faster (rows and
// tiles, 8 tokens bf16: 4524 x 2240 11 and 23 us, 16384 x 1024 13 and 17, 72999 x
// 2624 73 and 83, 151936 x 2048 118 and 137, 256000 x 2048 191 and 209; but 32000 x
// 2048 31 and 29, 32000 x 4096 57 and 47, 50257 x 4096 90 and 83, 128256 x 4096 203
// and 192.  Of 35 sizes three take the one that is more than 3 % slower, by a
// tenth at most: 16384 x 4096 35 and 33, 24576 x 2048 27 and 25, 256000 x 768 87 and 82).
bool takes_rows(const mhc_linear_ce_args& a, const Cut& c) {
  if (a.dtype == kF32 || c.tile < 3) return true;
  const int64_t cus = device_cu_count(), bytes = a.V * a.C * gemm::elem_bytes(a.dtype);
  const float rows = std::max(4.f, reading_us(bytes, 5.7f, ceil_div(a.V, ce::kRowsColumns), 3 * cus, 0.25f));
  return rows <= std::max(c.us + 2.f, reading_us(bytes, 5.6f, ceil_div(a.V, c.tile == 3 ? 128 : 64), 2 * cus, 0.5f));
}

FwdPlan plan_fwd(const mhc_linear_ce_args& a) {
  constexpr int kBn[] = {256, 256, 128, 128, 64};
  FwdPlan p;
  const int e = gemm::elem_bytes(a.dtype);
  p.direct = p.few = p.rows = false;
  if (a.T <= ce::kFewRows) {
    p.cut = gemm::cut_of(a.T, a.V, a.C, a.dtype, true, true, 1);
    p.rows = takes_rows(a, p.cut);
    p.few = p.direct = true;
    p.piece = a.V;
    p.x = gemm::pack_bytes(a.x, a.T, a.ldx, a.C, a.dtype);
    p.w = gemm::pack_bytes(a.w, a.V, a.ldw, a.C, a.dtype);
  } else if (in_halves(a)) {
    p.piece = halves_piece(a);
    const HalvesPlan h = plan_halves(a, p.piece, 3);
    p.cut = gemm::cut_of(a.T, p.piece, 3 * h.wide, kF16, true, true, 1);
    p.x = h.x;
    p.w = h.w;
  } else {
    p.piece = a.V;
    p.cut = gemm::cut_of(a.T, a.V, a.C, a.dtype, true, true, 1);
    p.direct = gemm::in_words(a.x, a.ldx, a.C, e) && ((a.T - 1) * a.ldx + a.C) * e < ((int64_t)1 << 31);
    p.few = p.direct && a.T <= 64 && p.cut.tile >= 3;
    p.x = p.direct ? 0 : up256((size_t)(a.T * padded(a.C, a.dtype)) * e);
    p.w = gemm::pack_bytes(a.w, a.V, a.ldw, a.C, a.dtype);
  }
  p.tiles = ceil_div(a.V, p.rows ? ce::kRowsColumns : kBn[p.cut.tile]);  // (pieces are whole tiles, but for the last)
  p.part = up256((size_t)(a.T * p.tiles) * sizeof(float2));
  p.at_target = up256((size_t)a.T * sizeof(float));
  p.total = p.x + p.w + p.part + p.at_target + (size_t)a.T * sizeof(double);
  return p;
}

// the parts of rows to `to`, their scales after them
int run_halves(Order order, const void* x, int64_t ld, char* to, const float** scales, const State* live, int64_t rows, int64_t C, int64_t wide,
               hipStream_t s) {
  float* const at = reinterpret_cast<float*>(to + up256((size_t)(rows * (order == kOnce ? 2 : 3) * wide) * 2));
  *scales = at;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(rows, 4), device_cu_count() * 16));
  const int *const count = live != nullptr ? live->head : nullptr, *const index = live != nullptr ? live->index : nullptr;
  const auto held = [&](auto kernel4, auto kernel16) { return C <= 1024 ? kernel4 : kernel16; };
  const auto kernel = order == kOfX   ? held(ce_halves_kernel<kOfX, 4>, ce_halves_kernel<kOfX, 16>)
                      : order == kOfW ? held(ce_halves_kernel<kOfW, 4>, ce_halves_kernel<kOfW, 16>)
                                      : held(ce_halves_kernel<kOnce, 4>, ce_halves_kernel<kOnce, 16>);
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, static_cast<const float*>(x), ld,
                     reinterpret_cast<_Float16*>(to), at, count, index, rows, (int)C, (int)wide);
  MHC_CHECK_LAUNCH("ce_halves_kernel");
  return MHC_OK;
}

// Whether the forward keeps the logits for the backward, which forms them again
// else: from a width on at which their way through memory and back is shorter
// than their product (4096 x 100000 bf16 kept and formed again, C = 512 2.20
// and 2.04 ms, 1024 3.13 and 3.34, 2048 5.02 and 5.88; 6144 x 50257, 4096 6.8
// and 8.3; 2000 x 32768 fp32, C = 64 0.449 and 0.433, 256 0.71 and 0.83, 2048
// 2.62 and 4.25), and up to an amount that a card of 288 GB does not miss.
constexpr int64_t kKeepBytes = (int64_t)2 << 30;

bool keeps_logits(const mhc_linear_ce_args& a) {
  return (a.T <= ce::few_tokens(a.dtype) || a.C >= (a.dtype == kF32 ? 256 : 768)) && a.T * ce::kept_pitch(a.V) * 4 <= kKeepBytes;
}

struct BwdPlan {
  int64_t piece;   // columns of the vocabulary
  bool parts;      // dx and dW are formed of fp16 parts
  bool joint;      // a piece's dx and dW go with the next one's dz
  Cut dz, dx, dw;  // dx.splits: parts of its reduction, each with sums of its own over all pieces
  HalvesPlan halves;
  size_t x, w, of_dz, sums, part, total;  // bytes; two of of_dz where joint
};

// columns of a piece whose dz takes kPieceBytes, at e bytes
int64_t piece_of(const mhc_linear_ce_args& a, int64_t e) {
  const int64_t pieces = std::max<int64_t>(1, ceil_div(a.T * a.V * e, kPieceBytes));
  return std::min(a.V, ceil_div(ceil_div(a.V, pieces), 256) * 256);
}

// Whether dx and dW of fp32 operands are formed of fp16 parts, from logits that
// were kept: where that is estimated shorter, with eight bytes more of each of
// dz's elements and eight of each of W's, and three launches (the whole call in
// parts and in fp32 tiles, C = 1024 and 32768 columns: 128 tokens 294 and 282 us,
// 520 665 and 742, 1000 887 and 1080; 2000 x 32768 x 256 890 and 713; 500 x 500 x
// 4096 169 and 155; 4096 x 100000 x 1024 9.9 and 11.8 ms).
bool in_parts(const mhc_linear_ce_args& a) {
  if (a.dtype != kF32 || a.logits == nullptr || 6 * padded(a.C, kF16) > gemm::kMaxRowBytes) return false;
  const int64_t wide = padded(a.C, kF16), of_parts = std::min(piece_of(a, 8), halves_piece(a)), plain = piece_of(a, 4);
  const float pieces = (float)ceil_div(a.V, of_parts);
  const float parts = pieces * (20.f + gemm::cut_of(a.T, a.C, 3 * of_parts, kF16, true, false).us + gemm::cut_of(of_parts, a.C, 3 * a.T, kF16, false, false).us) +
                      (float)(a.V * wide) * 8e-6f / 5.5f + (float)(a.T * a.V) * 8e-6f / 3.f;
  return parts < (float)ceil_div(a.V, plain) * (gemm::cut_of(a.T, a.C, plain, kF32, true, false).us + gemm::cut_of(plain, a.C, a.T, kF32, false, false).us);
}

bool few(const mhc_linear_ce_args& a) { return a.logits != nullptr && a.T <= ce::few_tokens(a.dtype); }

BwdPlan plan_bwd(const mhc_linear_ce_args& a, bool dx, bool dw) {
  BwdPlan p = {};
  const int64_t e = gemm::elem_bytes(a.dtype);
  if (few(a)) {
    p.total = ce::few_bytes(a);
    return p;
  }
  p.parts = in_parts(a);
  p.piece = piece_of(a, p.parts ? 8 : e);
  if (p.parts) {
    p.piece = std::min(p.piece, halves_piece(a));
    p.halves = plan_halves(a, p.piece, 2);
    p.dx = gemm::cut_of(a.T, a.C, 3 * p.piece, kF16, true, false);
    p.dw = gemm::cut_of(p.piece, a.C, 3 * a.T, kF16, false, false);
    // (a part of a reduction takes its k of all three products)
    const auto third = [](Cut& c, int64_t K) {
      const int kK = gemm::stage_k(kF16), deep = (int)ceil_div(K, kK), per = (int)ceil_div(deep, std::min(c.splits, deep));
      c.splits = (int)ceil_div(deep, per), c.kper = per * kK;
    };
    third(p.dx, p.piece);
    third(p.dw, a.T);
    p.of_dz = up256((size_t)(a.T * padded(p.piece, kF16)) * 2);
    if (dx) p.sums = up256((size_t)(p.dx.splits * a.T * a.C) * sizeof(float));
    p.part = dw ? up256(gemm::part_bytes(p.dw, p.piece, a.C)) : 0;
    p.total = 4 * p.of_dz + p.sums + p.halves.x + p.halves.w + p.part + ce::Parts::top_words(a.T, p.piece) * sizeof(uint32_t);
    return p;
  }
  if (a.logits != nullptr) {
    p.dz = Cut{};
  } else if (in_halves(a)) {
    p.piece = std::min(p.piece, halves_piece(a));
    p.halves = plan_halves(a, p.piece, 3);
    p.dz = gemm::cut_of(a.T, p.piece, 3 * p.halves.wide, kF16, true, true, 1);
  } else {
    p.dz = gemm::cut_of(a.T, p.piece, a.C, a.dtype, true, true, 1);
  }
  // (whichever is asked for: a gradient does not depend on that)
  p.dx = gemm::cut_of(a.T, a.C, p.piece, a.dtype, true, false);
  p.dw = gemm::cut_of(p.piece, a.C, a.T, a.dtype, false, false);
  if (a.dtype != kF32 && gemm::most_rows(true, a.C, a.dtype) >= 256) {
    // One launch of 256 x 256 tiles: as long as all of its stages take on all CUs (a twentieth more for its end), if dx's
    // reduction is cut so that no tile takes more than half of that, and at least as long as its longest tile.
    const gemm::TileCost& c = gemm::kTiles[0];
    const float cus = (float)device_cu_count();
    const int kK = gemm::stage_k(a.dtype), deep = (int)ceil_div(p.piece, kK), low = (int)ceil_div(a.T, kK), of_c = (int)ceil_div(a.C, kK);
    const float mt = (float)ceil_div(a.T, 256), mv = (float)ceil_div(p.piece, 256), mc = (float)ceil_div(a.C, 256);
    const float units = mt * mc * deep + mv * mc * low + (p.piece < a.V && a.logits == nullptr ? mt * mv * of_c : 0.f);
    const int splits = std::min(16, std::max(1, (int)ceilf(2.f * deep * cus / units))), per = (int)ceil_div(deep, splits);
    const float us = c.ends + std::max(1.05f * units / cus * gemm::stage_us(c, a.dtype, 1.f), std::max(std::max(per, low), of_c) * gemm::stage_us(c, a.dtype, 0.f));
    const float apart = p.dx.us + p.dw.us + (p.piece < a.V ? p.dz.us : 0.f);
    p.joint = us < apart;
    if (p.joint) p.dx.splits = (int)ceil_div(deep, per), p.dx.kper = per * kK;
  }
  p.x = up256((size_t)(a.T * padded(a.C, a.dtype) * e));
  p.w = gemm::pack_bytes(a.w, a.V, a.ldw, a.C, a.dtype);
  p.of_dz = up256((size_t)(a.T * padded(p.piece, a.dtype) * e));
  if (dx) p.sums = up256((size_t)(p.dx.splits * a.T * a.C) * sizeof(float));
  p.part = dw && !p.joint ? gemm::part_bytes(p.dw, p.piece, a.C) : 0;
  p.total = p.x + p.w + p.of_dz * (p.joint && p.piece < a.V ? 2 : 1) + p.sums + p.halves.x + p.halves.w + p.part;
  return p;
}

// The gradients from logits that were kept, all products of fp16 parts; sums: dx's, of every part of its reduction.
int run_bwd_parts(const mhc_linear_ce_args& a, const BwdPlan& p, const State& st, const float* dloss, float grad_scale, bool dx, void* dw, char* ws,
                  float*& sums, hipStream_t s) {
  const auto next = [&ws](size_t bytes) { return ws += bytes, ws - bytes; };
  const auto halves_of_dz = [&] { return reinterpret_cast<_Float16*>(next(p.of_dz)); };
  ce::Parts parts = {halves_of_dz(), halves_of_dz(), halves_of_dz(), halves_of_dz(), nullptr, nullptr, nullptr, nullptr, 0};
  sums = reinterpret_cast<float*>(next(p.sums));
  char *const of_x = next(p.halves.x), *const of_w = next(p.halves.w);
  float* const part = reinterpret_cast<float*>(next(p.part));
  parts.row = reinterpret_cast<uint32_t*>(ws);
  parts.col = parts.row + a.T;
  parts.rows = parts.col + p.piece;
  parts.cols = parts.rows + a.T * ceil_div(p.piece, 256);
  const int64_t wide = p.halves.wide;
  const ScaledBy by = {reinterpret_cast<const float*>(st.head) + 1, dloss, grad_scale};
  const ce::Kept kept = {a.logits, ce::kept_pitch(a.V)};
  ce::Halves halves;
  if (const int rc = run_halves(kOnce, a.x, a.ldx, of_x, &halves.x, &st, a.T, a.C, wide, s)) return rc;
  for (int64_t v0 = 0; v0 < a.V; v0 += p.piece) {
    const int64_t n = std::min(p.piece, a.V - v0);
    if (const int rc = run_halves(kOnce, static_cast<const float*>(a.w) + v0 * a.ldw, a.ldw, of_w, &halves.w, nullptr, n, a.C, wide, s)) return rc;
    parts.pitch = padded(n, kF16);
    const ce::Gradient g = {st.target, st.coef, st.top, st.inv, v0, 1.f};
    if (const int rc = ce::run_parts(g, kept, halves, parts, a.T, n, st.head, s)) return rc;
    if (dx) {
      const Product q = {Operand{parts.x_high, parts.pitch, parts.pitch}, Operand{of_w, 2 * wide, wide}, a.T, a.C, n,
                         Epilogue{nullptr, v0 > 0 ? sums : nullptr, sums, nullptr, MHC_ACT_NONE, 1}, p.dx.splits, p.dx.kper};
      if (const int rc = ce::run_dx_halves(q, parts.x_low, of_w + wide * 2, parts.row, p.dx, st.head, s)) return rc;
    }
    if (dw != nullptr) {
      const Product q = {Operand{parts.w_high, parts.pitch, parts.pitch}, Operand{of_x, 2 * wide, wide}, n, a.C, a.T,
                         Epilogue{nullptr, nullptr, static_cast<float*>(dw) + v0 * a.C, nullptr, MHC_ACT_NONE, 1}, 1, p.dw.kper};
      if (const int rc = ce::run_dw_halves(q, parts.w_low, of_x + wide * 2, parts.col, p.dw, st.head, by, part, s)) return rc;
    }
  }
  return MHC_OK;
}

int run_gather(const mhc_linear_ce_args& a, const State& st, void* to, hipStream_t s) {
  const uint32_t chunks = (uint32_t)(padded(a.C, a.dtype) * gemm::elem_bytes(a.dtype) / 16);
  const dim3 grid((unsigned)std::min(ceil_div(a.T * chunks, 256), (int64_t)device_cu_count() * 16));
  if (a.dtype == kF32)
    hipLaunchKernelGGL((ce_gather_kernel<float>), grid, dim3(256), 0, s, static_cast<const float*>(a.x), a.ldx, static_cast<float*>(to),
                       (const int*)st.head, (const int*)st.index, a.C, chunks);
  else
    hipLaunchKernelGGL((ce_gather_kernel<uint16_t>), grid, dim3(256), 0, s, static_cast<const uint16_t*>(a.x), a.ldx, static_cast<uint16_t*>(to),
                       (const int*)st.head, (const int*)st.index, a.C, chunks);
  MHC_CHECK_LAUNCH("ce_gather_kernel");
  return MHC_OK;
}

template <typename T>
int run_scatter(const mhc_linear_ce_args& a, const float* sums, int parts, const State& st, const float* dloss, float scale, void* dx, hipStream_t s) {
  const uint32_t groups = (uint32_t)ceil_div(a.C, 8);
  const dim3 grid((unsigned)std::min(ceil_div(a.T * groups, 256), (int64_t)device_cu_count() * 16));
  hipLaunchKernelGGL((ce_scatter_kernel<T>), grid, dim3(256), 0, s, sums, parts, st, dloss, scale * (1.f / ce::kDzUnit<T>), static_cast<T*>(dx), a.T, a.C,
                     groups);
  MHC_CHECK_LAUNCH("ce_scatter_kernel");
  return MHC_OK;
}

int check_args(const mhc_linear_ce_args* a) {
  MHC_CHECK_ARG(a != nullptr, "null pointer: args");
  MHC_CHECK_ARG(a->T >= 0 && a->V >= 1 && a->C >= 1, "T must be >= 0, V and C >= 1 (got %lld, %lld, %lld)", (long long)a->T, (long long)a->V,
                (long long)a->C);
  MHC_CHECK_ARG(a->T < ((int64_t)1 << 28) && a->V < ((int64_t)1 << 22) && a->C < ((int64_t)1 << 22),
                "T must be below 2^28, V and C below 2^22 (got %lld, %lld, %lld)", (long long)a->T, (long long)a->V, (long long)a->C);
  // (a launch has fewer than 2^32 threads: tiles of 256 x 256 with 512 each, or of 64 x 64 with 256 for small T or V)
  MHC_CHECK_ARG((a->T / 256 + 1) * (std::max(a->V, a->C) / 256 + 1) < ((int64_t)1 << 22), "T times V is too large (got %lld, %lld)",
                (long long)a->T, (long long)a->V);
  MHC_CHECK_ARG(a->dtype == kF32 || a->dtype == kBF16 || a->dtype == kF16, "unsupported dtype %d", a->dtype);
  MHC_CHECK_ARG(a->denominator >= 0, "denominator must be >= 0");
  if (a->T == 0) return MHC_OK;
  MHC_CHECK_ARG(a->x && a->w && a->targets, "null pointer");
  MHC_CHECK_ARG((a->ldx >= a->C || a->T == 1) && (a->ldw >= a->C || a->V == 1), "ldx and ldw must be at least C");
  MHC_CHECK_ARG(aligned(a->logits, 16), "logits must be 16-byte aligned");
  MHC_CHECK_ARG(a->weights == nullptr || a->weights_dtype == MHC_DTYPE_F32 || a->weights_dtype == MHC_DTYPE_U8, "weights must be fp32 or bytes");
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

extern "C" size_t mhc_linear_ce_state_bytes(int64_t T) { return T < 0 ? 0 : mhc::ce::State::bytes(T); }

extern "C" size_t mhc_linear_ce_logits_bytes(const mhc_linear_ce_args* a) {
  if (a == nullptr || a->T <= 0 || a->V <= 0 || a->T >= ((int64_t)1 << 28) || a->V >= ((int64_t)1 << 22)) return 0;
  return mhc::keeps_logits(*a) ? (size_t)(a->T * mhc::ce::kept_pitch(a->V) * 4) : 0;
}

extern "C" size_t mhc_linear_ce_fwd_workspace_bytes(const mhc_linear_ce_args* a) {
  if (a == nullptr || a->T <= 0 || a->V <= 0 || a->C <= 0) return 0;
  return mhc::plan_fwd(*a).total;
}

extern "C" int mhc_linear_ce_fwd(const mhc_linear_ce_args* args, float* loss, float* logp, void* state, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_args(args)) return rc;
  const mhc_linear_ce_args& a = *args;
  MHC_CHECK_ARG(loss != nullptr && state != nullptr && (logp != nullptr || a.T == 0), "null pointer");
  MHC_CHECK_ARG(aligned(state, 16) && aligned(workspace, 16), "state and workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const State st(state, a.T);
  FwdPlan p = {};
  if (a.T > 0) p = plan_fwd(a);
  MHC_CHECK_ARG(workspace_bytes >= p.total && (p.total == 0 || workspace != nullptr), "workspace too small");
  if (!p.few) {
    if (a.T <= 8 * kFew) hipLaunchKernelGGL((ce_live_kernel<kFew>), dim3(1), dim3(kFew), 0, s, a, logp, st);
    else hipLaunchKernelGGL((ce_live_kernel<kMany>), dim3(1), dim3(kMany), 0, s, a, logp, st);
    MHC_CHECK_LAUNCH("ce_live_kernel");
  }
  char* ws = static_cast<char*>(workspace);
  float2* part = nullptr;
  float* at_target = nullptr;
  double* terms = nullptr;
  if (a.T > 0) {
    char *const x = ws, *const w = ws + p.x;
    part = reinterpret_cast<float2*>(ws + p.x + p.w);
    at_target = reinterpret_cast<float*>(ws + p.x + p.w + p.part);
    terms = reinterpret_cast<double*>(ws + p.x + p.w + p.part + p.at_target);
    ce::SumsOf of = {st.target, part, at_target, p.tiles, 0, {a.logits, ce::kept_pitch(a.V)}};
    if (in_halves(a)) {
      const int64_t wide = padded(a.C, kF16);
      ce::Halves halves;
      if (const int rc = run_halves(kOfX, a.x, a.ldx, x, &halves.x, &st, a.T, a.C, wide, s)) return rc;
      for (of.v0 = 0; of.v0 < a.V; of.v0 += p.piece) {
        const int64_t n = std::min(p.piece, a.V - of.v0);
        if (const int rc = run_halves(kOfW, static_cast<const float*>(a.w) + of.v0 * a.ldw, a.ldw, w, &halves.w, nullptr, n, a.C, wide, s)) return rc;
        const Product q = {Operand{x, 3 * wide, 3 * wide}, Operand{w, 3 * wide, 3 * wide}, a.T, n, 3 * wide, {}, 1, 0};
        if (const int rc = ce::run_sums_halves(q, p.cut, st.head, of, halves, s)) return rc;
      }
    } else {
      Product q = {Operand{a.x, a.ldx, a.C}, {}, a.T, a.V, a.C, {}, 1, 0};
      if (a.T <= ce::kFewRows) {
        char* to = x;
        if (const int rc = gemm::operand(q.a, a.x, a.T, a.ldx, a.C, a.dtype, to, s)) return rc;
      } else if (!p.direct) {
        if (const int rc = run_gather(a, st, x, s)) return rc;
        const int64_t wide = padded(a.C, a.dtype);
        q.a = Operand{x, wide, wide};
      }
      ws = w;
      if (const int rc = gemm::operand(q.b, a.w, a.V, a.ldw, a.C, a.dtype, ws, s)) return rc;
      const ce::Runs& run = runs_of(a.dtype);
      const int rc = p.rows  ? run.sums_rows(q, of, ce::FewTokens{a, st, logp}, s)
                     : p.few ? run.sums_few(q, p.cut, of, ce::FewTokens{a, st, logp}, s)
                             : run.sums(q, ce::RowsOf{p.direct ? st.index : nullptr, a.T}, p.cut, st.head, of, {}, s);
      if (rc != MHC_OK) return rc;
    }
    if (p.rows)
      hipLaunchKernelGGL((ce_rows_kernel<16>), dim3((unsigned)a.T), dim3(16 * kWave), 0, s, st, (const float2*)part, (const float*)at_target, p.tiles, logp,
                         terms);
    else
      hipLaunchKernelGGL((ce_rows_kernel<1>), dim3((unsigned)std::min<int64_t>(ceil_div(a.T, 4), 1 << 20)), dim3(256), 0, s, st, (const float2*)part,
                         (const float*)at_target, p.tiles, logp, terms);
    MHC_CHECK_LAUNCH("ce_rows_kernel");
  }
  if (a.T <= kFew) hipLaunchKernelGGL((ce_loss_kernel<kFew>), dim3(1), dim3(kFew), 0, s, st, (const double*)terms, loss);
  else hipLaunchKernelGGL((ce_loss_kernel<kMany>), dim3(1), dim3(kMany), 0, s, st, (const double*)terms, loss);
  MHC_CHECK_LAUNCH("ce_loss_kernel");
  return MHC_OK;
}

extern "C" size_t mhc_linear_ce_bwd_workspace_bytes(const mhc_linear_ce_args* a, int want_dx, int want_dw) {
  if (a == nullptr || a->T <= 0 || a->V <= 0 || a->C <= 0) return 0;
  return mhc::plan_bwd(*a, want_dx != 0, want_dw != 0).total;
}

extern "C" int mhc_linear_ce_bwd(const mhc_linear_ce_args* args, const void* state, const float* dloss, float grad_scale, void* dx, void* dw,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_args(args)) return rc;
  const mhc_linear_ce_args& a = *args;
  MHC_CHECK_ARG(a.T > 0, "T must be > 0");
  MHC_CHECK_ARG(state != nullptr, "null pointer");
  MHC_CHECK_ARG(aligned(state, 16) && aligned(workspace, 16), "state and workspace must be 16-byte aligned");
  if (dx == nullptr && dw == nullptr) return MHC_OK;
  const BwdPlan p = plan_bwd(a, dx != nullptr, dw != nullptr);
  MHC_CHECK_ARG(workspace_bytes >= p.total && workspace != nullptr, "workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const State st(const_cast<void*>(state), a.T);
  const int64_t e = gemm::elem_bytes(a.dtype), wide = padded(a.C, a.dtype);
  char* ws = static_cast<char*>(workspace);
  if (few(a)) return ce::run_few(a, st, dloss, grad_scale, dx, dw, ws, s);
  if (p.parts) {
    float* sums;
    const int rc = run_bwd_parts(a, p, st, dloss, grad_scale, dx != nullptr, dw, ws, sums, s);
    return rc != MHC_OK || dx == nullptr ? rc : run_scatter<float>(a, sums, p.dx.splits, st, dloss, grad_scale, dx, s);
  }
  const Operand x = {ws, wide, wide};
  if (const int rc = run_gather(a, st, ws, s)) return rc;
  ws += p.x;
  Operand w;
  if (const int rc = gemm::operand(w, a.w, a.V, a.ldw, a.C, a.dtype, ws, s)) return rc;
  char* const dz[2] = {ws, ws + (p.joint && p.piece < a.V ? p.of_dz : 0)};
  float* const sums = reinterpret_cast<float*>(dz[1] + p.of_dz);
  char* const of_halves = dz[1] + p.of_dz + p.sums;
  float* const part = reinterpret_cast<float*>(of_halves + p.halves.x + p.halves.w);
  ce::Halves halves = {};
  const ce::Kept kept = {a.logits, ce::kept_pitch(a.V)};
  if (kept.z == nullptr && in_halves(a)) {
    if (const int rc = run_halves(kOfX, a.x, a.ldx, of_halves, &halves.x, &st, a.T, a.C, p.halves.wide, s)) return rc;
  }
  const float* const unit = reinterpret_cast<const float*>(st.head) + 1;
  const float lift = a.dtype == kF16 ? ce::kDzUnit<_Float16> : 1.f;
  const ce::Runs& run = runs_of(a.dtype);
  const ScaledBy by = {unit, dloss, grad_scale / lift};
  // the products of the piece from column v0 on, whose dz is in buffer b
  const auto columns = [&](int64_t v0) { return std::min(p.piece, a.V - v0); };
  const auto rows_of = [&](int64_t v0) { return Operand{static_cast<const char*>(w.p) + v0 * w.ld * e, w.ld, w.width}; };
  const auto pitch = [&](int64_t v0) { return padded(columns(v0), a.dtype); };
  const auto of_dz = [&](int64_t v0, int b) {
    return Product{x, rows_of(v0), a.T, columns(v0), a.C, Epilogue{nullptr, nullptr, dz[b], nullptr, MHC_ACT_NONE, a.dtype == kF32}, 1, p.dz.kper};
  };
  const auto gradient = [&](int64_t v0) { return Gradient{st.target, st.coef, st.top, st.inv, v0, lift}; };
  const auto of_dx = [&](int64_t v0, int b) {
    return Product{Operand{dz[b], pitch(v0), pitch(v0)}, rows_of(v0), a.T, a.C, columns(v0),
                   Epilogue{nullptr, v0 > 0 ? sums : nullptr, sums, nullptr, MHC_ACT_NONE, 1}, p.dx.splits, p.dx.kper};
  };
  const auto of_dw = [&](int64_t v0, int b) {
    char* const out = static_cast<char*>(dw) + v0 * a.C * e;
    return Product{Operand{dz[b], pitch(v0), pitch(v0)}, x, columns(v0), a.C, a.T,
                   Epilogue{nullptr, nullptr, out, nullptr, MHC_ACT_NONE, a.dtype == kF32}, 1, p.dw.kper};
  };
  int b = 0;
  for (int64_t v0 = 0; v0 < a.V; v0 += p.piece) {
    if (kept.z != nullptr) {
      if (v0 == 0 || !p.joint) {
        if (const int rc = run.dz_of_kept(gradient(v0), kept, dz[b], pitch(v0), a.T, columns(v0), st.head, s)) return rc;
      }
    } else if (in_halves(a)) {
      const int64_t wide = 3 * p.halves.wide;
      char* const w_halves = of_halves + p.halves.x;
      if (const int rc = run_halves(kOfW, rows_of(v0).p, w.ld, w_halves, &halves.w, nullptr, columns(v0), a.C, p.halves.wide, s)) return rc;
      Product q = of_dz(v0, b);
      q.a = Operand{of_halves, wide, wide}, q.b = Operand{w_halves, wide, wide}, q.K = wide;
      if (const int rc = ce::run_dz_halves(q, p.dz, st.head, pitch(v0), gradient(v0), halves, s)) return rc;
    } else if (v0 == 0 || !p.joint) {
      if (const int rc = run.dz(of_dz(v0, b), p.dz, st.head, pitch(v0), gradient(v0), s)) return rc;
    }
    if (p.joint) {
      ce::Joint j = {of_dx(v0, b), of_dw(v0, b), {}, a.T * a.C, 0, by, {}, kept};
      if (dx == nullptr) j.dx.M = 0;
      if (dw == nullptr) j.dw.M = 0;
      const int all = (int)ceil_div(a.T, gemm::stage_k(a.dtype)) * gemm::stage_k(a.dtype);
      j.dw.kper = all;
      j.dz.splits = 1;
      if (const int64_t next = v0 + p.piece; next < a.V) {
        j.dz = of_dz(next, b ^ 1);
        j.width = pitch(next);
        j.g = gradient(next);
      }
      if (const int rc = run.joint(j, st.head, s)) return rc;
      b ^= 1;
      continue;
    }
    if (dx != nullptr) {
      if (const int rc = run.dx(of_dx(v0, b), p.dx, st.head, s)) return rc;
    }
    if (dw != nullptr) {
      if (const int rc = run.dw(of_dw(v0, b), p.dw, st.head, by, part, s)) return rc;
    }
  }
  if (dx == nullptr) return MHC_OK;
  if (a.dtype == kF32) return run_scatter<float>(a, sums, p.dx.splits, st, dloss, grad_scale, dx, s);
  if (a.dtype == kBF16) return run_scatter<__bf16>(a, sums, p.dx.splits, st, dloss, grad_scale, dx, s);
  return run_scatter<_Float16>(a, sums, p.dx.splits, st, dloss, grad_scale, dx, s);
}
