// linear_cross_entropy's products for fp32 operands, of fp16 parts.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

// The larger of two bit patterns.
struct MoreOp {
  MHC_DEV float operator()(float a, float b) const {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)));
  }
};

// dz from logits that were kept, 8 columns of a row a thread: what both kernels
// below do with it.  FAST: a bound of its magnitude; the hardware's exponential
// is 0 where the other one gives subnormal numbers, which are below 2^-126.
template <bool FAST, int ROWS, typename Use>
MHC_DEV void each_dz(const Gradient& g, const Kept& kept, int64_t N, int64_t rows, int64_t m0, int64_t n, Use use) {
  constexpr int kEach = 8, kAhead = 4;
  const float* const from = kept.z + g.v0 + n;
  const int64_t m1 = min(m0 + ROWS, rows);
  for (int64_t m = m0 + threadIdx.x / 32; m < m1; m += kEach * kAhead) {
    f32x4 z[kAhead][2];
    Gradient::Row r[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {  // (rows past the last one read it once more: a load under a condition would wait for itself)
      const int64_t at = min(m + q * kEach, m1 - 1);
      const f32x4* const p = reinterpret_cast<const f32x4*>(from + at * kept.pitch);
      z[q][0] = p[0];
      z[q][1] = p[1];
      r[q] = g.row(at);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (m + q * kEach >= m1) break;
      const int64_t mine = r[q].to < 0 ? -1 : r[q].to - g.v0 - n;
      float d[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float e = gemm::exp_of<FAST>(z[q][k / 4][k % 4] - r[q].t);  // (where it is NaN, so is `each`)
        d[k] = r[q].each * (FAST ? fmaxf(e, 0x1p-126f) : e) - (mine == k ? r[q].c : 0.f);
        d[k] = n + k < N ? d[k] : 0.f;
      }
      use(m + q * kEach, d);
    }
  }
}

// The largest magnitudes of a workgroup's part of each row of dz w[v], to
// rows[row][part], and of each column of dz x[t], to cols[part][column].  (As
// bits, of which NaN's are the largest; put together by a launch of their own:
// with atomic maxima of 128 workgroups at the same lines 67 us for 900 x 32768,
// so 43 and 5.)  The hardware's exponential does: what is lifted to 2^14 has a
// factor of four to fp16's range.
__global__ __launch_bounds__(256) void tops_kernel(const Gradient g, const Kept kept, const Halves halves, const Parts parts, int64_t N, const int* live) {
  __shared__ uint32_t lds[8][256];
  const uint32_t wide = (uint32_t)ceil_div(N, 256), part = blockIdx.x % wide;
  const int64_t rows = *live, m0 = (int64_t)(blockIdx.x / wide) * Parts::kRows, n = (int64_t)part * 256 + threadIdx.x % 32 * 8;
  if (m0 >= rows) return;
  const auto bits = [](float v) { return __builtin_bit_cast(uint32_t, fabsf(v)); };
  float w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = halves.w[min(n + k, N - 1)];
  uint32_t col[8] = {};
  const int64_t from = min(n, (N - 1) / 8 * 8);  // (threads past the last column read it once more, and count nothing)
  each_dz<true, Parts::kRows>(g, kept, n < N ? N : 0, rows, m0, from, [&](int64_t m, const float(&d)[8]) {
    const float x = halves.x[m];
    uint32_t row = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      row = max(row, bits(d[k] * w[k]));
      col[k] = max(col[k], bits(d[k] * x));
    }
    row = __builtin_bit_cast(uint32_t, group_reduce<32>(__builtin_bit_cast(float, row), MoreOp{}));
    if (threadIdx.x % 32 == 0) parts.rows[m * wide + part] = row;
  });
#pragma unroll
  for (int k = 0; k < 8; ++k) lds[threadIdx.x / 32][threadIdx.x % 32 * 8 + k] = col[k];
  __syncthreads();
  uint32_t top = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) top = max(top, lds[q][threadIdx.x]);
  const int64_t mine = (int64_t)part * 256 + threadIdx.x;
  if (mine < N) parts.cols[m0 / Parts::kRows * N + mine] = top;
}

// the largest of each row's and each column's parts: a wave for a row, a thread for a column
__global__ __launch_bounds__(256) void join_tops_kernel(const Parts parts, int64_t N, uint32_t of_rows, const int* live) {
  const int64_t rows = *live;
  if (blockIdx.x < of_rows) {
    const int64_t m = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave, wide = ceil_div(N, 256);
    if (m >= rows) return;
    float top = 0.f;
    for (int64_t k = threadIdx.x % kWave; k < wide; k += kWave) top = MoreOp{}(top, __builtin_bit_cast(float, parts.rows[m * wide + k]));
    top = group_reduce<kWave>(top, MoreOp{});
    if (threadIdx.x % kWave == 0) parts.row[m] = __builtin_bit_cast(uint32_t, top);
  } else {
    const int64_t n = (int64_t)(blockIdx.x - of_rows) * 256 + threadIdx.x, high = ceil_div(rows, Parts::kRows);
    if (n >= N) return;
    uint32_t top = 0;
#pragma unroll 8
    for (int64_t k = 0; k < high; ++k) top = max(top, parts.cols[k * N + n]);
    parts.col[n] = top;
  }
}

// a vector of parts: the nearest fp16 numbers, and those nearest to what is left
MHC_DEV void put_parts(_Float16* high, _Float16* low, const float (&v)[8]) {
  f16x4 h[2], l[2];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    h[k / 4][k % 4] = (_Float16)v[k];
    l[k / 4][k % 4] = (_Float16)(v[k] - (float)h[k / 4][k % 4]);
  }
  __builtin_memcpy(high, h, 16);
  __builtin_memcpy(low, l, 16);
}

// dz, each element as two parts for each of its two products: 12 bytes go by for
// each (900 x 32768: 354 MB in 73 us, 4.8 TB/s).
__global__ __launch_bounds__(256) void parts_kernel(const Gradient g, const Kept kept, const Halves halves, const Parts parts, int64_t N, const int* live) {
  const uint32_t wide = (uint32_t)ceil_div(parts.pitch, 256);
  const int64_t rows = *live, m0 = (int64_t)(blockIdx.x / wide) * 32, n = (int64_t)(blockIdx.x % wide) * 256 + threadIdx.x % 32 * 8;
  if (n >= parts.pitch) return;
  int w[8], col[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    w[k] = power_of(halves.w[min(n + k, N - 1)]);
    col[k] = power_of(lift_by(lift_of(parts.col[min(n + k, N - 1)])));
  }
  each_dz<false, 32>(g, kept, N, rows, m0, n, [&](int64_t m, const float(&d)[8]) {
    const int x = power_of(halves.x[m]), row = power_of(lift_by(lift_of(parts.row[m])));
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = times_power(d[k], w[k] + row);
    put_parts(parts.x_high + m * parts.pitch + n, parts.x_low + m * parts.pitch + n, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = times_power(d[k], x + col[k]);
    put_parts(parts.w_high + m * parts.pitch + n, parts.w_low + m * parts.pitch + n, v);
  });
}

int run_parts(const Gradient& g, const Kept& kept, const Halves& halves, const Parts& parts, int64_t rows, int64_t N, const int* live, hipStream_t s) {
  hipLaunchKernelGGL(tops_kernel, dim3((unsigned)(ceil_div(rows, Parts::kRows) * ceil_div(N, 256))), dim3(256), 0, s, g, kept, halves, parts, N, live);
  MHC_CHECK_LAUNCH("tops_kernel");
  const uint32_t of_rows = (uint32_t)ceil_div(rows, 4);
  hipLaunchKernelGGL(join_tops_kernel, dim3(of_rows + (unsigned)ceil_div(N, 256)), dim3(256), 0, s, parts, N, of_rows, live);
  MHC_CHECK_LAUNCH("join_tops_kernel");
  hipLaunchKernelGGL(parts_kernel, dim3((unsigned)(ceil_div(rows, 32) * ceil_div(parts.pitch, 256))), dim3(256), 0, s, g, kept, halves, parts, N, live);
  MHC_CHECK_LAUNCH("parts_kernel");
  return MHC_OK;
}

// A product of parts: high times high, low times high and high times low in one
// tile of sums, whose rows are lowered again; SUMS and limits as in
// live_tile_kernel, the scale as ScaledBy (by.a NULL: 1).  Bound by the matrix
// instructions: 900 x 1024 x 32768 in 16 parts 183 us, 32768 x 1024 x 900 178
// (1.0 PFLOP/s of fp16); fp32 tiles 324 and 319.
template <bool AK, bool SUMS, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void halves_tile_kernel(Product p, const void* a_low, const void* b_low, const uint32_t* tops, const int* live,
                                                                   const ScaledBy by) {
  using B = gemm::TileBytes<_Float16, BM, BN, WM, WN, NS>;
  constexpr int JM = BM / WM / 16, JN = BN / WN / 16;
  __shared__ __attribute__((aligned(1024))) char smem[B::kAll];
  const int64_t part = p.M * p.N;
  if (!limit<AK, BM, BN>(p, live, blockIdx.x)) return;
  only_sums(p.e);
  if constexpr (SUMS) move_to_part(p.e, blockIdx.y * part);
  else if (p.splits > 1) p.e.out = static_cast<float*>(p.e.out) + blockIdx.y * part;
  const gemm::Place<BM, BN, WM, WN> at(p, blockIdx.x, (int)blockIdx.y);
  f32x4 acc[JN][JM] = {};
#pragma unroll 1
  for (int q = 0; q < 3; ++q) {
    Product one = p;
    if (q == 1) one.a.p = a_low;
    if (q == 2) one.b.p = b_low;
    gemm::sum_tile<_Float16, AK, false, BM, BN, WM, WN, NS>(one, at, smem, acc);
    __syncthreads();  // nobody reads the stages any more
  }
  const int64_t m0 = at.m0 + at.wm, n0 = at.n0 + at.wn;
  const float scale = by.a != nullptr ? by.a[0] * (by.b != nullptr ? by.b[0] : 1.f) * by.c : 1.f;
#pragma unroll
  for (int j = 0; j < JM; ++j) {
    const float low = lower_by(lift_of(tops[min(m0 + j * 16 + at.lane % 16, p.M - 1)]));
#pragma unroll
    for (int i = 0; i < JN; ++i) acc[i][j] = acc[i][j] * low * scale;
  }
  gemm::store_tile<float, JM, JN, WM * WN, B::kStages, 2>(p.e, smem, acc, m0, p.M, n0, p.N, at.wave, at.lane);
}

template <bool AK, bool SUMS, int BM, int BN, int WM, int WN, int NS>
int launch_halves(const Product& p, const void* a_low, const void* b_low, const uint32_t* tops, const int* live, const ScaledBy& by, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(p.M, BM) * ceil_div(p.N, BN)), (unsigned)p.splits), block(64 * WM * WN);
  hipLaunchKernelGGL((halves_tile_kernel<AK, SUMS, BM, BN, WM, WN, NS>), grid, block, 0, s, p, a_low, b_low, tops, live, by);
  MHC_CHECK_LAUNCH("halves_tile_kernel");
  return MHC_OK;
}

template <bool AK, bool SUMS>
int run_halves_tiles(Product p, const void* a_low, const void* b_low, const uint32_t* tops, const Cut& c, const int* live, const ScaledBy& by,
                     float* part, hipStream_t s) {
  const Epilogue e = p.e;
  p.splits = c.splits;
  p.kper = c.kper;
  if (c.splits > 1 && !SUMS) p.e = Epilogue{nullptr, nullptr, part, nullptr, MHC_ACT_NONE, 1};
  int rc;
  switch (c.tile) {
    case 0: rc = launch_halves<AK, SUMS, 256, 256, 2, 4, 2>(p, a_low, b_low, tops, live, by, s); break;
    case 1: rc = launch_halves<AK, SUMS, 128, 256, 2, 4, 2>(p, a_low, b_low, tops, live, by, s); break;
    case 2: rc = launch_halves<AK, SUMS, 128, 128, 4, 2, 2>(p, a_low, b_low, tops, live, by, s); break;
    case 3: rc = launch_halves<AK, SUMS, 64, 128, 4, 2, 3>(p, a_low, b_low, tops, live, by, s); break;
    default: rc = launch_halves<AK, SUMS, 64, 64, 4, 1, 3>(p, a_low, b_low, tops, live, by, s); break;
  }
  if (rc != MHC_OK || c.splits == 1 || SUMS) return rc;
  return gemm::launch_join<float>(e, part, c.splits, p.M, p.N, s);
}

int run_dx_halves(const Product& p, const void* a_low, const void* b_low, const uint32_t* tops, const Cut& c, const int* live, hipStream_t s) {
  return run_halves_tiles<true, true>(p, a_low, b_low, tops, c, live, ScaledBy{}, nullptr, s);
}
int run_dw_halves(const Product& p, const void* a_low, const void* b_low, const uint32_t* tops, const Cut& c, const int* live, const ScaledBy& by,
                  float* part, hipStream_t s) {
  return run_halves_tiles<false, false>(p, a_low, b_low, tops, c, live, by, part, s);
}

int run_sums_halves(const Product& p, const Cut& c, const int* live, const SumsOf& of, const Halves& halves, hipStream_t s) {
  return run_sums<_Float16, true>(p, RowsOf{nullptr, p.M}, c, live, of, halves, s);
}

int run_dz_halves(const Product& p, const Cut& c, const int* live, int64_t width, const Gradient& g, const Halves& halves, hipStream_t s) {
  return run_live<_Float16, true, true, false, float>(p, c, live, width, GradientOfHalves{g, halves}, nullptr, s);
}

}  // namespace ce
}  // namespace mhc
