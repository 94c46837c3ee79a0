// knj_int8.cu -- rows as signed 8-bit codes with one f32 scale each, the form in which the int8 products (knj_expert_tc.cu) take
// their rows, and the product of few rows:
//   scale = most * f32(1/127), most = the row's largest magnitude;  code = the whole number nearest to v * (1 / scale), ties to even
// in f32, so that any program with IEEE arithmetic forms the same bits. |v| <= most keeps the product within 127 (1 + 2^-22), so a code
// never passes 127. A row whose `most` is below 2^-100 is zeros under a zero scale: there the scale or its inverse would leave the
// normal range. A row that holds a NaN or an infinity gets that as its scale over codes of zero, and products of the row are NaN.
//
// Bound by bytes: a row is read once and held in registers between its maximum and its codes (rows up to 32768 values in whole
// 16-byte units; others are read twice, the second time from L1 or L2).
#include "knj_fp8.cuh"

using namespace knj;

namespace {

struct RowScale {
  float scale, inverse;
  uint32_t mask;   // of the codes: none of a row that is not finite
};
__device__ __forceinline__ RowScale row_scale(float most) {
  RowScale s;
  s.scale = __fmul_rn(most, 1.0f / 127.0f);
  s.inverse = __frcp_rn(s.scale);
  if (most < 0x1p-100f) s.scale = s.inverse = 0.0f;
  s.mask = most <= 3.402823466e38f ? 0xffffffffu : 0u;
  return s;
}
// 1.5 * 2^23: added to a value of up to 2^22, the sum's last bits are the nearest whole number, ties to even
constexpr float kWhole = 12582912.0f;
// Both roundings of the definition: of the product and, by the sum, to a whole number. Of packed pairs (f32x2) the two are fused into
// one, whatever their names say, and codes of ties come out otherwise.
__device__ __forceinline__ float2 whole2(float2 v, float inverse) {
  return make_float2(__fadd_rn(__fmul_rn(v.x, inverse), kWhole), __fadd_rn(__fmul_rn(v.y, inverse), kWhole));
}
// codes of four values
__device__ __forceinline__ uint32_t codes4(float2 a, float2 b, const RowScale &s) {
  a = whole2(a, s.inverse);
  b = whole2(b, s.inverse);
  const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  return __byte_perm(lo, hi, 0x5410) & s.mask;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// maximum over the CTA's warps
__device__ __forceinline__ float cta_max_nan(float v) {
  __shared__ float red[32];
  v = warp_max_nan(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_max_nan((threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.f);
}

// eight consecutive values
__device__ __forceinline__ void load8(const void *x, int dtype, int64_t i, float2 (&v)[4]) {
  if (dtype == KNJ_DT_F32) {
    const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
    const float4 a = q[0], b = q[1];
    v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w); v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
    return;
  }
  const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + i);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = dtype == KNJ_DT_BF16 ? make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u))
                                : __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
}

// K8 runs of eight values a row, a thread holds up to RUNS of them. One warp per row (WARP: rows of up to 256 RUNS values, eight to a
// CTA) or one CTA.
template <int RUNS, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) int8_rows_vec_kernel(const void *x, int dtype, int64_t ldx, int rows, int K8, uint8_t *q, float *scale) {
  grid_dep_wait();
  // The products' tables, maps and barriers stand ready when the last rows are done, whatever the number of CTAs. (us in a graph without, with: dense
  // 16 x 1000 x 2048 8.8, 8.0, 301 x 1000 x 2048 12.2, 11.6, 2048 x 4096 x 4096 35.4, 34.3; down of 512 tokens, Zipf 62, 49; all others equal.)
  grid_dep_signal();
  const int per = WARP ? 32 : blockDim.x, at = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= rows) return;
  float2 v[RUNS][4];
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    const int i = at + r * per;
    if (i < K8) load8(x, dtype, row * ldx + 8 * i, v[r]);
    else v[r][0] = v[r][1] = v[r][2] = v[r][3] = make_float2(0.f, 0.f);
  }
#pragma unroll
  for (int r = 0; r < RUNS; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max3_abs_nan(most, v[r][j].x, v[r][j].y);
  const RowScale s = row_scale(WARP ? warp_max_nan(most) : cta_max_nan(most));
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    const int i = at + r * per;
    if (i < K8) *reinterpret_cast<uint2 *>(q + (row * K8 + i) * 8) = make_uint2(codes4(v[r][0], v[r][1], s), codes4(v[r][2], v[r][3], s));
  }
  if (at == 0) scale[row] = s.scale;
}

// any rows: one CTA each, read twice
__global__ void __launch_bounds__(256) int8_rows_kernel(const void *x, int dtype, int64_t ldx, int K, uint8_t *q, float *scale) {
  grid_dep_wait();
  const int64_t row = blockIdx.x;
  float most = 0.f;
  for (int i = threadIdx.x; i < K; i += 256) most = max3_abs_nan(most, load_as_f32(x, dtype, row * ldx + i), 0.f);
  const RowScale s = row_scale(cta_max_nan(most));
  for (int i = threadIdx.x; i < K; i += 256) {
    const float2 v = make_float2(load_as_f32(x, dtype, row * ldx + i), 0.f);
    q[row * K + i] = (uint8_t)codes4(v, v, s);
  }
  if (threadIdx.x == 0) scale[row] = s.scale;
}

// Few rows times a matrix: y[r][n] = f32(sum over k of codes[r][k] W[n][k]) * (scale[r] * ws[n]), the rows' codes formed by every CTA for
// itself in shared memory. One launch and no workspace, where rows and product on the tensor cores are two launches. Bound by the matrix,
// read once: a warp takes pairs of matrix rows, a lane 16 bytes of either at a time, which meet the codes in dp4a; the sums are whole
// numbers, so the bits are those of the other form whatever their order.
// us in a graph, this form and the two launches, for 1, 2, 4 rows: 2048 x 2048 3.3, 3.9, 4.2 and 7.3, 7.4, 8.2; 16384 x 4096 (10.2 at HBM's
// rate) 12.9, 13.8, 17.2 and 18.6, 18.5, 19.0. Of 8 rows every 16 bytes of the matrix meet eight reads of shared memory: 27 us against 18,
// so that more than four rows take the other. (Host time of a call with one row: 9.1 us, so 13.7.)
constexpr int kFewRows = 4, kFewBytes = 40 * 1024;   // rows; bytes of codes, which need no opting in

template <int M>
__global__ void __launch_bounds__(256, 4) int8_few_kernel(const int8_t *W, const float *ws, int K, int N, const void *x, int dtype, int64_t ldx, int vec,
                                                          int m, void *y, int y_dtype, int64_t ldy) {
  extern __shared__ __align__(16) uint8_t codes[];   // [M][K]
  __shared__ float part[8], scale[M];
  constexpr int kWpr = 8 / M;   // warps of a row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, units = K / 16, pairs = N / 2 + (N & 1);
  grid_dep_wait();
  int pair = blockIdx.x * 8 + warp;
  uint4 w[2][4];
  auto load = [&](int at, int from) {
    const int8_t *a = W + (int64_t)(2 * at) * K, *b = W + (int64_t)min(2 * at + 1, N - 1) * K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = from + lane + 32 * i;
      if (u < units) {
        w[0][i] = __ldcg(reinterpret_cast<const uint4 *>(a) + u);
        w[1][i] = __ldcg(reinterpret_cast<const uint4 *>(b) + u);
      }
    }
  };
  if (pair < pairs) load(pair, 0);   // on its way while the codes are formed
  const int row = warp / kWpr, first = warp % kWpr * 32 + lane;
  auto value8 = [&](int i, float2 (&v)[4]) {
    if (vec) {
      load8(x, dtype, row * ldx + 8 * i, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = make_float2(load_as_f32(x, dtype, row * ldx + 8 * i + 2 * j), load_as_f32(x, dtype, row * ldx + 8 * i + 2 * j + 1));
    }
  };
  float most = 0.f;
  if (row < m)
    for (int i = first; i < K / 8; i += 32 * kWpr) {
      float2 v[4];
      value8(i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) most = max3_abs_nan(most, v[j].x, v[j].y);
    }
  most = warp_max_nan(most);
  if (lane == 0) part[warp] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWpr; ++i) most = max_nan(most, part[row * kWpr + i]);
  const RowScale s = row_scale(most);
  for (int i = first; i < K / 8; i += 32 * kWpr) {   // zeros of rows behind the last
    float2 v[4];
    if (row < m) value8(i, v);
    else v[0] = v[1] = v[2] = v[3] = make_float2(0.f, 0.f);
    *reinterpret_cast<uint2 *>(codes + row * K + 8 * i) = make_uint2(codes4(v[0], v[1], s), codes4(v[2], v[3], s));
  }
  if (warp % kWpr == 0 && lane == 0) scale[row] = s.scale;
  __syncthreads();
  for (; pair < pairs; pair += gridDim.x * 8) {
    int acc[2][M] = {};
    for (int from = 0; from < units; from += 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = from + lane + 32 * i;
        if (u >= units) continue;
#pragma unroll
        for (int r = 0; r < M; ++r) {
          const uint4 c = *reinterpret_cast<const uint4 *>(codes + r * K + 16 * u);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            acc[h][r] = __dp4a((int)w[h][i].x, (int)c.x, __dp4a((int)w[h][i].y, (int)c.y,
                        __dp4a((int)w[h][i].z, (int)c.z, __dp4a((int)w[h][i].w, (int)c.w, acc[h][r]))));
        }
      }
      const bool more = from + 128 < units;
      const int next = more ? pair : pair + gridDim.x * 8;
      if (next < pairs) load(next, more ? from + 128 : 0);
    }
    int mine = 0;   // lane 2 r + h: of row r and the pair's row h
#pragma unroll
    for (int r = 0; r < M; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[h][r]);
        if (lane == 2 * r + h) mine = sum;
      }
    const int r = lane >> 1, n = 2 * pair + (lane & 1);
    if (r < m && n < N) store_from_f32(y, y_dtype, r * ldy + n, __int2float_rn(mine) * (scale[r < M ? r : 0] * __ldcg(ws + n)));
  }
}

}  // namespace

namespace knj {
static int few_rows(int m) { return m <= 2 ? m : kFewRows; }   // that a kernel is built for
bool int8_few(int m, int K) { return m <= kFewRows && few_rows(m) * (int64_t)K <= kFewBytes; }

int int8_few_launch(const void *W, const float *ws, int K, int N, const void *x, int dtype, int64_t ldx, int m, void *y, int y_dtype, int64_t ldy, cudaStream_t st) {
  const int vec = aligned16(x) && (m == 1 || ldx * (dtype == KNJ_DT_F32 ? 4 : 2) % 16 == 0);
  const int blocks = (N - 1) / 16 + 1, most = 4 * sm_count(), M = few_rows(m);
  const dim3 grid(blocks < most ? blocks : most), block(256);
  const size_t smem = (size_t)M * K;
  const int8_t *w = static_cast<const int8_t *>(W);
  if (M == 1) KNJ_CUDA(launch_chain(int8_few_kernel<1>, grid, block, smem, st, w, ws, K, N, x, dtype, ldx, vec, m, y, y_dtype, ldy));
  else if (M == 2) KNJ_CUDA(launch_chain(int8_few_kernel<2>, grid, block, smem, st, w, ws, K, N, x, dtype, ldx, vec, m, y, y_dtype, ldy));
  else KNJ_CUDA(launch_chain(int8_few_kernel<kFewRows>, grid, block, smem, st, w, ws, K, N, x, dtype, ldx, vec, m, y, y_dtype, ldy));
  return launch_status("int8_few_kernel");
}
}  // namespace knj

extern "C" int knj_int8_rows_launch(const void *x, int x_dtype, int64_t ldx, int rows, int K, void *q, float *scale, knj_stream_t s) {
  KNJ_REQUIRE(rows >= 0 && K > 0, "knj_int8_rows: bad sizes");
  if (rows == 0) return KNJ_OK;
  KNJ_REQUIRE(x && q && scale, "knj_int8_rows: null pointer");
  KNJ_REQUIRE(x_dtype >= KNJ_DT_F32 && x_dtype <= KNJ_DT_F16, "knj_int8_rows: rows are f32, bf16 or f16");
  KNJ_REQUIRE(ldx >= K, "knj_int8_rows: row stride shorter than the rows");
  const cudaStream_t st = as_stream(s);
  uint8_t *codes = static_cast<uint8_t *>(q);
  constexpr int kRuns = 4;
  const bool units = K % 8 == 0 && aligned16(x) && ldx * (x_dtype == KNJ_DT_F32 ? 4 : 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  if (units && K <= 32 * 8 * kRuns) {
    KNJ_CUDA(launch_chain(int8_rows_vec_kernel<kRuns, true>, dim3((unsigned)((rows + 7ll) / 8)), dim3(256), 0, st, x, x_dtype, ldx, rows, K / 8, codes, scale));
    return launch_status("int8_rows_vec_kernel");
  }
  if (units && K <= 1024 * 8 * kRuns) {
    int threads = 64;
    while (threads * 8 * kRuns < K) threads *= 2;
    KNJ_CUDA(launch_chain(int8_rows_vec_kernel<kRuns, false>, dim3((unsigned)rows), dim3(threads), 0, st, x, x_dtype, ldx, rows, K / 8, codes, scale));
    return launch_status("int8_rows_vec_kernel");
  }
  KNJ_CUDA(launch_chain(int8_rows_kernel, dim3((unsigned)rows), dim3(256), 0, st, x, x_dtype, ldx, K, codes, scale));
  return launch_status("int8_rows_kernel");
}
