// knj_int8.cu -- rows as signed 8-bit codes with one f32 scale each, the form in which the int8 products (knj_expert_tc.cu) take
// their rows:
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
  if (gridDim.x <= 148u) grid_dep_signal();
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

}  // namespace

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
