// knj_block_norm.cu -- what stands between two blocks of a residual stream, in one pass over the rows: the norm after a
// block, its gate, the scaled residual add and the norm in front of the next block; and rows as e4m3 codes.
//   n = y * rsqrt(mean(y^2) + eps) * post_w   (or y)
//   s = beta * x + alpha * g * n
//   h = s * rsqrt(mean(s^2) + eps) * pre_w    (from s before it is rounded to the stream's type)
// The reference's rows (src/model/model.cpp:258-271 rmsnorm_rows, :652 residual add) are the case y = NULL and the case
// without weights and gate.
#include "knj_fp8.cuh"

using namespace knj;

namespace {

struct NormParams {
  const void *x, *y, *post_w, *gate, *pre_w;
  void *stream, *h;
  float *h_scale;
  int64_t ldx, ldy, ldg, ld_stream, ldh;
  int T, H, x_dtype, y_dtype, w_dtype, gate_dtype, gate_kind, gate_sigmoid, stream_dtype, h_dtype;
  float alpha, beta, eps;
};

__device__ __forceinline__ float gate_value(const NormParams &p, int64_t i) {
  const float g = load_as_f32(p.gate, p.gate_dtype, i);
  return p.gate_sigmoid ? 1.0f / (1.0f + expf(-g)) : g;
}

__device__ __forceinline__ float block_sum(float v, float *red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float tot = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) tot += red[i];
  return tot;
}

// 1 / sqrt(mean square + eps) of a row whose sum of squares is `tot`. Where the squares of a large row leave the f32 range
// they are summed once more from values * 2^-64 (`again`); eps does not count there.
constexpr float kDown = 0x1p-64f;
template <class Again>
__device__ __forceinline__ float rms_inverse(float tot, int H, float eps, Again again) {
  if (tot <= 3.402823466e38f || tot != tot) return 1.0f / sqrtf(tot / (float)H + eps);
  return kDown / sqrtf(again() / (float)H);
}

// One CTA per row, the row of s in shared memory.
__global__ void __launch_bounds__(256) block_norm_kernel(const NormParams p) {
  extern __shared__ float row[];
  __shared__ float red[8];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  float rs = 1.f;
  if (p.y && p.post_w) {
    float ss = 0.f;
    for (int i = tid; i < p.H; i += 256) {
      const float v = load_as_f32(p.y, p.y_dtype, t * p.ldy + i);
      ss = fmaf(v, v, ss);
    }
    rs = rms_inverse(block_sum(ss, red), p.H, p.eps, [&] {
      float q = 0.f;
      for (int i = tid; i < p.H; i += 256) {
        const float v = load_as_f32(p.y, p.y_dtype, t * p.ldy + i) * kDown;
        q = fmaf(v, v, q);
      }
      return block_sum(q, red);
    });
  }
  float ss = 0.f;
  for (int i = tid; i < p.H; i += 256) {
    float s = p.beta * load_as_f32(p.x, p.x_dtype, t * p.ldx + i);
    if (p.y) {
      float n = load_as_f32(p.y, p.y_dtype, t * p.ldy + i);
      if (p.post_w) n = n * rs * load_as_f32(p.post_w, p.w_dtype, i);
      if (p.gate_kind) n *= gate_value(p, p.gate_kind == KNJ_GATE_CHANNEL ? i : p.gate_kind == KNJ_GATE_ROW ? t * p.ldg : t * p.ldg + i);
      s = fmaf(p.alpha, n, s);
    }
    row[i] = s;
    ss = fmaf(s, s, ss);
    if (p.stream) store_from_f32(p.stream, p.stream_dtype, t * p.ld_stream + i, s);
  }
  if (!p.h) return;
  const float hs = rms_inverse(block_sum(ss, red), p.H, p.eps, [&] {
    float q = 0.f;
    for (int i = tid; i < p.H; i += 256) q = fmaf(row[i] * kDown, row[i] * kDown, q);
    return block_sum(q, red);
  });
  if (p.h_dtype != KNJ_DT_E4M3) {
    for (int i = tid; i < p.H; i += 256) store_from_f32(p.h, p.h_dtype, t * p.ldh + i, row[i] * hs * load_as_f32(p.pre_w, p.w_dtype, i));
    return;
  }
  const int groups = (p.H + kFp8Group - 1) / kFp8Group;
  for (int g = tid >> 5; g < groups; g += 8) {
    float v[4], most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kFp8Group + 4 * lane + j;
      v[j] = i < p.H ? row[i] * hs * load_as_f32(p.pre_w, p.w_dtype, i) : 0.f;
      most = max_nan(most, fabsf(v[j]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    const Fp8Scale sc = fp8_scale(most);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kFp8Group + 4 * lane + j;
      if (i < p.H) static_cast<uint8_t *>(p.h)[t * p.ldh + i] = (uint8_t)e4m3_pair(v[j] * sc.inverse, 0.f);
    }
    if (lane == 0) p.h_scale[t * groups + g] = sc.scale;
  }
}

// One warp per group.
__global__ void __launch_bounds__(256) fp8_rows_kernel(const void *x, int dtype, int64_t ldx, int64_t n_groups, int K, int groups,
                                                       uint8_t *q, float *scale) {
  const int lane = threadIdx.x & 31;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < n_groups; w += (int64_t)gridDim.x * 8) {
    const int64_t t = w / groups;
    const int g = (int)(w - t * groups);
    float v[4], most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kFp8Group + 4 * lane + j;
      v[j] = i < K ? load_as_f32(x, dtype, t * ldx + i) : 0.f;
      most = max_nan(most, fabsf(v[j]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    const Fp8Scale sc = fp8_scale(most);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kFp8Group + 4 * lane + j;
      if (i < K) q[t * K + i] = (uint8_t)e4m3_pair(v[j] * sc.inverse, 0.f);
    }
    if (lane == 0) scale[w] = sc.scale;
  }
}

}  // namespace

extern "C" {

int knj_block_norm_launch(const knj_block_norm_args *a, knj_stream_t s) {
  KNJ_REQUIRE(a, "knj_block_norm: null argument block");
  KNJ_REQUIRE(a->n_tokens >= 0 && a->hidden > 0, "knj_block_norm: bad sizes");
  if (a->n_tokens == 0) return KNJ_OK;
  KNJ_REQUIRE(a->hidden <= KNJ_BLOCK_NORM_MAX_HIDDEN, "knj_block_norm: hidden=%d above %d", a->hidden, KNJ_BLOCK_NORM_MAX_HIDDEN);
  KNJ_REQUIRE(a->x && (a->stream_out || a->h), "knj_block_norm: null pointer");
  KNJ_REQUIRE((a->h != nullptr) == (a->pre_w != nullptr), "knj_block_norm: h and pre_w go together");
  KNJ_REQUIRE(a->y || (!a->post_w && a->gate_kind == KNJ_GATE_NONE), "knj_block_norm: post_w and gate need a block output y");
  KNJ_REQUIRE(a->gate_kind >= KNJ_GATE_NONE && a->gate_kind <= KNJ_GATE_FULL && (a->gate != nullptr) == (a->gate_kind != KNJ_GATE_NONE),
              "knj_block_norm: gate and gate_kind do not match");
  auto float_type = [](int dt) { return dt >= KNJ_DT_F32 && dt <= KNJ_DT_F16; };
  KNJ_REQUIRE(float_type(a->x_dtype) && (!a->y || float_type(a->y_dtype)) && (!a->gate || float_type(a->gate_dtype)) &&
                  (!a->stream_out || float_type(a->stream_dtype)),
              "knj_block_norm: x, y, gate and the stream are f32, bf16 or f16");
  KNJ_REQUIRE(!(a->pre_w || a->post_w) || float_type(a->w_dtype), "knj_block_norm: norm weights are f32, bf16 or f16");
  KNJ_REQUIRE(!a->h || float_type(a->h_dtype) || a->h_dtype == KNJ_DT_E4M3, "knj_block_norm: bad h_dtype %d", a->h_dtype);
  KNJ_REQUIRE(!a->h || a->h_dtype != KNJ_DT_E4M3 || a->h_scale, "knj_block_norm: e4m3 rows need h_scale");
  const int H = a->hidden;
  KNJ_REQUIRE(a->ldx >= H && (!a->y || a->ldy >= H) && (!a->stream_out || a->ld_stream >= H) && (!a->h || a->ldh >= H) &&
                  (a->gate_kind != KNJ_GATE_FULL || a->ldg >= H) && (a->gate_kind != KNJ_GATE_ROW || a->ldg >= 1),
              "knj_block_norm: row strides shorter than the rows");
  NormParams p{};
  p.x = a->x; p.y = a->y; p.post_w = a->post_w; p.gate = a->gate; p.pre_w = a->pre_w; p.stream = a->stream_out; p.h = a->h;
  p.h_scale = a->h_scale; p.ldx = a->ldx; p.ldy = a->ldy; p.ldg = a->ldg; p.ld_stream = a->ld_stream; p.ldh = a->ldh;
  p.T = a->n_tokens; p.H = H; p.x_dtype = a->x_dtype; p.y_dtype = a->y_dtype; p.w_dtype = a->w_dtype; p.gate_dtype = a->gate_dtype;
  p.gate_kind = a->gate_kind; p.gate_sigmoid = a->gate_sigmoid; p.stream_dtype = a->stream_dtype; p.h_dtype = a->h_dtype;
  p.alpha = a->alpha; p.beta = a->beta; p.eps = a->eps;
  const size_t smem = (size_t)H * 4;
  if (smem > 48 * 1024) KNJ_CUDA(cudaFuncSetAttribute(block_norm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KNJ_BLOCK_NORM_MAX_HIDDEN * 4));
  block_norm_kernel<<<a->n_tokens, 256, smem, as_stream(s)>>>(p);
  return launch_status("block_norm_kernel");
}

int knj_fp8_rows_launch(const void *x, int x_dtype, int64_t ldx, int rows, int K, void *q, float *scale, knj_stream_t s) {
  KNJ_REQUIRE(rows >= 0 && K > 0, "knj_fp8_rows: bad sizes");
  if (rows == 0) return KNJ_OK;
  KNJ_REQUIRE(x && q && scale, "knj_fp8_rows: null pointer");
  KNJ_REQUIRE(x_dtype >= KNJ_DT_F32 && x_dtype <= KNJ_DT_F16, "knj_fp8_rows: rows are f32, bf16 or f16");
  KNJ_REQUIRE(ldx >= K, "knj_fp8_rows: row stride shorter than the rows");
  const int groups = (K + kFp8Group - 1) / kFp8Group;
  const int64_t n = (int64_t)rows * groups, blocks = (n + 7) / 8, cap = (int64_t)sm_count() * 32;
  fp8_rows_kernel<<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, as_stream(s)>>>(x, x_dtype, ldx, n, K, groups, static_cast<uint8_t *>(q), scale);
  return launch_status("fp8_rows_kernel");
}

}  // extern "C"
