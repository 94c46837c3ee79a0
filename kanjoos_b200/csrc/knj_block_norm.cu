// knj_block_norm.cu -- what stands between two blocks of a residual stream, in one pass over the rows: the norm after a
// block, its gate, the scaled residual add and the norm in front of the next block; and rows as e4m3 codes.
//   n = y * rsqrt(mean(y^2) + eps) * post_w   (or y)
//   s = beta * x + alpha * g * n
//   h = s * rsqrt(mean(s^2) + eps) * pre_w    (from s before it is rounded to the stream's type)
// The reference's rows (src/model/model.cpp:258-271 rmsnorm_rows, :652 residual add) are the case y = NULL and the case
// without weights and gate.
#include "knj_fp8.cuh"
#include <stdlib.h>

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
  return p.gate_sigmoid ? __fdividef(1.0f, 1.0f + expf(-g)) : g;
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

// ---- rows whose strides and bases are whole 16-byte units, H a multiple of 8 ----------------------------------------

// eight consecutive elements as they lie in memory; the four-byte type takes both words
struct Raw8 {
  uint4 a, b;
};
template <bool WIDE>
__device__ __forceinline__ Raw8 load_raw8(const void *base, int64_t i) {
  Raw8 r;
  if constexpr (WIDE) {
    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + i);
    r.a = q[0];
    r.b = q[1];
  } else {
    r.a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + i);
  }
  return r;
}
__device__ __forceinline__ void unpack16(const uint4 &u, bool bf16, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (bf16) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
template <bool WIDE>
__device__ __forceinline__ void values8(const Raw8 &r, bool bf16, float (&v)[8]) {
  if constexpr (WIDE) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
  } else {
    unpack16(r.a, bf16, v);
  }
}
__device__ __forceinline__ void load8(const void *base, int dtype, int64_t i, float (&v)[8]) {
  if (dtype == KNJ_DT_F32) values8<true>(load_raw8<true>(base, i), false, v);
  else values8<false>(load_raw8<false>(base, i), dtype == KNJ_DT_BF16, v);
}
__device__ __forceinline__ void store8(void *base, int dtype, int64_t i, const float (&v)[8]) {
  if (dtype == KNJ_DT_F32) {
    float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(base) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == KNJ_DT_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}
// sixteen lanes hold a group of 128: the scale, and this lane's eight codes
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float &scale) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max_nan(most, fabsf(v[j]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  const Fp8Scale sc = fp8_scale(most);
  scale = sc.scale;
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j] = e4m3_pair(v[2 * j] * sc.inverse, v[2 * j + 1] * sc.inverse);
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// TPR threads per row (a warp, or the CTA's 256), thread i holds the elements 8 (i + TPR c) .. + 7, c < NC, of the row in
// registers: one pass over memory, the loads of all chunks under way before the first sum. Bound by HBM from a few hundred rows on
// and by two dependent sums and the launch below that.
template <int TPR, int NC, bool XW, int Y>  // XW: x is f32; Y: 0 no block output, 1 two-byte, 2 f32
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) block_norm_vec_kernel(const NormParams p) {
  __shared__ float red[8];
  grid_dep_wait();
  const int tid = threadIdx.x, i0 = TPR == 32 ? tid & 31 : tid;
  const int64_t t = TPR == 32 ? (int64_t)blockIdx.x * 8 + (tid >> 5) : blockIdx.x;
  if (TPR == 32 && t >= p.T) return;
  auto row_sum = [&](float v) {
    if constexpr (TPR == 32) return warp_sum(v);
    else return block_sum(v, red);
  };
  const int H8 = p.H >> 3;
  Raw8 xr[NC], yr[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = i0 + TPR * c;
    if (i < H8) {
      xr[c] = load_raw8<XW>(p.x, t * p.ldx + 8 * i);
      if constexpr (Y != 0) yr[c] = load_raw8<Y == 2>(p.y, t * p.ldy + 8 * i);
    }
  }
  float rs = 1.f;
  if (Y != 0 && p.post_w) {
    auto squares = [&](float down) {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (i0 + TPR * c < H8) {
          float v[8];
          values8<Y == 2>(yr[c], p.y_dtype == KNJ_DT_BF16, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) ss = fmaf(v[j] * down, v[j] * down, ss);
        }
      }
      return row_sum(ss);
    };
    rs = rms_inverse(squares(1.f), p.H, p.eps, [&] { return squares(kDown); });
  }
  float gr = 1.f;
  if (Y != 0 && p.gate_kind == KNJ_GATE_ROW) gr = gate_value(p, t * p.ldg);
  float s[NC][8], ss = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = i0 + TPR * c;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[c][j] = 0.f;
    if (i < H8) {
      values8<XW>(xr[c], p.x_dtype == KNJ_DT_BF16, s[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[c][j] *= p.beta;
      if constexpr (Y != 0) {
        float n[8], w[8];
        values8<Y == 2>(yr[c], p.y_dtype == KNJ_DT_BF16, n);
        if (p.post_w) {
          load8(p.post_w, p.w_dtype, 8 * i, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) n[j] *= rs * w[j];
        }
        if (p.gate_kind == KNJ_GATE_CHANNEL || p.gate_kind == KNJ_GATE_FULL) {
          load8(p.gate, p.gate_dtype, (p.gate_kind == KNJ_GATE_FULL ? t * p.ldg : 0) + 8 * i, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) n[j] *= p.gate_sigmoid ? __fdividef(1.0f, 1.0f + expf(-w[j])) : w[j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) n[j] *= gr;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s[c][j] = fmaf(p.alpha, n[j], s[c][j]);
      }
      if (p.stream) store8(p.stream, p.stream_dtype, t * p.ld_stream + 8 * i, s[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(s[c][j], s[c][j], ss);
    }
  }
  if (!p.h) return;
  const float hs = rms_inverse(row_sum(ss), p.H, p.eps, [&] {
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) q = fmaf(s[c][j] * kDown, s[c][j] * kDown, q);
    return row_sum(q);
  });
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = i0 + TPR * c;
    if (i < H8) {
      float w[8];
      load8(p.pre_w, p.w_dtype, 8 * i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[c][j] *= hs * w[j];
      if (p.h_dtype != KNJ_DT_E4M3) store8(p.h, p.h_dtype, t * p.ldh + 8 * i, s[c]);
    }
    if (p.h_dtype == KNJ_DT_E4M3) {
      float scale;
      const uint2 q = codes8(s[c], scale);   // every lane takes part; lanes behind the row hold zeros
      if (i < H8) *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.h) + t * p.ldh + 8 * i) = q;
      if (i < H8 && (i & 15) == 0) p.h_scale[t * ((p.H + kFp8Group - 1) / kFp8Group) + (i >> 4)] = scale;
    }
  }
}

template <int TPR, int NC>
cudaError_t launch_vec(const NormParams &p, cudaStream_t st) {
  auto go = [&](auto kern) {
    return launch_chain(kern, dim3((unsigned)(TPR == 32 ? (p.T + 7) / 8 : p.T)), dim3(TPR == 32 ? 256 : TPR), 0, st, p);
  };
  const bool xw = p.x_dtype == KNJ_DT_F32;
  if (!p.y) return xw ? go(block_norm_vec_kernel<TPR, NC, true, 0>) : go(block_norm_vec_kernel<TPR, NC, false, 0>);
  if (p.y_dtype != KNJ_DT_F32) return xw ? go(block_norm_vec_kernel<TPR, NC, true, 1>) : go(block_norm_vec_kernel<TPR, NC, false, 1>);
  return xw ? go(block_norm_vec_kernel<TPR, NC, true, 2>) : go(block_norm_vec_kernel<TPR, NC, false, 2>);
}

// Eight values per lane, sixteen lanes per group; each lane has kUnroll groups' loads under way.
constexpr int kRowsUnroll = 4;
template <bool XW>
__global__ void __launch_bounds__(256) fp8_rows_vec_kernel(const void *x, int dtype, int64_t ldx, int rows, int K8, int groups, uint8_t *q,
                                                           float *scale) {
  grid_dep_wait();
  if (gridDim.x <= 148u) grid_dep_signal();
  const int lane16 = threadIdx.x & 15;
  const int64_t n = (int64_t)rows * groups, stride = (int64_t)gridDim.x * 16;
  for (int64_t g0 = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); __any_sync(0xffffffffu, g0 < n); g0 += stride * kRowsUnroll) {
    Raw8 r[kRowsUnroll];
    int64_t row[kRowsUnroll];
    int i[kRowsUnroll];
#pragma unroll
    for (int u = 0; u < kRowsUnroll; ++u) {
      const int64_t g = g0 + u * stride;
      row[u] = n <= 0x7fffffff ? (int64_t)((uint32_t)g / (uint32_t)groups) : g / groups;
      i[u] = (int)(g - row[u] * groups) * 16 + lane16;
      if (g >= n) i[u] = K8;
      r[u].a = r[u].b = make_uint4(0, 0, 0, 0);
      if (i[u] < K8) r[u] = load_raw8<XW>(x, row[u] * ldx + 8 * i[u]);
    }
#pragma unroll
    for (int u = 0; u < kRowsUnroll; ++u) {
      float v[8], sc;
      values8<XW>(r[u], dtype == KNJ_DT_BF16, v);
      const uint2 c = codes8(v, sc);
      if (i[u] < K8) {
        *reinterpret_cast<uint2 *>(q + (row[u] * K8 + i[u]) * 8) = c;
        if (lane16 == 0) scale[row[u] * groups + (i[u] >> 4)] = sc;
      }
    }
  }
}

// ---- any rows ------------------------------------------------------------------------------------------------------

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
  auto units = [](const void *base, int64_t ld, int dtype) { return aligned16(base) && ld * (dtype == KNJ_DT_F32 ? 4 : 2) % 16 == 0; };
  const bool vec = H % 8 == 0 && H <= 16384 && units(p.x, p.ldx, p.x_dtype) && (!p.y || units(p.y, p.ldy, p.y_dtype)) && aligned16(p.post_w) &&
                   aligned16(p.pre_w) && (!p.stream || units(p.stream, p.ld_stream, p.stream_dtype)) &&
                   (p.gate_kind != KNJ_GATE_CHANNEL || aligned16(p.gate)) &&
                   (p.gate_kind != KNJ_GATE_FULL || units(p.gate, p.ldg, p.gate_dtype)) &&
                   (!p.h || (p.h_dtype == KNJ_DT_E4M3 ? aligned16(p.h) && p.ldh % 8 == 0 : units(p.h, p.ldh, p.h_dtype)));
  if (vec) {
    // A warp per row where the rows alone fill the GPU (eight warps per SM and more) and fit its registers, else a CTA per row.
    const char *ev = getenv("KNJ_X");
    const int x = ev ? atoi(ev) : 0;
    if (x == 128) KNJ_CUDA((launch_vec<128, 2>(p, as_stream(s))));
    else if (x == 256) KNJ_CUDA((launch_vec<256, 1>(p, as_stream(s))));
    else if (x == 64) KNJ_CUDA((launch_vec<64, 4>(p, as_stream(s))));
    else if (H <= 2048 && p.T >= 8 * sm_count()) KNJ_CUDA(H <= 512 ? (launch_vec<32, 2>(p, as_stream(s))) : (launch_vec<32, 8>(p, as_stream(s))));
    else if (H <= 2048) KNJ_CUDA((launch_vec<256, 1>(p, as_stream(s))));
    else if (H <= 4096) KNJ_CUDA((launch_vec<256, 2>(p, as_stream(s))));
    else if (H <= 8192) KNJ_CUDA((launch_vec<256, 4>(p, as_stream(s))));
    else KNJ_CUDA((launch_vec<256, 8>(p, as_stream(s))));
    return launch_status("block_norm_vec_kernel");
  }
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
  const int64_t n = (int64_t)rows * groups, cap = (int64_t)sm_count() * 32;
  if (K % 8 == 0 && aligned16(x) && ldx * (x_dtype == KNJ_DT_F32 ? 4 : 2) % 16 == 0 && aligned16(q)) {
    // four groups of sixteen lanes each: as many CTAs as one pass needs, up to eight per SM
    const int64_t want = (n + 16 * kRowsUnroll - 1) / (16 * kRowsUnroll), few = n < 16ll * sm_count() * kRowsUnroll ? (n + 15) / 16 : want;
    const dim3 grid((unsigned)(few < cap / 4 ? few : cap / 4));
    if (x_dtype == KNJ_DT_F32)
      KNJ_CUDA(launch_chain(fp8_rows_vec_kernel<true>, grid, dim3(256), 0, as_stream(s), x, x_dtype, ldx, rows, K / 8, groups, static_cast<uint8_t *>(q), scale));
    else
      KNJ_CUDA(launch_chain(fp8_rows_vec_kernel<false>, grid, dim3(256), 0, as_stream(s), x, x_dtype, ldx, rows, K / 8, groups, static_cast<uint8_t *>(q), scale));
    return launch_status("fp8_rows_vec_kernel");
  }
  const int64_t blocks = (n + 7) / 8;
  fp8_rows_kernel<<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, as_stream(s)>>>(x, x_dtype, ldx, n, K, groups, static_cast<uint8_t *>(q), scale);
  return launch_status("fp8_rows_kernel");
}

}  // extern "C"
