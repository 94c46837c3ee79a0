// knj_expert_tc.cu -- products of routed rows with expert matrices held in bf16, fp16 or e4m3 (one scale for each block of
// 128 x 128), grouped by expert, and the dense e4m3 product, which is the same with one expert and all rows.
#include "knj_fp8.cuh"

using namespace knj;

namespace {

struct GemmParams {
  const void *x, *w0, *w1;
  const float *xs, *ws0, *ws1;
  const int32_t *pair_idx, *pair_cnt, *row_map;  // pair_idx null: one expert, pair i is row i
  void *out;
  int64_t ldx, ldo, idx_stride;
  int dtype, out_dtype, N, K, E, row_div, n_rows, n_pairs;
  float out_scale;
};

__device__ __forceinline__ float operand(const void *base, int dtype, int64_t i) {
  if (dtype != KNJ_DT_E4M3) return load_as_f32(base, dtype, i);
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)static_cast<const uint8_t *>(base)[i]));
  return __half2float(__ushort_as_half((unsigned short)(h2 & 0xffff)));
}

constexpr int kTN = 64, kTM = 16, kTK = 32;

// 64 outputs x 16 pairs of one expert, operands staged in shared memory as f32
template <bool GATEUP>
__global__ void __launch_bounds__(256) expert_gemm_kernel(const GemmParams p) {
  __shared__ float sx[kTM][kTK + 1], sw[GATEUP ? 2 : 1][kTN][kTK + 1];
  __shared__ int s_pair[kTM], s_row[kTM];
  const int e = blockIdx.z, n0 = blockIdx.x * kTN, m0 = blockIdx.y * kTM, tid = threadIdx.x;
  const int cnt = p.pair_idx ? min((int64_t)p.pair_cnt[e], p.idx_stride) : p.n_pairs;
  if (m0 >= cnt) return;
  if (tid < kTM) {
    int pr = -1, rw = -1;
    if (m0 + tid < cnt) {
      pr = p.pair_idx ? p.pair_idx[e * p.idx_stride + m0 + tid] : m0 + tid;
      if (pr < 0 || pr >= p.n_pairs) pr = -1;
      if (pr >= 0) rw = p.row_map ? p.row_map[pr] : pr / p.row_div;
      if (rw < 0 || rw >= p.n_rows) rw = -1;
    }
    s_pair[tid] = pr;
    s_row[tid] = rw;
  }
  __syncthreads();
  const int kb_n = (p.K + 127) / 128, nb_n = (p.N + 127) / 128;
  const int n = tid & 63, mg = tid >> 6;
  float acc[GATEUP ? 2 : 1][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kTK) {
    for (int i = tid; i < kTM * kTK; i += 256) {
      const int m = i / kTK, k = k0 + i % kTK;
      float v = 0.f;
      if (s_row[m] >= 0 && k < p.K) {
        v = operand(p.x, p.dtype, s_row[m] * p.ldx + k);
        if (p.dtype == KNJ_DT_E4M3) v *= p.xs[(int64_t)s_row[m] * kb_n + k / 128];
      }
      sx[m][i % kTK] = v;
    }
    for (int i = tid; i < kTN * kTK; i += 256) {
      const int r = i / kTK, k = k0 + i % kTK;
#pragma unroll
      for (int mat = 0; mat < (GATEUP ? 2 : 1); ++mat) {
        float v = 0.f;
        if (n0 + r < p.N && k < p.K) {
          v = operand(mat ? p.w1 : p.w0, p.dtype, ((int64_t)e * p.N + n0 + r) * p.K + k);
          if (p.dtype == KNJ_DT_E4M3) v *= (mat ? p.ws1 : p.ws0)[((int64_t)e * nb_n + (n0 + r) / 128) * kb_n + k / 128];
        }
        sw[mat][r][i % kTK] = v;
      }
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < kTK; ++k)
#pragma unroll
      for (int mat = 0; mat < (GATEUP ? 2 : 1); ++mat)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[mat][j] = fmaf(sw[mat][n][k], sx[mg * 4 + j][k], acc[mat][j]);
    __syncthreads();
  }
  if (n0 + n >= p.N) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pr = s_pair[mg * 4 + j];
    if (pr < 0) continue;
    float v = acc[0][j];
    if constexpr (GATEUP) v = v / (1.0f + expf(-v)) * acc[1][j];
    store_from_f32(p.out, p.out_dtype, pr * p.ldo + n0 + n, v * p.out_scale);
  }
}

template <bool GATEUP>
int launch_gemm(const GemmParams &p, cudaStream_t st) {
  const int64_t most = p.pair_idx ? (p.idx_stride < p.n_pairs ? p.idx_stride : p.n_pairs) : p.n_pairs;
  const int64_t gy = (most + kTM - 1) / kTM;
  KNJ_REQUIRE(gy <= 65535, "expert product: %lld pairs of one expert", (long long)most);
  expert_gemm_kernel<GATEUP><<<dim3((p.N + kTN - 1) / kTN, (unsigned)gy, p.E), 256, 0, st>>>(p);
  return launch_status("expert_gemm_kernel");
}

int check_expert(const knj_expert_gemm_args *a, bool gateup, const char *who) {
  KNJ_REQUIRE(a, "%s: null argument block", who);
  KNJ_REQUIRE(a->n_pairs >= 0 && a->n_rows >= 0 && a->N > 0 && a->K > 0 && a->n_experts >= 1 && a->n_experts <= 256, "%s: bad sizes", who);
  if (a->n_pairs == 0) return KNJ_OK;
  KNJ_REQUIRE(a->w_dtype >= KNJ_DT_BF16 && a->w_dtype <= KNJ_DT_E4M3, "%s: expert matrices are bf16, f16 or e4m3", who);
  KNJ_REQUIRE(a->x_dtype == a->w_dtype, "%s: rows (type %d) and matrices (type %d) are of one type", who, a->x_dtype, a->w_dtype);
  KNJ_REQUIRE(a->x && a->w0 && (!gateup || a->w1) && a->pair_idx && a->pair_cnt && a->out, "%s: null pointer", who);
  KNJ_REQUIRE(a->w_dtype != KNJ_DT_E4M3 || (a->x_scale && a->w0_scale && (!gateup || a->w1_scale)), "%s: e4m3 operands need their scales", who);
  const int64_t esz = a->w_dtype == KNJ_DT_E4M3 ? 1 : 2;
  KNJ_REQUIRE(a->K * esz % 16 == 0 && a->ldx * esz % 16 == 0, "%s: rows of K=%d and stride %lld are not whole 16-byte units", who, a->K,
              (long long)a->ldx);
  KNJ_REQUIRE(aligned16(a->x) && aligned16(a->w0) && (!gateup || aligned16(a->w1)), "%s: bases must be 16-byte aligned", who);
  KNJ_REQUIRE(a->ldx >= a->K && a->ldo >= a->N && a->idx_stride >= 1, "%s: strides shorter than the rows", who);
  KNJ_REQUIRE(a->row_map || a->row_div >= 1, "%s: row_div=%d", who, a->row_div);
  KNJ_REQUIRE(a->out_dtype >= KNJ_DT_F32 && a->out_dtype <= KNJ_DT_F16, "%s: outputs are f32, bf16 or f16", who);
  return KNJ_OK;
}

GemmParams params_of(const knj_expert_gemm_args *a) {
  GemmParams p{};
  p.x = a->x; p.w0 = a->w0; p.w1 = a->w1; p.xs = a->x_scale; p.ws0 = a->w0_scale; p.ws1 = a->w1_scale; p.pair_idx = a->pair_idx;
  p.pair_cnt = a->pair_cnt; p.row_map = a->row_map; p.out = a->out; p.ldx = a->ldx; p.ldo = a->ldo; p.idx_stride = a->idx_stride;
  p.dtype = a->w_dtype; p.out_dtype = a->out_dtype; p.N = a->N; p.K = a->K; p.E = a->n_experts; p.row_div = a->row_div > 0 ? a->row_div : 1;
  p.n_rows = a->n_rows; p.n_pairs = a->n_pairs; p.out_scale = a->out_scale;
  return p;
}

inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

extern "C" {

int knj_expert_gateup_launch(const knj_expert_gemm_args *a, knj_stream_t s) {
  const int rc = check_expert(a, true, "knj_expert_gateup");
  if (rc || a->n_pairs == 0) return rc;
  return launch_gemm<true>(params_of(a), as_stream(s));
}

int knj_expert_proj_launch(const knj_expert_gemm_args *a, knj_stream_t s) {
  const int rc = check_expert(a, false, "knj_expert_proj");
  if (rc || a->n_pairs == 0) return rc;
  return launch_gemm<false>(params_of(a), as_stream(s));
}

size_t knj_fp8_matmul_workspace_bytes(int m, int n_in) {
  if (m <= 0 || n_in <= 0) return 0;
  return up256((size_t)m * n_in) + up256((size_t)m * ((n_in + 127) / 128) * 4);
}

int knj_fp8_matmul_launch(const void *W, const float *W_scale, int n_in, int n_out, const void *x, int x_dtype, int64_t ldx, int m, void *y,
                          int y_dtype, int64_t ldy, void *workspace, size_t workspace_bytes, int *status, knj_stream_t s) {
  KNJ_REQUIRE(m >= 0 && n_in > 0 && n_out > 0, "knj_fp8_matmul: bad sizes");
  if (m == 0) return KNJ_OK;
  KNJ_REQUIRE(W && W_scale && x && y, "knj_fp8_matmul: null pointer");
  KNJ_REQUIRE(n_in % 16 == 0, "knj_fp8_matmul: n_in=%d must be a multiple of 16", n_in);
  KNJ_REQUIRE(aligned16(W), "knj_fp8_matmul: the matrix must be 16-byte aligned");
  KNJ_REQUIRE(x_dtype >= KNJ_DT_F32 && x_dtype <= KNJ_DT_F16, "knj_fp8_matmul: rows are f32, bf16 or f16");
  KNJ_REQUIRE(y_dtype >= KNJ_DT_F32 && y_dtype <= KNJ_DT_F16, "knj_fp8_matmul: outputs are f32, bf16 or f16");
  KNJ_REQUIRE(ldx >= n_in && ldy >= n_out, "knj_fp8_matmul: row strides shorter than the rows");
  const size_t need = knj_fp8_matmul_workspace_bytes(m, n_in);
  if (!workspace || workspace_bytes < need) {
    set_error("knj_fp8_matmul: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return KNJ_E_WORKSPACE;
  }
  KNJ_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "knj_fp8_matmul: workspace must be 256-byte aligned");
  uint8_t *q = static_cast<uint8_t *>(workspace);
  float *qs = reinterpret_cast<float *>(q + up256((size_t)m * n_in));
  const int rc = knj_fp8_rows_launch(x, x_dtype, ldx, m, n_in, q, qs, s);
  if (rc) return rc;
  GemmParams p{};
  p.x = q; p.xs = qs; p.w0 = W; p.ws0 = W_scale; p.out = y; p.ldx = n_in; p.ldo = ldy; p.dtype = KNJ_DT_E4M3; p.out_dtype = y_dtype;
  p.N = n_out; p.K = n_in; p.E = 1; p.row_div = 1; p.n_rows = m; p.n_pairs = m; p.out_scale = 1.0f;
  (void)status;
  return launch_gemm<false>(p, as_stream(s));
}

}  // extern "C"
