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
  float alpha, beta, eps, inv_h;
  int *status;
  long long wait_cycles;  // limit of the ring's waits
  int stall;              // test hook: the first row of CTA 0 never counts as landed
};

thread_local int t_stall = 0;   // knj_block_norm_test_stall

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
// they are summed once more from values * 2^-80 (`again`), of which the largest and the smallest such row's squares are in it; eps does not
// count there.
constexpr float kDown = 0x1p-80f;
// rsqrtf is off by 2 units in the last place; an IEEE root and two divisions are a hundred instructions of every thread and row.
template <class Again>
__device__ __forceinline__ float rms_inverse(float tot, float inv_h, float eps, Again again) {
  if (tot <= 3.402823466e38f || tot != tot) return rsqrtf(fmaf(tot, inv_h, eps));
  return kDown * rsqrtf(again() * inv_h);
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
// the branch on the type stands outside the loop: inside, both conversions of every value are formed and one is picked
__device__ __forceinline__ void unpack16(const uint4 &u, bool bf16, float2 (&v)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if (bf16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
  }
}
template <bool WIDE>
__device__ __forceinline__ void values8(const Raw8 &r, bool bf16, float2 (&v)[4]) {
  if constexpr (WIDE) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
  } else {
    unpack16(r.a, bf16, v);
  }
}
__device__ __forceinline__ void load8(const void *base, int dtype, int64_t i, float2 (&v)[4]) {
  if (dtype == KNJ_DT_F32) values8<true>(load_raw8<true>(base, i), false, v);
  else values8<false>(load_raw8<false>(base, i), dtype == KNJ_DT_BF16, v);
}
__device__ __forceinline__ void store8(void *base, int dtype, const float2 (&v)[4]) {
  if (dtype == KNJ_DT_F32) {
    float4 *q = static_cast<float4 *>(base);
    q[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    q[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    return;
  }
  uint32_t w[4];
  if (dtype == KNJ_DT_BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 h = __float22bfloat162_rn(v[j]);
      w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __float22half2_rn(v[j]);
      w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  *static_cast<uint4 *>(base) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float2 mul2(float2 a, float b) { return __fmul2_rn(a, make_float2(b, b)); }
__device__ __forceinline__ float2 sigmoid2(float2 g) {
  return make_float2(__fdividef(1.0f, 1.0f + expf(-g.x)), __fdividef(1.0f, 1.0f + expf(-g.y)));
}
__device__ __forceinline__ uint2 codes8(const float2 (&v)[4], float inverse) {
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 q = mul2(v[j], inverse);
    c[j] = e4m3_pair(q.x, q.y);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
// scale of a group that LANES lanes in a row hold, RUNS runs of eight values each
template <int LANES, int RUNS>
__device__ __forceinline__ Fp8Scale group_scale(const float2 (*v)[4]) {
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < RUNS; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max3_abs_nan(most, v[r][j].x, v[r][j].y);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  return fp8_scale(most);
}

// sum over the CTA; `red` has two rows of 16 (zero behind the CTA's warps), used in turn, so that one barrier a sum is enough
__device__ __forceinline__ float cta_sum(float v, float (*red)[16], int &turn) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  float *at = red[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
  __syncthreads();
  const float4 *q = reinterpret_cast<const float4 *>(at);
  float4 a = q[0], b = q[1];
  if (warps > 8) {
    const float4 c = q[2], d = q[3];
    a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
    b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
  }
  return ((a.x + b.x) + (a.y + b.y)) + ((a.z + b.z) + (a.w + b.w));
}

// The part of a bounded wait that follows its first try, a function of its own: inlined it cost the loop around it 2 us of 53.
__device__ __noinline__ bool wait_on(uint64_t *bar, uint32_t parity, long long limit, volatile int *fail) {
  return mbar_wait_for(bar, parity, limit, fail);
}

// One CTA walks over rows; a thread holds NC runs of eight values of each, and of the weights: post_w with a gate per channel and
// alpha folded in, so that a row costs a dozen operations a value (formed anew for each row, and with the gate's exponential, 57:
// 16384 rows of 2048 took 106 us, issue slots half full). Eight threads in a row hold sixteen runs in turn, a group of e4m3 codes
// (NC = 1: sixteen threads). RING: the next rows travel through a ring of `depth` rows in shared memory, bulk copies on a barrier
// each; a row ahead in registers was 24 KB under way per SM, too few for HBM (74 us). 16384 rows of 2048 in bf16 with e4m3 rows out,
// 235 MB: 51.6 us, 4.55 TB/s; bound by the two sums over the CTA that wait for one another, with five warps per scheduler (four, with
// the block's output unpacked once: 57.7). Six with the weights in shared memory: 67 us, the rows no longer fit 80 registers.
// Without the ring, one row per CTA straight into registers: bound by the launch and the two sums (one row of 2048: 2.6 us).
// A wait of the ring that gives up does so for the whole CTA and for good: from then on it starts no copy and asks no barrier (one
// whose phase never completed would pass the next lap's wait), every row that it still has is NaN, and its copies under way are given
// kLinger cycles to land before its shared memory is handed on.
constexpr int kMaxRing = 8;
constexpr long long kLinger = 1ll << 20;
template <int NC, bool XW, int Y, bool RING>  // XW: x is f32; Y: 0 no block output, 1 two-byte, 2 f32
__global__ void __maxnreg__(!RING || NC == 4 ? 128 : NC == 1 ? 64 : Y == 0 ? 80 : XW || Y == 2 ? 128 : 96) block_norm_vec_kernel(const NormParams p, const int depth) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(16) float red[2][16];
  __shared__ uint64_t bars[kMaxRing];
  __shared__ volatile int s_fail;
  int turn = 0;
  if (threadIdx.x < 32) red[threadIdx.x >> 4][threadIdx.x & 15] = 0.f;
  __syncthreads();
  grid_dep_wait();
  constexpr int kLanes = NC == 1 ? 16 : 8;
  const int tid = threadIdx.x, H8 = p.H >> 3, first = (tid / kLanes) * (kLanes * NC) + tid % kLanes;   // runs first + kLanes c
  const bool xb = p.x_dtype == KNJ_DT_BF16, yb = p.y_dtype == KNJ_DT_BF16;
  Raw8 xr[NC], yr[NC];
  const int x_bytes = p.H * (XW ? 4 : 2), y_bytes = Y == 0 ? 0 : p.H * (Y == 2 ? 4 : 2);
  auto send = [&](int slot, int64_t t) {   // one thread
    uint8_t *at = ring + (size_t)slot * (x_bytes + y_bytes);
    mbar_expect_tx(&bars[slot], (uint32_t)(x_bytes + y_bytes));
    bulk_g2s(at, static_cast<const uint8_t *>(p.x) + t * p.ldx * (XW ? 4 : 2), (uint32_t)x_bytes, &bars[slot]);
    if (Y != 0) bulk_g2s(at + x_bytes, static_cast<const uint8_t *>(p.y) + t * p.ldy * (Y == 2 ? 4 : 2), (uint32_t)y_bytes, &bars[slot]);
  };
  auto fetch = [&](const void *x, const void *y, int64_t xo, int64_t yo) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = first + kLanes * c;
      xr[c].a = xr[c].b = yr[c].a = yr[c].b = make_uint4(0, 0, 0, 0);
      if (i < H8) {
        xr[c] = load_raw8<XW>(x, xo + 8 * i);
        if constexpr (Y != 0) yr[c] = load_raw8<Y == 2>(y, yo + 8 * i);
      }
    }
  };
  if constexpr (RING) {
    if (tid == 0) {
      for (int r = 0; r < depth; ++r) mbar_init(&bars[r], p.stall && blockIdx.x == 0 && r == 0 ? 2 : 1);
      s_fail = 0;
      mbar_init_fence();
      int64_t t = blockIdx.x;
      for (int r = 0; r < depth && t < p.T; ++r, t += gridDim.x) send(r, t);
    }
    __syncthreads();
  } else {
    fetch(p.x, p.y, blockIdx.x * p.ldx, blockIdx.x * p.ldy);
  }
  // alpha * post_w * gate per channel, and pre_w; kept in registers where they fit, else formed for each row
  auto post_of = [&](int c, float2 (&f)[4]) {
    const int i = first + kLanes * c;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(p.alpha, p.alpha);
    if (Y == 0 || i >= H8) return;
    float2 w[4];
    if (p.post_w) {
      load8(p.post_w, p.w_dtype, 8 * i, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __fmul2_rn(f[j], w[j]);
    }
    if (p.gate_kind == KNJ_GATE_CHANNEL) {
      load8(p.gate, p.gate_dtype, 8 * i, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __fmul2_rn(f[j], p.gate_sigmoid ? sigmoid2(w[j]) : w[j]);
    }
  };
  auto pre_of = [&](int c, float2 (&f)[4]) {
    const int i = first + kLanes * c;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(0.f, 0.f);
    if (p.h && i < H8) load8(p.pre_w, p.w_dtype, 8 * i, f);
  };
  constexpr bool kKeep = NC <= 2;
  float2 post[kKeep ? NC : 1][4], pre[kKeep ? NC : 1][4];
  if constexpr (kKeep) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      post_of(c, post[c]);
      pre_of(c, pre[c]);
    }
  }
  // sum of squares over the row, of values * kDown where `down`; of(c, v): the run's values
  auto squares = [&](auto of, bool down) {
    float2 a = make_float2(0.f, 0.f), b = a;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float2 v[4];
      of(c, v);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 x = down ? mul2(v[j], kDown) : v[j], y = down ? mul2(v[j + 1], kDown) : v[j + 1];
        a = __ffma2_rn(x, x, a);
        b = __ffma2_rn(y, y, b);
      }
    }
    a = __fadd2_rn(a, b);
    return cta_sum(a.x + a.y, red, turn);
  };
  const int groups = (p.H + kFp8Group - 1) / kFp8Group;
  int slot = 0;
  uint32_t phase = 0;
  auto advance = [&] {
    if (++slot == depth) {
      slot = 0;
      phase ^= 1u;
    }
  };
  // where this thread's first run of the row lies in what is written, moved on row by row
  const int s_esz = p.stream_dtype == KNJ_DT_F32 ? 4 : 2, h_esz = p.h_dtype == KNJ_DT_E4M3 ? 1 : p.h_dtype == KNJ_DT_F32 ? 4 : 2;
  uint8_t *s_at = static_cast<uint8_t *>(p.stream) + (blockIdx.x * p.ld_stream + 8 * first) * s_esz;
  uint8_t *h_at = static_cast<uint8_t *>(p.h) + (blockIdx.x * p.ldh + 8 * first) * h_esz;
  const int64_t s_step = gridDim.x * p.ld_stream * s_esz, h_step = gridDim.x * p.ldh * h_esz;
  int64_t t = blockIdx.x;
  for (; t < p.T; t += gridDim.x, s_at += s_step, h_at += h_step) {
    float2 s[NC][4];
    if constexpr (RING) {
      const bool landed = mbar_try_wait(&bars[slot], phase) || wait_on(&bars[slot], phase, p.wait_cycles, &s_fail);
      const uint8_t *at = ring + (size_t)slot * (x_bytes + y_bytes);
      fetch(at, at + x_bytes, 0, 0);
      if (__syncthreads_or(!landed)) break;                // every thread has its part of the row
      if (tid == 0 && t + (int64_t)depth * gridDim.x < p.T) {
        fence_proxy_async();                               // the slot was read through the generic proxy
        send(slot, t + (int64_t)depth * gridDim.x);
      }
      advance();
    }
    float rs = 1.f;
    // y is unpacked here and once more below: in the type it came in it takes half of the registers meanwhile
    auto y_of = [&](int c, float2 (&v)[4]) { values8<Y == 2>(yr[c], yb, v); };
    if (Y != 0 && p.post_w) rs = rms_inverse(squares(y_of, false), p.inv_h, p.eps, [&] { return squares(y_of, true); });
    // The inverse norm meets y before anything else does: y * rs is of order one, y times a gate may be infinite and rs times one denormal.
    float row_gate = 1.f;
    if (Y != 0 && p.gate_kind == KNJ_GATE_ROW) row_gate = gate_value(p, t * p.ldg);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = first + kLanes * c;
      if (!kKeep) post_of(c, post[0]);
      values8<XW>(xr[c], xb, s[c]);
      if (i < H8) {
        float2 n[4];
        if constexpr (Y != 0) y_of(c, n);
        if (Y != 0 && p.gate_kind == KNJ_GATE_FULL) {
          float2 w[4];
          load8(p.gate, p.gate_dtype, t * p.ldg + 8 * i, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) n[j] = __fmul2_rn(mul2(n[j], rs), p.gate_sigmoid ? sigmoid2(w[j]) : w[j]);
        } else if (Y != 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) n[j] = mul2(n[j], rs);
          if (p.gate_kind == KNJ_GATE_ROW) {
#pragma unroll
            for (int j = 0; j < 4; ++j) n[j] = mul2(n[j], row_gate);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[c][j] = mul2(s[c][j], p.beta);
          if constexpr (Y != 0) s[c][j] = __ffma2_rn(n[j], post[kKeep ? c : 0][j], s[c][j]);
        }
        if (p.stream) store8(s_at + 8 * kLanes * c * s_esz, p.stream_dtype, s[c]);
      }
    }
    if (!p.h) continue;
    auto s_of = [&](int c, float2 (&v)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = s[c][j];
    };
    const float hs = rms_inverse(squares(s_of, false), p.inv_h, p.eps, [&] { return squares(s_of, true); });
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (!kKeep) pre_of(c, pre[0]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[c][j] = __fmul2_rn(mul2(s[c][j], hs), pre[kKeep ? c : 0][j]);   // zeros behind the row
    }
    if (p.h_dtype != KNJ_DT_E4M3) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (first + kLanes * c < H8) store8(h_at + 8 * kLanes * c * h_esz, p.h_dtype, s[c]);
    } else {
      constexpr int kRuns = 16 / kLanes;   // of a thread in a group
#pragma unroll
      for (int c = 0; c < NC; c += kRuns) {
        const Fp8Scale sc = group_scale<kLanes, kRuns>(&s[c]);   // every lane takes part
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
          if (first + kLanes * (c + r) < H8) *reinterpret_cast<uint2 *>(h_at + 8 * kLanes * (c + r)) = codes8(s[c + r], sc.inverse);
        const int i = first + kLanes * c;
        if (i < H8 && (i & 15) == 0) p.h_scale[t * groups + (i >> 4)] = sc.scale;
      }
    }
  }
  if constexpr (RING) {
    if (t >= p.T) return;
    if (tid == 0) {
      if (p.status) atomicExch(p.status, 1);
      for (int64_t r = t; r < p.T && r < t + (int64_t)depth * gridDim.x; r += gridDim.x, advance()) mbar_wait_for(&bars[slot], phase, kLinger, nullptr);
    }
    const float nan = __int_as_float(0x7fffffff);
    const float2 v[4] = {{nan, nan}, {nan, nan}, {nan, nan}, {nan, nan}};
    for (; t < p.T; t += gridDim.x, s_at += s_step, h_at += h_step)
#pragma unroll 1
      for (int c = 0; c < NC; ++c) {
        const int i = first + kLanes * c;
        if (i >= H8) continue;
        if (p.stream) store8(s_at + 8 * kLanes * c * s_esz, p.stream_dtype, v);
        if (!p.h) continue;
        if (p.h_dtype != KNJ_DT_E4M3) store8(h_at + 8 * kLanes * c * h_esz, p.h_dtype, v);
        else *reinterpret_cast<uint2 *>(h_at + 8 * kLanes * c) = codes8(v, 1.f);
        if (p.h_dtype == KNJ_DT_E4M3 && (i & 15) == 0) p.h_scale[t * groups + (i >> 4)] = nan;
      }
  }
}

template <int NC, bool RING>
cudaError_t launch_vec(const NormParams &p, int threads, unsigned ctas, int depth, size_t smem, cudaStream_t st) {
  auto go = [&](auto kern) {
    if (smem > 40 * 1024) {   // 48 KB less the static part need no opt-in
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
      if (e != cudaSuccess) return e;
    }
    return launch_chain(kern, dim3(ctas), dim3(threads), smem, st, p, depth);
  };
  const bool xw = p.x_dtype == KNJ_DT_F32;
  if (!p.y) return xw ? go(block_norm_vec_kernel<NC, true, 0, RING>) : go(block_norm_vec_kernel<NC, false, 0, RING>);
  if (p.y_dtype != KNJ_DT_F32) return xw ? go(block_norm_vec_kernel<NC, true, 1, RING>) : go(block_norm_vec_kernel<NC, false, 1, RING>);
  return xw ? go(block_norm_vec_kernel<NC, true, 2, RING>) : go(block_norm_vec_kernel<NC, false, 2, RING>);
}
template <int NC>
cudaError_t launch_vec(const NormParams &p, int threads, cudaStream_t st) {
  // Rows that one wave of CTAs holds (512 threads per SM) take one CTA each; more walk through the ring, as many CTAs as are resident
  // and their rows under way as fit 160 KB per SM.
  if (p.T <= sm_count() * (512 / threads)) return launch_vec<NC, false>(p, threads, (unsigned)p.T, 0, 0, st);
  const bool wide = p.x_dtype == KNJ_DT_F32 || p.y_dtype == KNJ_DT_F32;
  const int resident = NC == 1 ? 1024 : NC == 4 ? 512 : !p.y ? 768 : wide ? 512 : 640, per_sm = threads < resident ? resident / threads : 1;
  const int cap = sm_count() * per_sm;
  const size_t row = (size_t)p.H * ((p.x_dtype == KNJ_DT_F32 ? 4 : 2) + (!p.y ? 0 : p.y_dtype == KNJ_DT_F32 ? 4 : 2));
  int depth = (int)(160 * 1024 / per_sm / row);
  int ctas = cap;
  if (depth < 2) {   // long rows: one CTA per SM
    depth = (int)(200 * 1024 / row);
    if (depth < 1) depth = 1;
    ctas = sm_count();
  }
  if (depth > kMaxRing) depth = kMaxRing;
  return launch_vec<NC, true>(p, threads, (unsigned)ctas, depth, depth * row, st);
}

// Eight lanes per group, two runs of eight values each. The loop is short on purpose: 40 registers keep six CTAs on an SM, and their
// loads cover HBM's latency (8192 x 4096 bf16, 101 MB: 17.7 us in a loop over more than L2, 24.6 by itself with the launch; a group or
// three more per lane under way, by itself: 24.6 and 28.7).
constexpr int kRowsCtas = 6;
template <bool XW>
__global__ void __launch_bounds__(256, kRowsCtas) fp8_rows_vec_kernel(const void *x, int dtype, int64_t ldx, int rows, int K8, int groups,
                                                                      uint8_t *q, float *scale) {
  grid_dep_wait();
  if (gridDim.x <= 148u) grid_dep_signal();
  const int lane8 = threadIdx.x & 7;
  const int64_t n = (int64_t)rows * groups, stride = (int64_t)gridDim.x * 32;
  for (int64_t g = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3); __any_sync(0xffffffffu, g < n); g += stride) {
    const int64_t row = n <= 0x7fffffff ? (int64_t)((uint32_t)g / (uint32_t)groups) : g / groups;
    const int i = g < n ? (int)(g - row * groups) * 16 + lane8 : K8;
    float2 v[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Raw8 r;
      r.a = r.b = make_uint4(0, 0, 0, 0);
      if (i + 8 * h < K8) r = load_raw8<XW>(x, row * ldx + 8 * (i + 8 * h));
      values8<XW>(r, dtype == KNJ_DT_BF16, v[h]);
    }
    const Fp8Scale sc = group_scale<8, 2>(v);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (i + 8 * h < K8) *reinterpret_cast<uint2 *>(q + (row * K8 + i + 8 * h) * 8) = codes8(v[h], sc.inverse);
    if (lane8 == 0 && i < K8) scale[g] = sc.scale;
  }
}

// ---- any rows ------------------------------------------------------------------------------------------------------

// element of a lane's k-th value of a group of 128
__device__ __forceinline__ int any_at(int group, int lane, int k) { return group * kFp8Group + 32 * k + lane; }
template <class F>
__device__ __forceinline__ void of_type(int dtype, F f) {   // f(example of the type): the branch around a run of loads, not inside
  if (dtype == KNJ_DT_F32) f(float());
  else if (dtype == KNJ_DT_BF16) f(__nv_bfloat16());
  else f(__half());
}
__device__ __forceinline__ void any_load(const void *base, int dtype, int64_t row, int group, int lane, int n, float (&v)[4]) {
  of_type(dtype, [&](auto ex) {
    const decltype(ex) *q = static_cast<const decltype(ex) *>(base) + row;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = any_at(group, lane, k);
      v[k] = i < n ? (float)q[i] : 0.f;
    }
  });
}
__device__ __forceinline__ void any_store(void *base, int dtype, int64_t row, int group, int lane, int n, const float (&v)[4]) {
  of_type(dtype, [&](auto ex) {
    decltype(ex) *q = static_cast<decltype(ex) *>(base) + row;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = any_at(group, lane, k);
      if (i < n) q[i] = (decltype(ex))v[k];
    }
  });
}
// a warp's group as codes; every lane takes part
__device__ __forceinline__ void any_codes(const float (&v)[4], uint8_t *q, float *scale, int64_t row, int group, int lane, int n) {
  float most = max3_abs_nan(max3_abs_nan(0.f, v[0], v[1]), v[2], v[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  const Fp8Scale sc = fp8_scale(most);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = any_at(group, lane, k);
    if (i < n) q[row + i] = (uint8_t)e4m3_pair(v[k] * sc.inverse, 0.f);
  }
  if (lane == 0) *scale = sc.scale;
}

// One CTA per row; a warp holds NC groups of 128 values, a lane every 32nd value of each, so that any row's accesses are runs of 32
// elements. Two groups a warp: 40 registers, six CTAs of 256 threads: 16384 x 2047, e4m3 rows out, 145 us
// (with 48 registers and five CTAs 167); bound by a row's sums, during which nothing of another row is under way in its CTA.
template <int NC>
__global__ void __launch_bounds__(NC == 2 ? 512 : 1024, NC == 2 ? 3 : 1) block_norm_any_kernel(const NormParams p) {
  __shared__ float red[32];
  grid_dep_wait();
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, H = p.H;
  const int groups = (H + kFp8Group - 1) / kFp8Group;
  float s[NC][4], n[NC][4], w[4];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    any_load(p.x, p.x_dtype, t * p.ldx, warp + warps * c, lane, H, s[c]);
    if (p.y) any_load(p.y, p.y_dtype, t * p.ldy, warp + warps * c, lane, H, n[c]);
  }
  auto squares = [&](const float (&v)[NC][4], float down) {
    float a = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) a = fmaf(v[c][k] * down, v[c][k] * down, a);
    return block_sum(a, red);
  };
  // the inverse norm meets y before anything else does: see the 16-byte form
  auto times = [&](float f) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) n[c][k] *= f;
  };
  if (p.y && p.post_w) times(rms_inverse(squares(n, 1.f), p.inv_h, p.eps, [&] { return squares(n, kDown); }));
  if (p.gate_kind == KNJ_GATE_ROW) times(gate_value(p, t * p.ldg));
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int g = warp + warps * c;
    if (g >= groups) break;
#pragma unroll
    for (int k = 0; k < 4; ++k) s[c][k] *= p.beta;
    if (p.y) {
      if (p.post_w) {
        any_load(p.post_w, p.w_dtype, 0, g, lane, H, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) n[c][k] *= w[k];
      }
      if (p.gate_kind == KNJ_GATE_CHANNEL || p.gate_kind == KNJ_GATE_FULL) {
        any_load(p.gate, p.gate_dtype, p.gate_kind == KNJ_GATE_FULL ? t * p.ldg : 0, g, lane, H, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) n[c][k] *= p.gate_sigmoid ? __fdividef(1.0f, 1.0f + expf(-w[k])) : w[k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s[c][k] = any_at(g, lane, k) < H ? fmaf(n[c][k], p.alpha, s[c][k]) : 0.f;
    }
    if (p.stream) any_store(p.stream, p.stream_dtype, t * p.ld_stream, g, lane, H, s[c]);
  }
  if (!p.h) return;
  const float hs = rms_inverse(squares(s, 1.f), p.inv_h, p.eps, [&] { return squares(s, kDown); });
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int g = warp + warps * c;
    if (g >= groups) break;
    any_load(p.pre_w, p.w_dtype, 0, g, lane, H, w);
#pragma unroll
    for (int k = 0; k < 4; ++k) s[c][k] = s[c][k] * hs * w[k];
    if (p.h_dtype != KNJ_DT_E4M3) any_store(p.h, p.h_dtype, t * p.ldh, g, lane, H, s[c]);
    else any_codes(s[c], static_cast<uint8_t *>(p.h), p.h_scale + t * groups + g, t * p.ldh, g, lane, H);
  }
}

// Rows above 16384 values: one CTA per row, the row of s in shared memory.
__global__ void __launch_bounds__(256) block_norm_kernel(const NormParams p) {
  extern __shared__ float row[];
  __shared__ float red[32];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  float rs = 1.f;
  if (p.y && p.post_w) {
    float ss = 0.f;
    for (int i = tid; i < p.H; i += 256) {
      const float v = load_as_f32(p.y, p.y_dtype, t * p.ldy + i);
      ss = fmaf(v, v, ss);
    }
    rs = rms_inverse(block_sum(ss, red), p.inv_h, p.eps, [&] {
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
  const float hs = rms_inverse(block_sum(ss, red), p.inv_h, p.eps, [&] {
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
    float v[4];
    any_load(p.pre_w, p.w_dtype, 0, g, lane, p.H, v);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (any_at(g, lane, k) < p.H) v[k] *= row[any_at(g, lane, k)] * hs;
    any_codes(v, static_cast<uint8_t *>(p.h), p.h_scale + t * groups + g, t * p.ldh, g, lane, p.H);
  }
}

// One warp per group.
__global__ void __launch_bounds__(256) fp8_rows_kernel(const void *x, int dtype, int64_t ldx, int64_t n_groups, int K, int groups,
                                                       uint8_t *q, float *scale) {
  const int lane = threadIdx.x & 31;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < n_groups; w += (int64_t)gridDim.x * 8) {
    const int64_t t = w / groups;
    const int g = (int)(w - t * groups);
    float v[4];
    any_load(x, dtype, t * ldx, g, lane, K, v);
    any_codes(v, q, scale + w, t * K, g, lane, K);
  }
}

}  // namespace

namespace knj {
int block_norm_check(const knj_block_norm_args *a) {
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
  return KNJ_OK;
}
}  // namespace knj

extern "C" {

void knj_block_norm_test_stall(int on) { t_stall = on & 1; }

int knj_block_norm_launch(const knj_block_norm_args *a, knj_stream_t s) {
  const int rc = block_norm_check(a);
  if (rc || a->n_tokens == 0) return rc;
  const int H = a->hidden;
  NormParams p{};
  p.x = a->x; p.y = a->y; p.post_w = a->post_w; p.gate = a->gate; p.pre_w = a->pre_w; p.stream = a->stream_out; p.h = a->h;
  p.h_scale = a->h_scale; p.ldx = a->ldx; p.ldy = a->ldy; p.ldg = a->ldg; p.ld_stream = a->ld_stream; p.ldh = a->ldh;
  p.T = a->n_tokens; p.H = H; p.x_dtype = a->x_dtype; p.y_dtype = a->y_dtype; p.w_dtype = a->w_dtype; p.gate_dtype = a->gate_dtype;
  p.gate_kind = a->gate_kind; p.gate_sigmoid = a->gate_sigmoid; p.stream_dtype = a->stream_dtype; p.h_dtype = a->h_dtype;
  p.alpha = a->alpha; p.beta = a->beta; p.eps = a->eps; p.inv_h = 1.0f / (float)H;
  p.status = a->status; p.wait_cycles = decode_wait_cycles(); p.stall = t_stall;
  auto units = [](const void *base, int64_t ld, int dtype) { return aligned16(base) && ld * (dtype == KNJ_DT_F32 ? 4 : 2) % 16 == 0; };
  const bool vec = H % 8 == 0 && H <= 16384 && units(p.x, p.ldx, p.x_dtype) && (!p.y || units(p.y, p.ldy, p.y_dtype)) && aligned16(p.post_w) &&
                   aligned16(p.pre_w) && (!p.stream || units(p.stream, p.ld_stream, p.stream_dtype)) &&
                   (p.gate_kind != KNJ_GATE_CHANNEL || aligned16(p.gate)) &&
                   (p.gate_kind != KNJ_GATE_FULL || units(p.gate, p.ldg, p.gate_dtype)) &&
                   (!p.h || (p.h_dtype == KNJ_DT_E4M3 ? aligned16(p.h) && p.ldh % 8 == 0 : units(p.h, p.ldh, p.h_dtype)));
  if (vec) {
    // one run of eight values per thread up to 1024 values a row, two up to 8192, four up to 16384
    const int runs = H <= 1024 ? 1 : H <= 8192 ? 2 : 4;
    int threads = 32;
    while (threads * 8 * runs < H) threads *= 2;
    if (runs == 1) KNJ_CUDA((launch_vec<1>(p, threads, as_stream(s))));
    else if (runs == 2) KNJ_CUDA((launch_vec<2>(p, threads, as_stream(s))));
    else KNJ_CUDA((launch_vec<4>(p, threads, as_stream(s))));
    return launch_status("block_norm_vec_kernel");
  }
  if (H <= 16384) {
    // two groups of 128 per warp up to 4096 values, four behind that
    const int groups = (H + kFp8Group - 1) / kFp8Group, nc = H <= 4096 ? 2 : 4;
    const dim3 grid((unsigned)p.T), block(32 * ((groups + nc - 1) / nc));
    if (nc == 2) KNJ_CUDA(launch_chain(block_norm_any_kernel<2>, grid, block, 0, as_stream(s), p));
    else KNJ_CUDA(launch_chain(block_norm_any_kernel<4>, grid, block, 0, as_stream(s), p));
    return launch_status("block_norm_any_kernel");
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
    const int64_t want = (n + 31) / 32, most = (int64_t)kRowsCtas * sm_count();
    const dim3 grid((unsigned)(want < most ? want : most));
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
