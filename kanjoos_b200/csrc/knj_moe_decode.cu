// knj_moe_decode.cu -- a whole MoE block of a residual stream for up to sixteen tokens in one cooperative launch, experts in bf16,
// fp16, e4m3 (one scale for each block of 128 x 128) or int8 (one for each output channel):
//   h   = norm(x; pre_w)
//   y   = sum over the top_k experts of softmax weight * down(silu(gate(h)) * up(h))
//   out = beta * x + alpha * g * norm(y; post_w),   h_next = norm(out; next_w)
// What is computed between x and out stays in f32, and so does what the matrices are multiplied with: a row of f32 values goes to the
// tensor core as two 16-bit planes, hi = round(v) and lo = round(v - hi), which together hold 17 bits of v (bf16 experts, bf16 planes) or 22
// (fp16 planes under a power of two for each row, for the others: their codes are exact in fp16). The planes of eight rows fill the
// sixteen rows of mma.sync.m16n8k16, so that the second one costs nothing while a step's weights are on their way.
//
// Bound by the bytes of the experts that the tokens use, each read once: one token, 8 experts of 2048 x 768 in bf16, 75.5 MB. Weights go
// straight from HBM to registers (16 bytes a lane, eight loads under way), where they are MMA fragments as they lie: the order of K
// is free as long as both operands have the same, and a lane takes eight consecutive k of one matrix row for two MMAs.
// tcgen05 would want them in shared memory first and gives nothing: the tensor work of a token is a fiftieth of the time.
//
// Stages, with a barrier over the grid between them:
//   1  norm statistics (every CTA, all tokens) and router logits (an expert or two a CTA)
//   2  top-k (every CTA for itself); gate, up, silu: every CTA has the same number of matrix rows, of all active experts in a row
//   3  down, likewise
//   4  weighted sum, norm, gate, residual, next norm: a CTA for each token
// Every wait is bounded (knj_decode_wait_limit): on give-up the status word is raised and the outputs are NaN.
#include "knj_fp8.cuh"
#include "knj_topk.cuh"

using namespace knj;

namespace {

constexpr int kMaxTokens = KNJ_MOE_DECODE_MAX_TOKENS, kMaxK = 8, kMaxExperts = 256;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kDepth = 4;                      // steps of 64 bytes a matrix row whose loads are under way
constexpr int kRed = 32 * 1024;                // bytes of the partial sums of a batch of tiles
constexpr int kPanel = 176 * 1024;             // bytes of the planes of the rows in use
constexpr int kMaxItems = 64;
constexpr float kDown = 0x1p-64f;

enum Kind { kBf16 = 0, kF16 = 1, kE4 = 2, kS8 = 3 };

struct DecodeParams {
  const void *x, *pre_w, *post_w, *next_w, *gate;
  const uint16_t *router;
  const float *router_bias;
  const uint8_t *w_gate, *w_up, *w_down;
  const float *s_gate, *s_up, *s_down;
  void *out, *h_next;
  float *h_next_scale;
  int32_t *tap_exp;
  float *tap_w;
  float *logits, *act, *Y;
  unsigned *sync;               // [0] arrivals, [1] raised by a wait that gave up; zero before the launch
  int32_t *status;
  int64_t ldx, ldo, ldg, ldh;
  int T, H, F, E, k;
  int x_dtype, out_dtype, norm_dtype, gate_dtype, h_dtype, gate_kind, gate_sigmoid;
  int x_vec;                    // rows of x are whole 16-byte units
  float alpha, beta, eps;
  long long wait_cycles;
  int stall;                    // test hook: this barrier's target is out of reach
};
thread_local int t_stall = 0;

// a run of matrix rows of one expert, and the rows of activations that go through them: `n` of them from the expert's slot `first` on
struct Item {
  int expert, r0, r1, first, n, panel;
};
struct Plan {
  Item item[kMaxItems];
  int n_items, rounds_k;        // parts of K a tile is split into
};

struct Shared {
  float part[kWarps][4];
  float inv[kMaxTokens], mult[kMaxTokens], unmult[kMaxTokens];
  int sel_e[kMaxTokens][kMaxK];
  float sel_w[kMaxTokens][kMaxK];
  unsigned mask[kMaxExperts];
  int active[kMaxTokens * kMaxK];
  int n_active, ok;
  Plan plan[2];                 // gate and up, down
  unsigned row_max[kMaxTokens];
  float row_mult[kMaxTokens], row_unmult[kMaxTokens];   // of the panel's rows
  float red[2][kWarps];
};

// ---- small pieces -------------------------------------------------------------------------------------------------------

__device__ __forceinline__ unsigned ld_acquire(const unsigned *p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Barrier over the grid, number `n` of the launch. False for all threads of the CTA where it did not complete in time.
__device__ __forceinline__ bool grid_barrier(const DecodeParams &p, Shared &s, int n) {
  __syncthreads();
  if (threadIdx.x == 0) {
    asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(p.sync), "r"(1u) : "memory");
    const unsigned target = gridDim.x * (unsigned)n + (p.stall == n ? 1u : 0u);
    const long long t0 = clock64();
    int ok = 1;
    while (ld_acquire(p.sync) < target) {
      if (ld_acquire(p.sync + 1) != 0u || clock64() - t0 > p.wait_cycles) {
        atomicExch(p.sync + 1, 1u);
        atomicExch(p.status, 1);
        ok = 0;
        break;
      }
    }
    s.ok = ok;
  }
  __syncthreads();
  return s.ok != 0;
}

__device__ __forceinline__ uint4 load_weights(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// eight consecutive values of a row; `vec`: at a 16-byte boundary
__device__ __forceinline__ void load8(const void *base, int dtype, int64_t i, bool vec, float (&v)[8]) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = load_as_f32(base, dtype, i + j);
    return;
  }
  if (dtype == KNJ_DT_F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i), b = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + i);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = dtype == KNJ_DT_BF16 ? make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u))
                                          : __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

// The power of two under which a row with largest magnitude m goes into fp16 planes: m comes to 2^14 .. 2^15, so that the low plane of a
// value keeps its bits down to 2^-40 of m. (m of 0, infinity or NaN: any will do.)
__device__ __forceinline__ void row_power(float m, float &mult, float &unmult) {
  const int e = max((int)(__float_as_uint(m) >> 23 & 255u) - 127, -100);
  mult = __uint_as_float((uint32_t)(14 - e + 127) << 23);
  unmult = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
}

template <int KIND>
__device__ __forceinline__ void planes2(float a, float b, uint32_t &hi, uint32_t &lo) {
  if constexpr (KIND == kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
  }
}

template <int KIND>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (KIND == kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
}

// four codes as two pairs of fp16
template <int KIND>
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t &p0, uint32_t &p1) {
  if constexpr (KIND == kE4) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p0) : "h"((uint16_t)w));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p1) : "h"((uint16_t)(w >> 16)));
  } else {
    // 0x6400 + u is the fp16 of 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    p0 = *reinterpret_cast<const uint32_t *>(&x);
    p1 = *reinterpret_cast<const uint32_t *>(&y);
  }
}

__device__ __forceinline__ float cta_sum(float v, float *red) {   // red: kWarps words, not in use by an earlier sum
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) t += red[i];
  return t;
}

template <int KIND>
struct Geo {
  static constexpr int kElem = KIND <= kF16 ? 2 : 1;
  // bytes of a plane of K values: whole steps, and rows an odd 64 (of codes: 16) bytes apart, so that the eight lanes that a load of
  // shared memory serves at a time (two rows, four runs of k) find all banks
  __host__ __device__ static int pitch(int K) { return (2 * K + 127) / 128 * 128 + (kElem == 2 ? 64 : 16); }
  __host__ __device__ static int cap(int K) { const int c = kPanel / (2 * pitch(K)); return c < kMaxTokens ? c : kMaxTokens; }
};

// ---- products -----------------------------------------------------------------------------------------------------------

// What a warp does in a product: a tile is eight rows of gate and the same eight of up, or sixteen rows of down; `part` of `parts` of
// its K, and the tiles `group`, `group` + `groups`, .. of each item.
struct Split {
  int parts, groups, part, group, s0, s1;   // steps s0 .. s1-1
};

// The loads of a warp, kDepth steps ahead of its products: they walk over the same tiles and steps in the same order.
template <int KIND, bool GATEUP>
struct Feed {
  uint4 w[kDepth][2];
  float sc[kDepth][2];         // e4m3: scales of the blocks, for the columns of this lane's sums
  const uint8_t *p0, *p1;      // this lane's bytes of the tile
  const float *q0, *q1;        // scales' rows
  int item, tile, step;        // step: first of the block of kDepth
  bool row0, row1;             // rows of this item
};

template <int KIND, bool GATEUP>
struct Product {
  static constexpr int kElem = Geo<KIND>::kElem;
  static constexpr int kRows = GATEUP ? 8 : 16;
  const DecodeParams &p;
  const Plan &plan;
  Split sp;
  int K, N, row_bytes, lane;

  __device__ __forceinline__ int tiles(const Item &it) const { return (it.r1 - it.r0 + kRows - 1) / kRows; }
  __device__ __forceinline__ void at_tile(Feed<KIND, GATEUP> &f) const {   // pointers of the feed's tile; steps over items without one for this warp
    while (f.item < plan.n_items && f.tile >= tiles(plan.item[f.item])) {
      ++f.item;
      f.tile = sp.group;
    }
    if (f.item >= plan.n_items) return;
    const Item &it = plan.item[f.item];
    const int r = it.r0 + f.tile * kRows + (lane >> 2), r2 = GATEUP ? r : r + 8;
    f.row0 = r < it.r1;
    f.row1 = r2 < it.r1;
    const int64_t at = (int64_t)it.expert * N;
    f.p0 = (GATEUP ? p.w_gate : p.w_down) + (at + r) * row_bytes + (lane & 3) * 16;
    f.p1 = (GATEUP ? p.w_up : p.w_down) + (at + r2) * row_bytes + (lane & 3) * 16;
    if constexpr (KIND == kE4) {
      // sums of columns 2 (lane & 3), + 1: runs start at even rows, so both are in one block
      const int c = it.r0 + f.tile * kRows + 2 * (lane & 3), c2 = GATEUP ? c : c + 8, kb = (K + 127) / 128, nb = (N + 127) / 128;
      f.q0 = (GATEUP ? p.s_gate : p.s_down) + ((int64_t)it.expert * nb + min(c / 128, nb - 1)) * kb;
      f.q1 = (GATEUP ? p.s_up : p.s_down) + ((int64_t)it.expert * nb + min(c2 / 128, nb - 1)) * kb;
    }
  }
  __device__ __forceinline__ void start(Feed<KIND, GATEUP> &f) const {
    f.item = sp.group < sp.groups ? 0 : plan.n_items;
    f.tile = sp.group;
    f.step = sp.s0;
    at_tile(f);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) issue(f, d);
    next(f);
  }
  __device__ __forceinline__ void issue(Feed<KIND, GATEUP> &f, int d) const {
    const int s = f.step + d, off = s * 64;
    const bool any = f.item < plan.n_items && s < sp.s1, in = any && off + (lane & 3) * 16 < row_bytes;
    f.w[d][0] = in && f.row0 ? load_weights(f.p0 + off) : make_uint4(0, 0, 0, 0);
    f.w[d][1] = in && f.row1 ? load_weights(f.p1 + off) : make_uint4(0, 0, 0, 0);
    if constexpr (KIND == kE4) {
      f.sc[d][0] = any ? __ldg(f.q0 + (s >> 1)) : 0.f;
      f.sc[d][1] = any ? __ldg(f.q1 + (s >> 1)) : 0.f;
    }
  }
  __device__ __forceinline__ void next(Feed<KIND, GATEUP> &f) const {   // behind the issue of a whole block
    if (f.item >= plan.n_items) return;
    f.step += kDepth;
    if (f.step >= sp.s1) {
      f.step = sp.s0;
      f.tile += sp.groups;
      at_tile(f);
    }
  }

  // one step: eight rows' planes (of each GROUPS) times the two row tiles
  template <int GROUPS>
  __device__ __forceinline__ void step(const Feed<KIND, GATEUP> &f, int d, int s, const uint8_t *const (&rows)[2], int pitch, float (&acc)[2][2][4]) const {
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      const uint8_t *a = rows[q] + s * (128 / kElem);
      if constexpr (kElem == 2) {
        const uint4 h = *reinterpret_cast<const uint4 *>(a), l = *reinterpret_cast<const uint4 *>(a + pitch);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma<KIND>(acc[q][m], h.x, l.x, h.y, l.y, f.w[d][m].x, f.w[d][m].y);
          mma<KIND>(acc[q][m], h.z, l.z, h.w, l.w, f.w[d][m].z, f.w[d][m].w);
        }
      } else {
        const uint4 h0 = *reinterpret_cast<const uint4 *>(a), h1 = *reinterpret_cast<const uint4 *>(a + 16);
        const uint4 l0 = *reinterpret_cast<const uint4 *>(a + pitch), l1 = *reinterpret_cast<const uint4 *>(a + pitch + 16);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          float (&t)[4] = KIND == kE4 ? part : acc[q][m];
          uint32_t b0, b1;
          codes_f16<KIND>(f.w[d][m].x, b0, b1);
          mma<KIND>(t, h0.x, l0.x, h0.y, l0.y, b0, b1);
          codes_f16<KIND>(f.w[d][m].y, b0, b1);
          mma<KIND>(t, h0.z, l0.z, h0.w, l0.w, b0, b1);
          codes_f16<KIND>(f.w[d][m].z, b0, b1);
          mma<KIND>(t, h1.x, l1.x, h1.y, l1.y, b0, b1);
          codes_f16<KIND>(f.w[d][m].w, b0, b1);
          mma<KIND>(t, h1.z, l1.z, h1.w, l1.w, b0, b1);
          if constexpr (KIND == kE4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[q][m][i] = fmaf(f.sc[d][m], part[i], acc[q][m][i]);
          }
        }
      }
    }
  }
};

// slot `i` of an expert: the token of the i-th bit of its mask, and the pair
__device__ __forceinline__ int slot_token(unsigned mask, int i) {
  while (i-- > 0) mask &= mask - 1u;
  return __ffs(mask) - 1;
}
__device__ __forceinline__ int slot_pair(const Shared &s, int k, int e, int t) {
  int at = 0;
  for (int j = 1; j < k; ++j)
    if (s.sel_e[t][j] == e) at = j;
  return t * k + at;
}

// One product over this CTA's items: gate, up and silu into p.act, or down into p.Y. The first loads may be under way (`feed` started).
template <int KIND, bool GATEUP>
__device__ __forceinline__ void run_product(const DecodeParams &p, Shared &s, const Product<KIND, GATEUP> &pr, Feed<KIND, GATEUP> &feed, uint8_t *panel,
                                            float4 *red) {
  const int tid = threadIdx.x, lane = tid & 31;
  const Plan &plan = pr.plan;
  const int K = pr.K, pitch = Geo<KIND>::pitch(K), cap = Geo<KIND>::cap(K);
  const Split sp = pr.sp;
  int built = 0;   // items whose rows are in the panel
  for (int i = 0; i < plan.n_items; ++i) {
    const Item it = plan.item[i];
    if (i >= built) {
      // ---- the rows of this and the next items, as many as the panel takes ----
      int n = 0;
      for (built = i; built < plan.n_items && n + plan.item[built].n <= cap; ++built) n += plan.item[built].n;
      __syncthreads();   // the last panel and its powers are read
      if (!GATEUP && KIND != kBf16) {
        if (tid < kMaxTokens) s.row_max[tid] = 0u;
        __syncthreads();
      }
      auto row_of = [&](int r, int &e, int &slot) {
        int j = i;
        while (r >= plan.item[j].n) r -= plan.item[j++].n;
        e = plan.item[j].expert;
        slot = plan.item[j].first + r;
      };
      const int chunks = (K + 63) / 64 * 8;   // of eight values: whole steps
      if (!GATEUP && KIND != kBf16) {
        for (int r = 0; r < n; ++r) {
          int e, slot;
          row_of(r, e, slot);
          const float *src = p.act + (int64_t)slot_pair(s, p.k, e, slot_token(s.mask[e], slot)) * K;
          float m = 0.f;
          for (int c = tid; c < K / 4; c += kThreads) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(src) + c);
            m = max3_abs_nan(max3_abs_nan(m, v.x, v.y), v.z, v.w);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
          if (lane == 0) atomicMax(&s.row_max[r], __float_as_uint(m) & 0x7fffffffu);   // magnitudes order as their bits do, a NaN above all
        }
        __syncthreads();
      }
      for (int idx = tid; idx < n * chunks; idx += kThreads) {
        const int r = idx / chunks, c = idx - r * chunks;
        int e, slot;
        row_of(r, e, slot);
        const int t = slot_token(s.mask[e], slot);
        float v[8], mult = 1.f, unmult = 1.f;
        if (8 * c >= K) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.f;
        } else if (GATEUP) {
          load8(p.x, p.x_dtype, t * p.ldx + 8 * c, p.x_vec, v);
          if (p.pre_w) {
            float w[8];
            load8(p.pre_w, p.norm_dtype, 8 * c, true, w);
            const float inv = s.inv[t];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = v[j] * inv * w[j];
          }
        } else {
          const float4 *src = reinterpret_cast<const float4 *>(p.act + (int64_t)slot_pair(s, p.k, e, t) * K) + 2 * c;
          const float4 a = __ldcg(src), b = __ldcg(src + 1);
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
        if constexpr (KIND != kBf16) {
          if (GATEUP) {
            mult = s.mult[t];
            unmult = s.unmult[t];
          } else {
            row_power(__uint_as_float(s.row_max[r]), mult, unmult);
          }
        }
        uint4 hi, lo;
        planes2<KIND>(v[0] * mult, v[1] * mult, hi.x, lo.x);
        planes2<KIND>(v[2] * mult, v[3] * mult, hi.y, lo.y);
        planes2<KIND>(v[4] * mult, v[5] * mult, hi.z, lo.z);
        planes2<KIND>(v[6] * mult, v[7] * mult, hi.w, lo.w);
        uint8_t *dst = panel + (2 * r) * pitch + 16 * c;
        *reinterpret_cast<uint4 *>(dst) = hi;
        *reinterpret_cast<uint4 *>(dst + pitch) = lo;
        if (c == 0) s.row_unmult[r] = unmult;
      }
      __syncthreads();
    }
    // ---- the item's tiles ----
    int base = 0;
    for (int j = it.panel; j < i; ++j) base += plan.item[j].n;
    const int tiles = pr.tiles(it), rounds = (tiles + sp.groups - 1) / sp.groups, two = it.n > 8;
    const int batch = kRed / (kWarps * 512 * (1 + two));   // rounds whose sums fit
    const uint8_t *rows[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) rows[q] = panel + 2 * (base + min(8 * q + (lane >> 2), it.n - 1)) * pitch + (lane & 3) * (32 / pr.kElem);
    for (int round = 0; round < rounds; ++round) {
      const int in_batch = round % batch;
      if (sp.group < sp.groups && round * sp.groups + sp.group < tiles) {
        float acc[2][2][4];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[q][m][j] = 0.f;
        for (int st = sp.s0; st < sp.s1; st += kDepth) {
#pragma unroll
          for (int d = 0; d < kDepth; ++d) {
            if (st + d < sp.s1) {
              if (two) pr.template step<2>(feed, d, st + d, rows, pitch, acc);
              else pr.template step<1>(feed, d, st + d, rows, pitch, acc);
            }
            pr.issue(feed, d);
          }
          pr.next(feed);
        }
        float4 *dst = red + ((in_batch * (1 + two)) * kWarps + sp.group * sp.parts + sp.part) * 32 + lane;
        dst[0] = make_float4(acc[0][0][0] + acc[0][0][2], acc[0][0][1] + acc[0][0][3], acc[0][1][0] + acc[0][1][2], acc[0][1][1] + acc[0][1][3]);
        if (two)
          dst[kWarps * 32] = make_float4(acc[1][0][0] + acc[1][0][2], acc[1][0][1] + acc[1][0][3], acc[1][1][0] + acc[1][1][2], acc[1][1][1] + acc[1][1][3]);
      }
      if (in_batch != batch - 1 && round != rounds - 1) continue;
      __syncthreads();
      // ---- sums over the parts of K, in order ----
      const int first = (round - in_batch) * sp.groups, here = min(tiles - first, (in_batch + 1) * sp.groups);
      const int per = it.n * (GATEUP ? 8 : 16);   // outputs of a tile
      for (int o = tid; o < here * per; o += kThreads) {
        const int tile = o / per, rest = o - tile * per, tok = rest / (GATEUP ? 8 : 16), r = rest % (GATEUP ? 8 : 16);
        const int row = it.r0 + (first + tile) * Product<KIND, GATEUP>::kRows + r;
        if (row >= it.r1) continue;
        const int rd = tile / sp.groups, gr = tile - rd * sp.groups, q = tok >> 3;
        const float *src = reinterpret_cast<const float *>(red + ((rd * (1 + two) + q) * kWarps + gr * sp.parts) * 32 + (tok & 7) * 4 + ((r & 7) >> 1)) + (r & 1);
        float a = 0.f, b = 0.f;
        for (int part = 0; part < sp.parts; ++part) {
          a += src[part * 128 + (GATEUP ? 0 : (r >> 3) * 2)];
          if (GATEUP) b += src[part * 128 + 2];
        }
        const float un = KIND == kBf16 ? 1.0f : s.row_unmult[base + tok];
        a *= un;
        b *= un;
        const int t = slot_token(s.mask[it.expert], it.first + tok), pair = slot_pair(s, p.k, it.expert, t);
        if constexpr (KIND == kS8) {
          a *= __ldg((GATEUP ? p.s_gate : p.s_down) + (int64_t)it.expert * pr.N + row);
          if (GATEUP) b *= __ldg(p.s_up + (int64_t)it.expert * pr.N + row);
        }
        if (GATEUP) p.act[(int64_t)pair * pr.N + row] = a / (1.0f + expf(-a)) * b;
        else p.Y[(int64_t)pair * pr.N + row] = a;
      }
      __syncthreads();
    }
  }
}

// The rows of a product are dealt to the CTAs in equal numbers, in pairs of rows, over all active experts in a row; an expert's tokens
// that the panel does not take at once go through in passes.
__device__ void make_plan(Plan &plan, const Shared &s, int N, int cap) {
  const int64_t units = (int64_t)s.n_active * (N / 2);
  int64_t u = units * blockIdx.x / gridDim.x;
  const int64_t end = units * (blockIdx.x + 1) / gridDim.x;
  int n = 0, panel = 0, held = 0;
  while (u < end) {
    const int i = (int)(u / (N / 2)), e = s.active[i];
    const int64_t stop = min(end, (int64_t)(i + 1) * (N / 2));
    const int r0 = 2 * (int)(u - (int64_t)i * (N / 2)), r1 = r0 + 2 * (int)(stop - u), rows = __popc(s.mask[e]);
    for (int f = 0; f < rows && n < kMaxItems; f += cap) {
      const int c = min(cap, rows - f);
      if (held + c > cap) {
        panel = n;
        held = 0;
      }
      held += c;
      plan.item[n++] = Item{e, r0, r1, f, c, panel};
    }
    u = stop;
  }
  plan.n_items = n;
}

// Parts of K: those that take a warp the fewest steps, of which whole blocks of kDepth count; of equals the fewest parts.
__device__ __forceinline__ Split make_split(const Plan &plan, int rows_per_tile, int steps) {
  int tiles = 0;
  for (int i = 0; i < plan.n_items; ++i) tiles += (plan.item[i].r1 - plan.item[i].r0 + rows_per_tile - 1) / rows_per_tile;
  Split sp{};
  int best = 0x7fffffff;
  constexpr int kParts[7] = {1, 2, 3, 4, 5, 8, 16};
#pragma unroll
  for (int j = 0; j < 7; ++j) {
    const int parts = kParts[j], groups = kWarps / parts;
    const int cost = ((tiles + groups - 1) / groups) * (((steps + parts - 1) / parts + kDepth - 1) / kDepth);
    if (cost < best) {
      best = cost;
      sp.parts = parts;
      sp.groups = groups;
    }
  }
  const int warp = threadIdx.x >> 5;
  sp.group = warp / sp.parts;
  sp.part = warp - sp.group * sp.parts;
  sp.s0 = steps * sp.part / sp.parts;
  sp.s1 = steps * (sp.part + 1) / sp.parts;
  return sp;
}

// ---- stages 1 and 4 -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ float inverse_rms(float sum, int H, float eps) { return rsqrtf(fmaf(sum, 1.0f / (float)H, eps)); }

// Statistics of all tokens' rows and the logits of this CTA's experts. A token is shared by 16 / (T rounded up to a power of two) warps.
__device__ __forceinline__ void norms_and_logits(const DecodeParams &p, Shared &s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = p.T <= 1 ? 16 : p.T <= 2 ? 8 : p.T <= 4 ? 4 : p.T <= 8 ? 2 : 1;   // warps a token
  const int t = warp / per, w = warp - t * per, e0 = blockIdx.x, e1 = blockIdx.x + gridDim.x;
  float ss = 0.f, most = 0.f, d0 = 0.f, d1 = 0.f;
  if (t < p.T) {
    for (int c = w * 32 + lane; c < p.H / 8; c += per * 32) {
      float v[8], g[8];
      load8(p.x, p.x_dtype, t * p.ldx + 8 * c, p.x_vec, v);
      if (p.pre_w) load8(p.pre_w, p.norm_dtype, 8 * c, true, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = fmaf(v[j], v[j], ss);
        if (p.pre_w) v[j] *= g[j];
        most = max3_abs_nan(most, v[j], 0.f);
      }
      if (e0 < p.E) {
        load8(p.router, KNJ_DT_BF16, (int64_t)e0 * p.H + 8 * c, true, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) d0 = fmaf(v[j], g[j], d0);
      }
      if (e1 < p.E) {
        load8(p.router, KNJ_DT_BF16, (int64_t)e1 * p.H + 8 * c, true, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) d1 = fmaf(v[j], g[j], d1);
      }
    }
  }
  ss = warp_sum(ss);
  d0 = warp_sum(d0);
  d1 = warp_sum(d1);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lane == 0) {
    s.part[warp][0] = ss;
    s.part[warp][1] = most;
    s.part[warp][2] = d0;
    s.part[warp][3] = d1;
  }
  __syncthreads();
  if (warp < p.T) {   // a warp per token: a large row's squares are summed once more
    float tot = 0.f, m = 0.f, a = 0.f, b = 0.f;
    for (int i = 0; i < per; ++i) {
      tot += s.part[warp * per + i][0];
      m = max_nan(m, s.part[warp * per + i][1]);
      a += s.part[warp * per + i][2];
      b += s.part[warp * per + i][3];
    }
    float inv = 1.0f, down = 1.0f;
    if (p.pre_w) {
      if (tot > 3.402823466e38f) {   // squares of a large row left the range: from values * 2^-64, where eps does not count
        float q = 0.f;
        for (int c = lane; c < p.H; c += 32) {
          const float v = load_as_f32(p.x, p.x_dtype, warp * p.ldx + c) * kDown;
          q = fmaf(v, v, q);
        }
        inv = kDown * rsqrtf(warp_sum(q) * (1.0f / (float)p.H));
      } else {
        inv = inverse_rms(tot, p.H, p.eps);
      }
    }
    if (lane == 0) {
      s.inv[warp] = inv;
      row_power(m * inv, s.mult[warp], s.unmult[warp]);
      if (e0 < p.E) p.logits[warp * p.E + e0] = a * inv + (p.router_bias ? p.router_bias[e0] : 0.f);
      if (e1 < p.E) p.logits[warp * p.E + e1] = b * inv + (p.router_bias ? p.router_bias[e1] : 0.f);
    }
  }
}

__device__ __forceinline__ float gate_value(const DecodeParams &p, int t, int i) {
  if (p.gate_kind == KNJ_GATE_NONE) return 1.0f;
  const float g = load_as_f32(p.gate, p.gate_dtype, p.gate_kind == KNJ_GATE_CHANNEL ? i : p.gate_kind == KNJ_GATE_ROW ? t * p.ldg : t * p.ldg + i);
  return p.gate_sigmoid ? 1.0f / (1.0f + expf(-g)) : g;
}

// sum of squares of the row in shared memory and its inverse norm; a large row once more
__device__ __forceinline__ float row_inverse(const float *row, int H, float ss, float eps, float (*red)[kWarps]) {
  const float tot = cta_sum(ss, red[0]);
  if (!(tot > 3.402823466e38f)) return inverse_rms(tot, H, eps);
  float q = 0.f;
  for (int i = threadIdx.x; i < H; i += kThreads) q = fmaf(row[i] * kDown, row[i] * kDown, q);
  return kDown * rsqrtf(cta_sum(q, red[1]) * (1.0f / (float)H));
}

// One token's row: the pairs' rows in ascending order of their experts, then what stands behind the block.
__device__ __forceinline__ void finish_row(const DecodeParams &p, Shared &s, int t, float *row) {
  const int tid = threadIdx.x, H = p.H;
  int order[kMaxK];
  float weight[kMaxK];
#pragma unroll
  for (int i = 0; i < kMaxK; ++i) order[i] = 0, weight[i] = 0.f;
  for (int j = 0; j < p.k; ++j) {
    int rank = 0;
    for (int i = 0; i < p.k; ++i) rank += s.sel_e[t][i] < s.sel_e[t][j];
#pragma unroll
    for (int i = 0; i < kMaxK; ++i)
      if (i == rank) order[i] = j, weight[i] = s.sel_w[t][j];
  }
  float ss = 0.f;
  for (int i = tid; i < H; i += kThreads) {
    float y = 0.f, v[kMaxK];
#pragma unroll
    for (int j = 0; j < kMaxK; ++j) v[j] = j < p.k ? __ldcg(p.Y + ((int64_t)t * p.k + order[j]) * H + i) : 0.f;
#pragma unroll
    for (int j = 0; j < kMaxK; ++j)
      if (j < p.k) y = __fadd_rn(y, __fmul_rn(weight[j], v[j]));
    row[i] = y;
    ss = fmaf(y, y, ss);
  }
  float inv = 1.0f;
  if (p.post_w) inv = row_inverse(row, H, ss, p.eps, s.red);
  __syncthreads();
  ss = 0.f;
  for (int i = tid; i < H; i += kThreads) {
    float n = row[i];
    if (p.post_w) n = n * inv * load_as_f32(p.post_w, p.norm_dtype, i);
    const float v = p.beta * load_as_f32(p.x, p.x_dtype, t * p.ldx + i) + p.alpha * gate_value(p, t, i) * n;
    row[i] = v;
    ss = fmaf(v, v, ss);
    store_from_f32(p.out, p.out_dtype, t * p.ldo + i, v);
  }
  if (!p.next_w) return;
  inv = row_inverse(row, H, ss, p.eps, s.red);
  __syncthreads();
  if (p.h_dtype != KNJ_DT_E4M3) {
    for (int i = tid; i < H; i += kThreads) store_from_f32(p.h_next, p.h_dtype, t * p.ldh + i, row[i] * inv * load_as_f32(p.next_w, p.norm_dtype, i));
    return;
  }
  const int lane = tid & 31, groups = H / kFp8Group;
  for (int g = tid >> 5; g < groups; g += kWarps) {
    float v[4], most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kFp8Group + 32 * j + lane;
      v[j] = row[i] * inv * load_as_f32(p.next_w, p.norm_dtype, i);
      most = max3_abs_nan(most, v[j], 0.f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    const Fp8Scale sc = fp8_scale(most);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      static_cast<uint8_t *>(p.h_next)[t * p.ldh + g * kFp8Group + 32 * j + lane] = (uint8_t)e4m3_pair(v[j] * sc.inverse, 0.f);
    if (lane == 0) p.h_next_scale[(int64_t)t * groups + g] = sc.scale;
  }
}

// a wait gave up: NaN in the rows that this CTA would have written
__device__ void give_up(const DecodeParams &p) {
  const float nan = __int_as_float(0x7fffffff);
  for (int t = blockIdx.x; t < p.T; t += gridDim.x) {
    for (int i = threadIdx.x; i < p.H; i += kThreads) {
      store_from_f32(p.out, p.out_dtype, t * p.ldo + i, nan);
      if (p.next_w) {
        if (p.h_dtype == KNJ_DT_E4M3) static_cast<uint8_t *>(p.h_next)[t * p.ldh + i] = 0x7f;
        else store_from_f32(p.h_next, p.h_dtype, t * p.ldh + i, nan);
      }
    }
    if (p.next_w && p.h_dtype == KNJ_DT_E4M3)
      for (int g = threadIdx.x; g < p.H / kFp8Group; g += kThreads) p.h_next_scale[(int64_t)t * (p.H / kFp8Group) + g] = nan;
  }
}

template <int KIND>
__global__ void __launch_bounds__(kThreads, 1) moe_decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *panel = smem;
  float4 *red = reinterpret_cast<float4 *>(smem + kPanel);
  __shared__ Shared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (blockIdx.x == 0 && tid == 0) *p.status = 0;   // in front of the first barrier, behind which alone it is raised
  norms_and_logits(p, s);
  for (int e = tid; e < kMaxExperts; e += kThreads) s.mask[e] = 0u;
  if (!grid_barrier(p, s, 1)) return give_up(p);

  // ---- routing: a warp per token ----
  if (warp < p.T) {
    int e;
    float w;
    warp_topk(p.logits + warp * p.E, p.E, p.k, lane, e, w);
    if (lane < p.k) {
      s.sel_e[warp][lane] = e;
      s.sel_w[warp][lane] = w;
      atomicOr(&s.mask[e], 1u << warp);
      if (blockIdx.x == 0 && p.tap_exp) p.tap_exp[warp * p.k + lane] = e;
      if (blockIdx.x == 0 && p.tap_w) p.tap_w[warp * p.k + lane] = w;
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int b = 0; b < kMaxExperts; b += 32) {
      const bool on = s.mask[b + lane] != 0u;
      const unsigned all = __ballot_sync(0xffffffffu, on);
      if (on) s.active[n + __popc(all & ((1u << lane) - 1u))] = b + lane;
      n += __popc(all);
    }
    if (lane == 0) s.n_active = n;
    __syncwarp();
    if (lane < 2) make_plan(s.plan[lane], s, lane == 0 ? p.F : p.H, Geo<KIND>::cap(lane == 0 ? p.H : p.F));
  }
  __syncthreads();

  constexpr int kElem = Geo<KIND>::kElem;
  Product<KIND, true> up{p, s.plan[0], make_split(s.plan[0], 8, (p.H * kElem + 63) / 64), p.H, p.F, p.H * kElem, lane};
  Feed<KIND, true> feed_up;
  up.start(feed_up);
  run_product<KIND, true>(p, s, up, feed_up, panel, red);
  Product<KIND, false> down{p, s.plan[1], make_split(s.plan[1], 16, (p.F * kElem + 63) / 64), p.F, p.H, p.F * kElem, lane};
  Feed<KIND, false> feed_down;
  down.start(feed_down);   // the first weights of the down matrices travel while the grid meets
  if (!grid_barrier(p, s, 2)) return give_up(p);
  run_product<KIND, false>(p, s, down, feed_down, panel, red);
  if (!grid_barrier(p, s, 3)) return give_up(p);
  for (int t = blockIdx.x; t < p.T; t += gridDim.x) finish_row(p, s, t, reinterpret_cast<float *>(panel));
}

template <int KIND>
int launch(DecodeParams &p, cudaStream_t st) {
  constexpr int kSmem = kPanel + kRed;
  int dev = 0;
  KNJ_CUDA(cudaGetDevice(&dev));
  auto kern = moe_decode_kernel<KIND>;
  static bool opted[64] = {false};
  if (dev >= 0 && dev < 64 && !opted[dev]) {
    KNJ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    opted[dev] = true;
  }
  KNJ_CUDA(cudaMemsetAsync(p.sync, 0, 8, st));
  void *args[] = {&p};
  KNJ_CUDA(cudaLaunchCooperativeKernel(reinterpret_cast<const void *>(kern), dim3(sm_count()), dim3(kThreads), args, kSmem, st));
  return launch_status("moe_decode_kernel");
}

}  // namespace

namespace knj {
size_t moe_decode_workspace(int T, int H, int F, int E, int k) {
  auto up256 = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const size_t P = (size_t)T * k;
  return 256 + up256((size_t)T * E * 4) + up256(P * F * 4) + up256(P * H * 4);
}

int moe_decode_launch(const knj_moe_block_args *a, int32_t *status, knj_stream_t stream) {
  auto up256 = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const int T = a->n_tokens, H = a->hidden, F = a->ffn, E = a->n_experts, k = a->top_k;
  KNJ_REQUIRE(T <= kMaxTokens, "knj_moe_block_decode: %d tokens, at most %d", T, kMaxTokens);
  KNJ_REQUIRE(F <= KNJ_MOE_DECODE_MAX_FFN, "knj_moe_block_decode: ffn=%d above %d", F, KNJ_MOE_DECODE_MAX_FFN);
  KNJ_REQUIRE(sm_count() >= kMaxExperts / 2, "knj_moe_block_decode: a device of %d SMs or more needed", kMaxExperts / 2);
  KNJ_REQUIRE(aligned16(a->pre_w), "knj_moe_block_decode: pre_w must be 16-byte aligned");
  DecodeParams p{};
  p.x = a->x; p.pre_w = a->pre_w; p.post_w = a->post_w; p.next_w = a->next_w; p.gate = a->gate; p.router = a->w_router; p.router_bias = a->router_bias;
  p.w_gate = static_cast<const uint8_t *>(a->w_gate); p.w_up = static_cast<const uint8_t *>(a->w_up); p.w_down = static_cast<const uint8_t *>(a->w_down);
  p.s_gate = a->gate_scale; p.s_up = a->up_scale; p.s_down = a->down_scale; p.out = a->out; p.h_next = a->h_next; p.h_next_scale = a->h_next_scale;
  p.tap_exp = a->tap_pair_exp; p.tap_w = a->tap_pair_w;
  uint8_t *ws = static_cast<uint8_t *>(a->workspace);
  p.sync = reinterpret_cast<unsigned *>(ws + 128);   // behind the status word of the whole block
  ws += 256;
  p.logits = reinterpret_cast<float *>(ws);
  ws += up256((size_t)T * E * 4);
  p.act = reinterpret_cast<float *>(ws);
  ws += up256((size_t)T * k * F * 4);
  p.Y = reinterpret_cast<float *>(ws);
  p.status = status; p.ldx = a->ldx; p.ldo = a->ldo; p.ldg = a->ldg; p.ldh = a->ld_h_next;
  p.T = T; p.H = H; p.F = F; p.E = E; p.k = k;
  p.x_dtype = a->x_dtype; p.out_dtype = a->out_dtype; p.norm_dtype = a->w_norm_dtype; p.gate_dtype = a->gate_dtype; p.h_dtype = a->h_next_dtype;
  p.gate_kind = a->gate_kind; p.gate_sigmoid = a->gate_sigmoid;
  p.x_vec = aligned16(a->x) && a->ldx * (a->x_dtype == KNJ_DT_F32 ? 4 : 2) % 16 == 0;
  p.alpha = a->alpha; p.beta = a->beta; p.eps = a->eps;
  p.wait_cycles = decode_wait_cycles(); p.stall = t_stall;
  const cudaStream_t st = as_stream(stream);
  switch (a->w_dtype) {
    case KNJ_DT_BF16: return launch<kBf16>(p, st);
    case KNJ_DT_F16: return launch<kF16>(p, st);
    case KNJ_DT_E4M3: return launch<kE4>(p, st);
    default: return launch<kS8>(p, st);
  }
}
}  // namespace knj

extern "C" void knj_moe_block_decode_test_stall(int barrier) { t_stall = barrier >= 1 && barrier <= 3 ? barrier : 0; }
