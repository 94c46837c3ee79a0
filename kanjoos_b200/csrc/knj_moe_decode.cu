// knj_moe_decode.cu -- a whole MoE block of a residual stream for up to sixteen tokens in two kernels, experts in bf16,
// fp16, e4m3 (one scale for each block of 128 x 128) or int8 (one for each output channel):
//   h   = norm(x; pre_w)
//   y   = sum over the top_k experts of softmax weight * down(silu(gate(h)) * up(h))
//   out = beta * x + alpha * g * norm(y; post_w),   h_next = norm(out; next_w)
// What is computed between x and out stays in f32, and so does what the matrices are multiplied with: a row of f32 values goes to the
// tensor core as 16-bit planes, each the rounded rest that the ones in front of it leave. bf16 experts meet three bf16 planes, which hold
// all 24 bits of a value; the others two fp16 planes under a power of two for each row, which hold 22 (their codes are exact in fp16). In
// mma.sync.m16n8k16 sixteen matrix rows meet the eight planes of two (two planes: four) tokens, or eight rows the sixteen of five (eight),
// so that further planes cost little while weights are on their way. (Two planes in bf16, 17 bits, left the block's part off by 4e-6 of its
// norm, which an f32 stream shows. us with two planes and three: 128 experts of 2048 x 768, 1, 4, 16 tokens 32, 64, 145 and 33.5, 66, 148; 32
// of 1024 x 512, 16 tokens 36 and 40; 8 of 8192 x 2048, top 2, 16 tokens, whose planes take twice the passes, 319 and 376.) Rows so long
// that three planes of one leave the ring less than two slots, above 22656 values, stay with two.
//
// Bound by the bytes of the experts that the tokens use, each read once: one token, 8 experts of 2048 x 768 in bf16, 75.5 MB. A warp of
// its own streams this CTA's matrix rows, of gate and up and behind them of down, through a ring in shared memory; sixteen warps
// multiply. So the down matrices are on their way while other SMs are still at gate and up, and the ring's 130 KB and more keep HBM
// busy. A lane takes its weights as 16 bytes of a row, which are MMA fragments as they lie: the order of K is free as long as both operands
// have the same. tcgen05 gives nothing here: the tensor work of a token is a fiftieth of the time.
//
// The first kernel forms norm statistics and router logits. The second, cooperative, has a CTA for each SM:
//   1  top-k (every CTA for itself); gate, up, silu: every CTA has matrix rows of the same cost, of all active experts in a row
//   2  down, likewise, as soon as gate and up of the CTA's own experts are done everywhere (a count of rows for each expert; a barrier over
//      the grid in its place waits for the slowest SM of all: 16 tokens bf16 150 us, so 146, int8 4 tokens 53.6, so 52.2)
//   3  behind a barrier over the grid: weighted sum, norm, gate, residual, next norm, a CTA for each token
// (The first stage inside the cooperative kernel needed one barrier more and a fill that cleared its counter in front of the launch.)
// A block of 128 experts of 2048 x 768, top 8, takes 33.5 us for one token in bf16 and 148 for sixteen (5.2 TB/s over both kernels), in a graph.
// Every wait is bounded (knj_decode_wait_limit): on give-up the status word is raised and the outputs are NaN.
#include <type_traits>

#include "knj_fp8.cuh"

using namespace knj;

namespace {

constexpr int kMaxRows = 8;   // of activations that go through a matrix row at a time
constexpr int kMaxTokens = KNJ_MOE_DECODE_MAX_TOKENS, kMaxK = 8, kMaxExperts = 256;
// Seventeen warps leave 96 registers a thread, and the shared memory that the ring takes leaves no L1 for what does not fit: a spilled word
// comes back from L2, 1000 cycles under load. So the products' loops are kept small: forms with the planes of the tokens in registers
// spilled, and took three times as long.
constexpr int kThreads = 512, kWarps = kThreads / 32;   // that multiply; behind them the warp that copies
constexpr int kAll = kThreads + 32;
// A slot of the ring holds a tile: 64, 32, 16 or 8 matrix rows of up to 512, 1024, 2048 or 4096 bytes as they lie, in one or two copies.
// (A copy for each row passes the copy unit in some 100 cycles whatever its length: 768 bytes a row took as long as 1536, and rows of
// 2048 bytes more than HBM needs to bring them.) Longer rows come in slices of up to 4096 bytes, eight rows to a slot.
constexpr int kSlice = 4096;
constexpr int kSlot = 8 * kSlice;
constexpr int kMaxSlots = 6;
constexpr int kRed = 16 * 1024;                // bytes of the sums of a batch of tiles, 256 or 512 a tile and token
constexpr int kSmem = 213 * 1024;              // sums, planes of the rows in use, and the ring in what they leave
// int8: the scales of a slot's rows, up to 32 of gate and of up or 64 of down, in whole 16-byte units
constexpr int kScales = 80;
constexpr int kMaxItems = 64;
constexpr size_t kSyncAt = 128, kMaxAt = 256, kStatsAt = kMaxAt + kMaxTokens * kMaxK * 4,
                 kReadyAt = kStatsAt + 256, kHead = kReadyAt + kMaxExperts * 4;   // of the workspace
constexpr float kDown = 0x1p-80f;   // of rows whose squares leave the range: those of 2^128 and their sum are in it then, those of the smallest such row (2^56) too

enum Kind { kBf16 = 0, kBf16Many = 1, kF16 = 2, kE4 = 3, kS8 = 4 };   // kBf16Many: see launch_bf16

// Of a product: its rows in memory, and how they are cut
struct Shape {
  int K, N, row_bytes;
  int slices, slice;   // of a row, bytes
  int eight;           // tiles of eight rows, else sub-tiles of sixteen
  int subs;            // sub-tiles of a tile, among which a group's warps are split
  int planes;          // of a row of activations
  int outs;            // outputs of a tile: its matrix rows, of which of gate and up the first half is gate's
};

struct DecodeParams {
  Shape shape[2];      // gate and up, down
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
  unsigned *sync;               // [0] arrivals, [1] raised by a wait that gave up; cleared by the first kernel
  float2 *stats;                // [tokens] inverse norm, largest magnitude of the normalised row
  unsigned *ready;              // [experts] matrix rows of gate and up whose outputs are written; cleared by the first kernel
  unsigned *row_max;            // [pairs] bits of the largest magnitude of an activation row; cleared by the first kernel
  int32_t *status;
  int64_t ldx, ldo, ldg, ldh;
  int T, H, F, E, k;
  int x_dtype, out_dtype, norm_dtype, gate_dtype, h_dtype, gate_kind, gate_sigmoid;
  unsigned grid_inverse;        // 2^32 / CTAs, rounded down
  int x_vec;                    // rows of x are whole 16-byte units
  float alpha, beta, eps;
  long long wait_cycles;
  int stall;                    // test hook: 1 = no expert's rows are ever ready, 2 = the barrier's target is out of reach, 3 = plans have room for one item
};
thread_local int t_stall = 0;

// a run of matrix rows of one expert, and the rows of activations that go through them: `n` of them from the expert's slot `first` on
struct Item {
  int expert, r0, r1, first, n, panel;
};
struct Plan {
  Item item[kMaxItems];
  int n_items, rows;            // rows: most that are in the panel at a time
};

struct Shared {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  int fail;                     // raised by a wait that gave up; read as volatile
  float inv[kMaxTokens], mult[kMaxTokens], unmult[kMaxTokens];
  int sel_e[kMaxTokens][kMaxK];
  float sel_w[kMaxTokens][kMaxK];
  int order[kMaxTokens][kMaxK];   // a token's choices by ascending expert
  unsigned mask[kMaxExperts];
  uint8_t pair_at[kMaxExperts][kMaxTokens];   // pairs of an expert's tokens in ascending order
  int active[kMaxTokens * kMaxK];
  unsigned cost[kMaxTokens * kMaxK + 1];   // of the active experts in front
  int n_active, ok;
  Plan plan[2];                 // gate and up, down
  int row_tok[kMaxTokens], row_pair[kMaxTokens];        // of the panel's rows
  float row_mult[kMaxTokens], row_unmult[kMaxTokens];
  float red[4][kWarps];
  alignas(16) float scale[kMaxSlots][kScales];   // int8: of a slot's rows
};

static_assert(kSmem + sizeof(Shared) <= 227 * 1024, "shared memory of a block");

// ---- small pieces -------------------------------------------------------------------------------------------------------

__device__ __forceinline__ unsigned ld_acquire(const unsigned *p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// of the warps that multiply
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }
// Waits of thread 0 (of an expert's rows: of any thread) for a word that other CTAs add to: false where it did not come to `target` in time.
__device__ __forceinline__ bool reaches(const DecodeParams &p, const Shared &s, const unsigned *word, unsigned target) {
  const long long t0 = clock64();
  while (ld_acquire(word) < target)
    if (*reinterpret_cast<const volatile int *>(&s.fail) != 0 || ld_acquire(p.sync + 1) != 0u || clock64() - t0 > p.wait_cycles) return false;
  return true;
}
__device__ __forceinline__ void add_release(unsigned *word, unsigned n) { asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(word), "r"(n) : "memory"); }
// Barrier over the grid, in two halves, met by the warps that multiply. A CTA in which a wait has given up never arrives; grid_wait is
// false for all threads where the barrier did not complete in time.
__device__ __forceinline__ void grid_arrive(const DecodeParams &p, Shared &s) {
  meet();
  if (threadIdx.x == 0 && *reinterpret_cast<volatile int *>(&s.fail) == 0) add_release(p.sync, 1u);
}
__device__ __forceinline__ bool grid_wait(const DecodeParams &p, Shared &s) {
  if (threadIdx.x == 0) s.ok = *reinterpret_cast<volatile int *>(&s.fail) == 0 && reaches(p, s, p.sync, gridDim.x + (p.stall == 2 ? 1u : 0u));
  meet();
  return s.ok != 0;
}

// eight consecutive values of a row as they lie in memory, at a 16-byte boundary: without branches, so that many loads go out together
struct Raw8 {
  uint4 a, b;
};
__device__ __forceinline__ Raw8 load_raw8(const void *base, int dtype, int64_t i) {
  Raw8 r;
  const bool wide = dtype == KNJ_DT_F32;
  const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(base) + i * (wide ? 4 : 2));
  r.a = q[0];
  r.b = r.a;
  if (wide) r.b = q[1];
  return r;
}
__device__ __forceinline__ void values8(const Raw8 &r, int dtype, float (&v)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dtype == KNJ_DT_BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  } else if (dtype == KNJ_DT_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
      v[2 * j] = h.x;
      v[2 * j + 1] = h.y;
    }
  }
}
// the same of a row at any address
__device__ __forceinline__ void load8(const void *base, int dtype, int64_t i, bool vec, float (&v)[8]) {
  if (vec) {
    values8(load_raw8(base, dtype, i), dtype, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = load_as_f32(base, dtype, i + j);
  }
}

// The power of two under which a row with largest magnitude m goes into fp16 planes: m comes to 2^14 .. 2^15, so that the low plane of a
// value keeps its bits down to 2^-40 of m. (m of 0, infinity or NaN: any will do.)
__device__ __forceinline__ void row_power(float m, float &mult, float &unmult) {
  const int e = max((int)(__float_as_uint(m) >> 23 & 255u) - 127, -100);
  mult = __uint_as_float((uint32_t)(14 - e + 127) << 23);
  unmult = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
}

// a plane of two values, in which what it leaves out stays
template <int KIND>
__device__ __forceinline__ uint32_t plane2(float &a, float &b) {
  uint32_t bits;
  float2 f;
  if constexpr (KIND <= kBf16Many) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    f = __bfloat1622float2(h);
    bits = *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    f = __half22float2(h);
    bits = *reinterpret_cast<const uint32_t *>(&h);
  }
  a -= f.x;
  b -= f.y;
  return bits;
}

template <int KIND>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (KIND <= kBf16Many)
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

__device__ __forceinline__ float cta_sum(float v, float *red) {   // by all threads; red: a word for each warp, not in use by an earlier sum
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  meet();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) t += red[i];
  return t;
}

template <int KIND>
struct Geo {
  static constexpr int kElem = KIND <= kF16 ? 2 : 1;
  // Groups of warps that take the tiles in turn, and warps of one: so that a warp has about four runs of a slot, of rows of 2048 x 2 bytes eight.
  // (Of 4 and 2 groups, us: bf16 1 token 31.8, 33.4, 4 tokens 64.5, 67.4, 16 tokens 147, 150; e4m3 5 tokens 62.8, 59.8; int8 8 tokens 78.5,
  // 77.0, 16 tokens 107, 109.)
  static constexpr int kGroups = KIND <= kF16 ? 4 : 2, kTeam = kWarps / kGroups;
  // bytes of a plane of K values: whole runs of 128 bytes of weights, and rows an odd 64 (of codes: 16) bytes apart, for the banks as in the ring
  __host__ __device__ static int pitch(int K) { return (K * kElem + 127) / 128 * (256 / kElem) + (kElem == 2 ? 64 : 16); }
  __host__ __device__ static int planes(int K) { return KIND <= kBf16Many && 3 * pitch(K) <= kSmem - kRed - 2 * kSlot ? 3 : 2; }
  // Most rows of a pass. bf16: the planes of five are the sixteen rows or columns of two MMAs. (A form of up to eight besides, us: tiles of eight
  // rows, 1 token 35.9, so 33.6, 16 tokens 157, so 148; tiles of sixteen, 1 token 34.1, 16 tokens 151.)
  static constexpr int kMost = KIND == kBf16 ? 5 : kMaxRows;
  // rows of a pass: what leaves the ring two slots, or one
  __host__ __device__ static int pass(int K) {
    const int c = (kSmem - kRed - 2 * kSlot) / (planes(K) * pitch(K));
    return c < 1 ? 1 : c < kMost ? c : kMost;
  }
  // Rows in the panel at a time: what leaves it four slots, or those of a pass. (bf16: a pass of more rows is alone there.)
  __host__ __device__ static int cap(int K) {
    const int c = (kSmem - kRed - 4 * kSlot) / (planes(K) * pitch(K));
    if (KIND > kBf16Many && c < pass(K)) return pass(K);
    return c < 1 ? 1 : c < kMaxTokens ? c : kMaxTokens;
  }
};

// ---- products -----------------------------------------------------------------------------------------------------------

// place in the ring
struct Ring {
  int at, n;
  uint32_t parity;
  __device__ __forceinline__ void next() {
    if (++at == n) {
      at = 0;
      parity ^= 1u;
    }
  }
};

// The copying warp's side of a product. False after a wait that gave up.
template <int KIND>
__device__ __forceinline__ bool feed(const DecodeParams &p, Shared &s, int product, Ring &ring, uint8_t *slots, int &copied) {
  const int lane = threadIdx.x & 31;
  const Shape &sh = p.shape[product];
  const Plan &plan = s.plan[product];
  const bool up = product == 0, whole = sh.slices == 1;
  for (int i = 0; i < plan.n_items; ++i) {
    const Item it = plan.item[i];
    for (int first = it.r0; first < it.r1; first += sh.outs) {
      const int rows = min(sh.outs, it.r1 - first);
      // lane l copies the rows of matrix l, or row l % rows of matrix l / rows
      const int second = up && (whole ? lane == 1 : lane >= rows), r = whole ? 0 : lane - second * rows;
      const bool mine = lane < (whole ? 1 : rows) * (up ? 2 : 1);
      const uint8_t *src = (up ? (second ? p.w_up : p.w_gate) : p.w_down) + ((int64_t)it.expert * sh.N + first + r) * sh.row_bytes;
      const int dst = (second * sh.outs + r) * sh.slice;
      // int8: the rows' scales, in units of four (N is a multiple of 16), come with the first slice (a read past L1 ahead of each tile: one token 30.3 us, so 29.6)
      const int scale0 = first & ~3, scale_bytes = KIND == kS8 ? (((first + rows + 3) & ~3) - scale0) * 4 : 0;
      for (int sl = 0; sl < sh.slices; ++sl) {
        const int bytes = whole ? rows * sh.row_bytes : min(sh.slice, sh.row_bytes - sl * sh.slice);
        const bool ok = mbar_wait_for(&s.empty[ring.at], ring.parity ^ 1u, p.wait_cycles, &s.fail);
        if (!__all_sync(0xffffffffu, ok)) return false;
        if (lane == 0) mbar_expect_tx(&s.full[ring.at], (uint32_t)((bytes * (whole ? 1 : rows) + (sl == 0 ? scale_bytes : 0)) * (up ? 2 : 1)));
        __syncwarp();
        if (mine) bulk_g2s(slots + ring.at * kSlot + dst, src + sl * sh.slice, (uint32_t)bytes, &s.full[ring.at]);
        if (KIND == kS8 && sl == 0 && lane >= (up ? 30 : 31))
          bulk_g2s(&s.scale[ring.at][lane == 30 ? kScales / 2 : 0], (up ? (lane == 30 ? p.s_up : p.s_gate) : p.s_down) + (int64_t)it.expert * sh.N + scale0,
                   (uint32_t)scale_bytes, &s.full[ring.at]);
        ring.next();
        ++copied;
      }
    }
  }
  return true;
}

// A lane's part of a run of 128 bytes (two steps of 64) of sixteen rows: of rows g and g + 8 the bytes 16 j .. + 15 of either step. (Rows a
// multiple of 128 bytes apart lie on the same banks, and such a load takes two turns. SWAP: odd rows read their second step first, and the
// two change places in registers. Of bf16 and fp16 experts that pays, 16 tokens 162 -> 155 us; of codes the instructions are dearer.)
// left: bytes of the rows from the run's first on; what lies behind is zero.
template <int ROWS>   // two, or of tiles of eight rows one
struct Weights {
  uint4 w[2][ROWS];   // [step][row]
  template <bool SWAP>
  __device__ __forceinline__ void load(const uint8_t *row0, const uint8_t *row1, bool odd, int left) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const uint8_t *row = r == 0 ? row0 : row1;
      const int first = SWAP && odd ? 64 : 0;
      const uint4 a = *reinterpret_cast<const uint4 *>(row + first), b = *reinterpret_cast<const uint4 *>(row + 64 - first);
      w[0][r] = SWAP && odd ? b : a;
      w[1][r] = SWAP && odd ? a : b;
    }
    if (left < 128) {
      const int at = (threadIdx.x & 3) * 16;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (u * 64 + at >= left) w[u][0] = w[u][ROWS - 1] = make_uint4(0, 0, 0, 0);
    }
  }
};
// a lane's run of a plane for a step
template <int KIND>
struct Acts {
  uint4 b[KIND <= kF16 ? 1 : 2];
  __device__ __forceinline__ void load(const uint8_t *at) {
    b[0] = *reinterpret_cast<const uint4 *>(at);
    if constexpr (KIND > kF16) b[1] = *reinterpret_cast<const uint4 *>(at + 16);
  }
};
// One step of sixteen rows times SETS sets of eight planes, in the order that run_product gives them
template <int KIND, int SETS>
__device__ __forceinline__ void step(const uint4 (&w)[2], const uint8_t *x0, const uint8_t *x1, const uint8_t *x2, float (&acc0)[4], float (&acc1)[4],
                                     float (&acc2)[4]) {
  constexpr bool TWO = SETS >= 2;
  if constexpr (SETS == 3) step<KIND, 1>(w, x2, x2, x2, acc2, acc2, acc2);
  Acts<KIND> a, b;
  a.load(x0);
  if constexpr (TWO) b.load(x1);
  if constexpr (KIND <= kF16) {
    mma<KIND>(acc0, w[0].x, w[1].x, w[0].y, w[1].y, a.b[0].x, a.b[0].y);
    if constexpr (TWO) mma<KIND>(acc1, w[0].x, w[1].x, w[0].y, w[1].y, b.b[0].x, b.b[0].y);
    mma<KIND>(acc0, w[0].z, w[1].z, w[0].w, w[1].w, a.b[0].z, a.b[0].w);
    if constexpr (TWO) mma<KIND>(acc1, w[0].z, w[1].z, w[0].w, w[1].w, b.b[0].z, b.b[0].w);
  } else {
    const uint32_t r0[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, r1[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t c[4];
      codes_f16<KIND>(r0[i], c[0], c[2]);
      codes_f16<KIND>(r1[i], c[1], c[3]);
      const uint4 &p = a.b[i >> 1];
      mma<KIND>(acc0, c[0], c[1], c[2], c[3], i & 1 ? p.z : p.x, i & 1 ? p.w : p.y);
      if constexpr (TWO) {
        const uint4 &q = b.b[i >> 1];
        mma<KIND>(acc1, c[0], c[1], c[2], c[3], i & 1 ? q.z : q.x, i & 1 ? q.w : q.y);
      }
    }
  }
}

// One step of eight rows times sixteen planes, which are the MMA's rows here
template <int KIND>
__device__ __forceinline__ void step(const uint4 (&w)[1], const uint8_t *x0, const uint8_t *x1, float (&acc)[4]) {
  Acts<KIND> h, l;
  h.load(x0);
  l.load(x1);
  if constexpr (KIND <= kF16) {
    mma<KIND>(acc, h.b[0].x, l.b[0].x, h.b[0].y, l.b[0].y, w[0].x, w[0].y);
    mma<KIND>(acc, h.b[0].z, l.b[0].z, h.b[0].w, l.b[0].w, w[0].z, w[0].w);
  } else {
    const uint32_t r[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t b0, b1;
      codes_f16<KIND>(r[i], b0, b1);
      const uint4 &p = h.b[i >> 1], &q = l.b[i >> 1];
      mma<KIND>(acc, i & 1 ? p.z : p.x, i & 1 ? q.z : q.x, i & 1 ? p.w : p.y, i & 1 ? q.w : q.y, b0, b1);
    }
  }
}

// The rows of items i .. in the panel, as many as it takes: their planes, zeros behind K up to whole runs. Returns the item behind them.
template <int KIND, bool GATEUP>
__device__ __forceinline__ int build_panel(const DecodeParams &p, Shared &s, const Plan &plan, int K, uint8_t *panel, int i) {
  const int tid = threadIdx.x, pitch = Geo<KIND>::pitch(K), planes = Geo<KIND>::planes(K);
  int n = 0, built = i;
  for (; built < plan.n_items && plan.item[built].panel == i; ++built) n += plan.item[built].n;
  if (!GATEUP) {   // the experts' rows of activations, from the CTAs that gate and up were dealt to
    if (tid < built - i) {
      const int e = plan.item[i + tid].expert, pass = Geo<KIND>::pass(p.H);
      const unsigned whole = (unsigned)p.F * ((__popc(s.mask[e]) + pass - 1) / pass);
      if (!reaches(p, s, p.ready + e, whole + (p.stall == 1 ? 1u : 0u))) *reinterpret_cast<volatile int *>(&s.fail) = 1;
    }
    meet();
  }
  if (tid < n) {
    int r = tid, j = i;
    while (r >= plan.item[j].n) r -= plan.item[j++].n;
    const int pair = s.pair_at[plan.item[j].expert][plan.item[j].first + r], t = pair / p.k;
    s.row_tok[tid] = t;
    s.row_pair[tid] = pair;
    if constexpr (KIND > kBf16Many) {
      if (GATEUP) {
        s.row_mult[tid] = s.mult[t];
        s.row_unmult[tid] = s.unmult[t];
      } else {
        row_power(__uint_as_float(__ldcg(p.row_max + pair)), s.row_mult[tid], s.row_unmult[tid]);
      }
    }
  }
  meet();
  // of eight values, up to the end of a run of 128 bytes of weights; and of 32 such: a warp's
  constexpr int kRun = 128 / Geo<KIND>::kElem;
  const int chunks = (K + kRun - 1) / kRun * (kRun / 8), runs = (chunks + 31) / 32;
#pragma unroll 2
  for (int u = tid >> 5; u < n * runs; u += kWarps) {
    const int r = u / runs, c = (u - r * runs) * 32 + (tid & 31);
    if (c >= chunks) continue;
    float v[8];
    if (8 * c >= K) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    } else if (GATEUP) {
      const int t = s.row_tok[r];
      load8(p.x, p.x_dtype, t * p.ldx + 8 * c, p.x_vec, v);
      if (p.pre_w) {
        float w[8];
        load8(p.pre_w, p.norm_dtype, 8 * c, true, w);
        const float inv = s.inv[t];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * inv * w[j];
      }
    } else {
      const float4 *src = reinterpret_cast<const float4 *>(p.act + (int64_t)s.row_pair[r] * K) + 2 * c;
      const float4 a = __ldcg(src), b = __ldcg(src + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    if constexpr (KIND > kBf16Many) {
      const float mult = s.row_mult[r];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= mult;
    }
    uint8_t *dst = panel + (planes * r) * pitch + 16 * c;
#pragma unroll
    for (int i = 0; i < (KIND <= kBf16Many ? 3 : 2); ++i) {
      if (i == planes) break;
      uint4 q;
      q.x = plane2<KIND>(v[0], v[1]);
      q.y = plane2<KIND>(v[2], v[3]);
      q.z = plane2<KIND>(v[4], v[5]);
      q.w = plane2<KIND>(v[6], v[7]);
      *reinterpret_cast<uint4 *>(dst + i * pitch) = q;
    }
  }
  return built;
}

// The sums over the parts of K of the sub-tiles 0 .. n-1 of a batch, whose first output is `first`, and what becomes of them: a warp per
// sub-tile, lanes over tokens and outputs.
template <int KIND, bool GATEUP, bool EIGHT>
__device__ __forceinline__ void add_parts(const DecodeParams &p, Shared &s, const Item &it, int base, const float *red, int n, int first) {
  constexpr int kOuts = (GATEUP ? 8 : 16) / (EIGHT ? 2 : 1);
  const Shape &sh = p.shape[GATEUP ? 0 : 1];
  constexpr int kTeam = Geo<KIND>::kTeam;
  const int parts = kTeam / sh.subs, tokens = it.n;
  for (int u = threadIdx.x >> 5; u < n; u += kWarps)
    for (int o = threadIdx.x & 31; o < (tokens * kOuts + 31) / 32 * 32; o += 32) {
      const int r = o % kOuts, tok = o / kOuts, row = first + u * kOuts + r;
      const bool in = tok < tokens && row < it.r1;
      float a = 0.f, b = 0.f;
      if (in) {
        const float *src = red + (u * parts * tokens + tok) * 16 + r;
#pragma unroll
        for (int w = 0; w < kTeam; ++w) {
          if (w >= parts) break;
          a += src[w * tokens * 16];
          if (GATEUP) b += src[w * tokens * 16 + kOuts];
        }
        const float un = KIND <= kBf16Many ? 1.0f : s.row_unmult[base + tok];
        a *= un;
        b *= un;
        if (GATEUP) a = a / (1.0f + expf(-a)) * b;
        (GATEUP ? p.act : p.Y)[(int64_t)s.row_pair[base + tok] * sh.N + row] = a;
      }
      if constexpr (GATEUP && KIND > kBf16Many) {
        float m = in ? fabsf(a) : 0.f;
#pragma unroll
        for (int x = kOuts / 2; x > 0; x >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, x));
        // magnitudes order as their bits do, a NaN above all
        if (r == 0 && in) atomicMax(p.row_max + s.row_pair[base + tok], __float_as_uint(m) & 0x7fffffffu);
      }
    }
}

// One product over this CTA's items: gate, up and silu into p.act, or down into p.Y. The sixteen warps are groups, which take the tiles in
// turn, so that a tile's chain of waits, loads and MMAs runs beside others (all warps at one tile took three times as long as HBM needs to
// bring it). A group's warps are split among the sub-tiles, and a warp takes every parts-th run of 128 bytes of its rows; the sums meet in
// shared memory, [tile of the batch][sub-tile][part][token][row of 16].
// Every warp waits for every slot and releases it, in order, whether it reads it or not: a group that ran ahead or behind by the ring's
// length would take one phase of a barrier for another.
// A warp whose wait gives up raises s.fail, waits no more and frees no slot, but meets every barrier; what it forms then is never used.
template <int KIND, bool GATEUP, bool EIGHT>
__device__ __forceinline__ void run_product(const DecodeParams &p, Shared &s, Ring &ring, uint8_t *panel, float *sums, const uint8_t *slots) {
  constexpr int kElem = Geo<KIND>::kElem, kGroups = Geo<KIND>::kGroups, kTeam = Geo<KIND>::kTeam;
  constexpr int kOuts = (GATEUP ? 8 : 16) / (EIGHT ? 2 : 1), kRuns = (EIGHT ? 32 : 16) / kTeam;   // of a sub-tile; of a warp in a slice, at most
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  const Plan &plan = s.plan[GATEUP ? 0 : 1];
  const Shape &sh = p.shape[GATEUP ? 0 : 1];
  const int pitch = Geo<KIND>::pitch(sh.K), subs = sh.subs, parts = kTeam / subs, group = warp / kTeam, sub = warp & (subs - 1), part = (warp % kTeam) / subs;
  // this lane's bytes of row g of its sub-tile in a slot; row g + 8 is 8 rows behind it, or of gate and up row g of up. EIGHT: rows of gate, then of up
  const int row0 = (sub * kOuts + g) * sh.slice + part * 128 + j * 16;
  constexpr bool kSwap = KIND <= kF16;
  const bool odd = (g & 1) && (sh.slice & 64) == 0;
  int built = 0, base = 0, turn = 0;   // turn: whose tile it is
  bool ok = true;
  for (int i = 0; i < plan.n_items; ++i) {
    const Item &it = plan.item[i];
    if (i >= built) {
      meet();   // the last panel is read
      built = build_panel<KIND, GATEUP>(p, s, plan, sh.K, panel, i);
      base = 0;
      meet();
    }
    const int n = it.n, last = it.r1, batch = kRed / (64 * kTeam * n);   // tiles whose sums fit
    // This lane's runs of the planes that are the MMAs' columns g, 8 + g and 16 + g (EIGHT: rows). Two planes: both of the first four tokens, then of
    // the others; EIGHT: the first plane of eight tokens, then the second. Three planes of
    //   up to two tokens   each plane of either
    //   up to five         the first two planes of tokens 0 .. 3; their third and between them the planes of token 4
    //   kBf16Many          the first two planes of tokens 0 .. 3; the third of 0, 4, 1, 5 ..; the first two of tokens 4 .. 7
    //   EIGHT              the first plane of five tokens and the third of 0, 1, 2; the second plane of five and the third of 3, 4
    auto run_of = [&](int token, int plane) { return panel + (sh.planes * (base + min(token, n - 1)) + plane) * pitch + (part * 128 + j * 16) * (2 / kElem); };
    const uint8_t *x0, *x1;
    const uint8_t *x2 = panel;   // kBf16Many
    if constexpr (KIND <= kBf16Many && EIGHT) {
      x0 = g < 5 ? run_of(g, 0) : run_of(g - 5, sh.planes - 1);
      x1 = g < 5 ? run_of(g, 1) : run_of(g - 2, sh.planes - 1);
    } else if constexpr (KIND <= kBf16Many) {
      x0 = n <= 2 ? run_of(g & 1, min(g >> 1, 2)) : run_of(g >> 1, g & 1);
      if constexpr (KIND == kBf16) {
        x1 = g & 1 ? run_of(4, min(g >> 1, 2)) : run_of(g >> 1, 2);
      } else {
        x1 = run_of((g >> 1) + 4 * (g & 1), 2);
        x2 = run_of(4 + (g >> 1), g & 1);
      }
    } else {
      x0 = EIGHT ? run_of(g, 0) : run_of(g >> 1, g & 1);
      x1 = EIGHT ? run_of(g, 1) : run_of(4 + (g >> 1), g & 1);
    }
    int in_batch = 0;
    for (int first = it.r0; first < last; first += sh.outs) {
      if (turn != group) {
        for (int sl = 0; sl < sh.slices; ++sl) {
          if (ok && !mbar_wait_for(&s.full[ring.at], ring.parity, p.wait_cycles, &s.fail)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (lane == 0 && ok) mbar_arrive(&s.empty[ring.at]);
          ring.next();
        }
      } else {
        const bool mine = first + sub * kOuts < last;   // the last tile may have fewer sub-tiles
        // columns 0 .. 7, 8 .. 15, 16 .. (EIGHT: rows 0 .. 15, even and odd steps, 16 ..): no sum's order depends on a token's place. (Two accumulators for either four
        // tokens take registers that are not there: int8 16 tokens 110 us, so 100.)
        constexpr int kSets = KIND == kBf16Many ? 3 : 2, kLast = kSets - 1;
        float acc[kSets][4] = {};
        // e4m3: scales of the blocks of rows g and g + 8; EIGHT: of rows 2 j and 2 j + 1, which are in one, runs starting at even rows
        const float *sc0 = nullptr, *sc1 = nullptr;
        if constexpr (KIND == kE4) {
          const int kb = (sh.K + 127) / 128, nb = (sh.N + 127) / 128, row = first + sub * kOuts + (EIGHT ? 2 * j : g);
          const bool up = EIGHT && GATEUP && j >= 2;
          sc0 = (GATEUP ? (up ? p.s_up : p.s_gate) : p.s_down) + ((int64_t)it.expert * nb + min((row - (up ? 4 : 0)) / 128, nb - 1)) * kb + part;
          sc1 = EIGHT ? sc0 : (GATEUP ? p.s_up : p.s_down) + ((int64_t)it.expert * nb + min((row + (GATEUP ? 0 : 8)) / 128, nb - 1)) * kb + part;
        }
        float row_scale[2] = {1.f, 1.f};   // int8: of the rows whose sums this lane will hold, g and g + 8 or 2 j and 2 j + 1
        for (int sl = 0; sl < sh.slices; ++sl) {
          const int left = mine ? min(sh.slice, sh.row_bytes - sl * sh.slice) - part * 128 : 0;   // bytes from this warp's first run on
          float f[kRuns][2];
          if constexpr (KIND == kE4) {   // of all runs, ahead of the wait
#pragma unroll
            for (int r = 0; r < kRuns; ++r) {
              const int at = sl * (sh.slice / 128) + r * parts;
              f[r][0] = left > r * parts * 128 ? __ldg(sc0 + at) : 0.f;
              f[r][1] = EIGHT ? 0.f : left > r * parts * 128 ? __ldg(sc1 + at) : 0.f;
            }
          }
          if (ok && !mbar_wait_for(&s.full[ring.at], ring.parity, p.wait_cycles, &s.fail)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (KIND == kS8 && sl == 0) {   // row_scale's rows may lie behind the last copied one: what is read then is never used
            const float *a = s.scale[ring.at] + (first & 3) + sub * kOuts + (EIGHT ? 2 * j - (GATEUP && j >= 2 ? 4 : 0) : g);
            const int up = kScales / 2;
            row_scale[0] = a[EIGHT && GATEUP && j >= 2 ? up : 0];
            row_scale[1] = a[(EIGHT && GATEUP && j >= 2 ? up : 0) + (EIGHT ? 1 : GATEUP ? up : 8)];
          }
          const uint8_t *slot = slots + ring.at * kSlot + row0, *slot1 = slot + (GATEUP ? sh.outs : 8) * sh.slice;
          const int at = sl * sh.slice * (2 / kElem), run = parts * 128;
          auto runs = [&](auto sets) {
            auto one = [&](int r, int rest) {
              Weights<EIGHT ? 1 : 2> v;
              v.template load<kSwap>(slot + r * run, slot1 + r * run, odd, rest);
              // the second step may lie behind the row's end: its weights are zeros then, and the planes reach to the end of a run
              float t[2][4] = {};
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const int here = at + (r * run + u * 64) * (2 / kElem);
                if constexpr (EIGHT) step<KIND>(v.w[u], x0 + here, x1 + here, KIND == kE4 ? t[0] : acc[u]);
                else step<KIND, decltype(sets)::value>(v.w[u], x0 + here, x1 + here, x2 + here, KIND == kE4 ? t[0] : acc[0], KIND == kE4 ? t[1] : acc[1], acc[kLast]);
              }
              if constexpr (KIND == kE4) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  acc[0][c] = fmaf(f[r][EIGHT ? 0 : c >> 1], t[0][c], acc[0][c]);
                  if (decltype(sets)::value == 2) acc[1][c] = fmaf(f[r][c >> 1], t[1][c], acc[1][c]);
                }
              }
            };
            if constexpr (KIND <= kF16) {
#pragma unroll
              for (int r = 0; r < kRuns; ++r) {
                const int rest = left - r * run;
                if (rest <= 0) break;
                one(r, rest);
              }
            } else {   // two whole runs without a branch between them: the second's loads go ahead of the first's MMAs (e4m3 4 tokens 56 -> 54 us, 16 tokens
                       // 110 -> 107; bf16, whose runs are shorter, lost 5 to 10 % by it)
#pragma unroll
              for (int r = 0; r < kRuns; r += 2) {
                if (left >= (r + 1) * run + 128) {
                  one(r, 128);
                  one(r + 1, 128);
                } else {
                  if (left > r * run) one(r, left - r * run);
                  if (left > (r + 1) * run) one(r + 1, left - (r + 1) * run);
                  break;
                }
              }
            }
          };
          if (EIGHT || n <= (KIND <= kBf16Many ? 2 : 4)) runs(std::integral_constant<int, 1>());
          else runs(std::integral_constant<int, kSets>());
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(&s.empty[ring.at]);
          ring.next();
        }
        if (mine) {
          float *dst = sums + ((in_batch * subs + sub) * parts + part) * n * 16;
          if constexpr (KIND <= kBf16Many && EIGHT) {
            float v[4], third[2];
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = acc[0][c] + acc[1][c];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int from = (g < 3 ? 5 + g : 2 + g) * 4 + j;
              const float a = __shfl_sync(0xffffffffu, v[c], from), b = __shfl_sync(0xffffffffu, v[2 + c], from);
              third[c] = sh.planes == 2 ? 0.f : g < 3 ? a : b;
            }
            if (g < n) *reinterpret_cast<float2 *>(dst + g * 16 + 2 * j) = make_float2(v[0] + (v[2] + third[0]), v[1] + (v[3] + third[1]));
          } else if constexpr (KIND <= kBf16Many) {
            auto of_lane = [&](float v, int i) { return __shfl_sync(0xffffffffu, v, (lane & ~3) + i); };
            auto join = [&](float v) { return of_lane(v, 0) + (of_lane(v, 1) + of_lane(v, 2)); };   // a token's planes in three lanes
            dst += j * 16 + g;
            if (n <= 2) {
              const float a0 = join(acc[0][0]), b0 = join(acc[0][1]), a8 = join(acc[0][2]), b8 = join(acc[0][3]);
              if (j < n) {
                dst[0] = j == 0 ? a0 : b0;
                dst[8] = j == 0 ? a8 : b8;
              }
            } else {
              if (j < n) {
                dst[0] = acc[0][0] + (acc[0][1] + acc[1][0]);
                dst[8] = acc[0][2] + (acc[0][3] + acc[1][2]);
              }
              float e0, e8;
              if constexpr (KIND == kBf16) {
                e0 = join(acc[1][1]);
                e8 = join(acc[1][3]);
              } else {
                e0 = acc[kLast][0] + (acc[kLast][1] + acc[1][1]);
                e8 = acc[kLast][2] + (acc[kLast][3] + acc[1][3]);
              }
              if (4 + j < n) {
                dst[64] = e0;
                dst[72] = e8;
              }
            }
          } else if constexpr (EIGHT) {
            if (g < n)
              *reinterpret_cast<float2 *>(dst + g * 16 + 2 * j) = make_float2(((acc[0][0] + acc[1][0]) + (acc[0][2] + acc[1][2])) * row_scale[0],
                                                                              ((acc[0][1] + acc[1][1]) + (acc[0][3] + acc[1][3])) * row_scale[1]);
          } else {
            dst += j * 16 + g;
            if (j < n) {
              dst[0] = (acc[0][0] + acc[0][1]) * row_scale[0];
              dst[8] = (acc[0][2] + acc[0][3]) * row_scale[1];
            }
            if (4 + j < n) {
              dst[64] = (acc[1][0] + acc[1][1]) * row_scale[0];
              dst[72] = (acc[1][2] + acc[1][3]) * row_scale[1];
            }
          }
        }
      }
      turn = (turn + 1) % kGroups;
      if (++in_batch != batch && first + sh.outs < last) continue;
      meet();
      add_parts<KIND, GATEUP, EIGHT>(p, s, it, base, sums, in_batch * subs, first - (in_batch - 1) * sh.outs);
      in_batch = 0;
      meet();
    }
    if (GATEUP && threadIdx.x == 0 && *reinterpret_cast<volatile int *>(&s.fail) == 0) add_release(p.ready + it.expert, (unsigned)(last - it.r0));
    base += n;
  }
}

// A token's experts and weights, by one warp: top-k of the logits by (value descending, expert ascending), a softmax over the chosen ones (the
// others' part of the softmax over all falls out where the weights are renormalised). Lane l's experts are 32 i + l; every lane sorts its own
// (stable), and a round then takes the largest of the lanes' heads. -inf is the least of all values: with fewer than k others such experts
// follow, weight 0; of a row of -inf alone all weights are 0.
template <int EPL>
__device__ __forceinline__ void choose(const float *logits, int E, int k, int lane, int *sel_e, float *sel_w) {
  unsigned key[EPL];
  int id[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    // order-preserving: larger float <=> larger unsigned key; 0 only past the last expert
    const unsigned u = i * 32 + lane < E ? __float_as_uint(__ldcg(logits + i * 32 + lane)) : 0u;
    key[i] = i * 32 + lane < E ? max(1u, (u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;
    id[i] = i * 32 + lane;
  }
#pragma unroll
  for (int r = 0; r < EPL - 1; ++r)
#pragma unroll
    for (int i = EPL - 1; i > r; --i)
      if (key[i] > key[i - 1]) {
        const unsigned t = key[i]; key[i] = key[i - 1]; key[i - 1] = t;
        const int d = id[i]; id[i] = id[i - 1]; id[i - 1] = d;
      }
  unsigned mine = 0u;   // lane s < k: key of the s-th choice
#pragma unroll 1
  for (int s = 0; s < k; ++s) {
    const unsigned top = __reduce_max_sync(0xffffffffu, key[0]);
    const unsigned holders = __ballot_sync(0xffffffffu, key[0] == top);
    int src = __ffs(holders) - 1;
    if (holders & (holders - 1u))   // equal logits: the smallest id among the lanes that hold one
      src = __reduce_min_sync(0xffffffffu, key[0] == top ? id[0] : 0x7fffffff) & 31;
    if (lane == s) mine = top;
    if (lane == src) {
      sel_e[s] = id[0];
#pragma unroll
      for (int i = 0; i + 1 < EPL; ++i) {
        key[i] = key[i + 1];
        id[i] = id[i + 1];
      }
      key[EPL - 1] = 0u;
    }
  }
  const float v = __uint_as_float((mine & 0x80000000u) ? mine & 0x7fffffffu : ~mine), most = __shfl_sync(0xffffffffu, v, 0);
  const float e = lane < k && v != -INFINITY ? expf(v - most) : 0.f;
  float sum = e;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane < k) sel_w[lane] = sum == 0.f ? 0.f : e / sum;
  __syncwarp();
}

// What a matrix row costs where n tokens go through it, in sixteenths of the cheapest: more tokens read more of the panel at each step.
// (Gate and up of 16 tokens, time of the CTAs whose fullest expert has 1, 2, 3, 4, 5 tokens: bf16 80, 86, 90, 97, 100 us, int8 53, 54, 56, 56, 68.)
template <int KIND>
__device__ __forceinline__ int row_cost(int n) {
  constexpr int kMost = Geo<KIND>::kMost;
  const int full = n / kMost, last = n - full * kMost;
  auto pass = [](int m) { return KIND <= kF16 ? 15 + m : m <= 4 ? 16 : 20; };
  return full * pass(kMost) + (last ? pass(last) : 0);
}
// The matrix rows of a product, of all active experts in a row, are dealt to the CTAs by their cost, in pairs of rows. Where CTA b's begin:
// position `at` of the active list, pair `unit` of its `half`. By a whole warp; every CTA forms the same borders.
struct Border {
  int at;
  unsigned unit;
};
__device__ __forceinline__ Border border(const DecodeParams &p, const Shared &s, unsigned half, unsigned b) {
  const int lane = threadIdx.x & 31;
  if (b == gridDim.x) return Border{s.n_active, 0u};
  const unsigned total = s.cost[s.n_active] * half;   // below 128 x 46 x 20480
  const unsigned pos = (unsigned)((unsigned long long)total * b * p.grid_inverse >> 32);
  int at = -1;
#pragma unroll
  for (int i = 0; i < kMaxTokens * kMaxK / 32; ++i) {
    const int j = 32 * i + lane;
    at += __popc(__ballot_sync(0xffffffffu, j < s.n_active && s.cost[j] * half <= pos));
  }
  const unsigned unit = (unsigned)__fdividef((float)(pos - s.cost[at] * half), (float)(s.cost[at + 1] - s.cost[at]));
  return Border{at, min(unit, half)};
}
// This CTA's items between two borders; an expert's tokens go through in passes of up to kMaxRows. False where there are more items than room
// for them (a device of KNJ_MOE_DECODE_MIN_SMS SMs comes to 32 of kMaxItems: a share of the cost and two experts at its borders).
__device__ __forceinline__ bool make_plan(Plan &plan, const Shared &s, int N, int pass, int cap, Border from, Border to, int most_items) {
  bool fits = true;
  int n = 0, panel = 0, held = 0, most = 0;
  for (int i = from.at; i <= to.at && i < s.n_active; ++i) {
    const unsigned begin = i == from.at ? from.unit : 0u, end = i == to.at ? to.unit : N / 2;
    const int e = s.active[i], rows = __popc(s.mask[e]);
    for (int f = 0; begin < end && f < rows; f += pass) {
      if (n == most_items) {
        fits = false;
        break;
      }
      const int c = min(pass, rows - f);
      if (held + c > cap) {
        panel = n;
        held = 0;
      }
      held += c;
      most = max(most, held);
      plan.item[n++] = Item{e, 2 * (int)begin, 2 * (int)end, f, c, panel};
    }
  }
  plan.n_items = n;
  plan.rows = most;
  return fits;
}

// ---- stages 1 and 4 -----------------------------------------------------------------------------------------------------

// four consecutive values; `vec`: at a 16-byte (two-byte types: 8-byte) boundary
__device__ __forceinline__ float4 load4(const void *base, int dtype, int64_t i, bool vec) {
  if (!vec) return make_float4(load_as_f32(base, dtype, i), load_as_f32(base, dtype, i + 1), load_as_f32(base, dtype, i + 2), load_as_f32(base, dtype, i + 3));
  if (dtype == KNJ_DT_F32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i);
  const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + i);
  if (dtype == KNJ_DT_BF16)
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ bool fours(const void *base, int64_t ld, int dtype) {
  const int64_t unit = dtype == KNJ_DT_F32 ? 16 : 8;
  return reinterpret_cast<uintptr_t>(base) % unit == 0 && ld * (dtype == KNJ_DT_F32 ? 4 : 2) % unit == 0;
}
__device__ __forceinline__ void store4(void *base, int dtype, int64_t i, bool vec, float4 v) {
  if (!vec) {
    store_from_f32(base, dtype, i, v.x);
    store_from_f32(base, dtype, i + 1, v.y);
    store_from_f32(base, dtype, i + 2, v.z);
    store_from_f32(base, dtype, i + 3, v.w);
    return;
  }
  if (dtype == KNJ_DT_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(base) + i) = v;
    return;
  }
  uint2 u;
  if (dtype == KNJ_DT_BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    u = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  } else {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    u = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  }
  *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + i) = u;
}

__device__ __forceinline__ float inverse_rms(float sum, int H, float eps) { return rsqrtf(fmaf(sum, 1.0f / (float)H, eps)); }

// sum of squares of the row in shared memory and its inverse norm; a large row once more
__device__ __forceinline__ float row_inverse(const float *row, int H, float ss, float eps, float (*red)[kWarps]) {
  const float tot = cta_sum(ss, red[0]);
  if (!(tot > 3.402823466e38f)) return inverse_rms(tot, H, eps);
  float q = 0.f;
  for (int i = threadIdx.x; i < H; i += kThreads) q = fmaf(row[i] * kDown, row[i] * kDown, q);
  return kDown * rsqrtf(cta_sum(q, red[1]) * (1.0f / (float)H));
}

// What stands behind the experts, of one token: a thread holds runs of four channels, the first of them with all that does not depend on
// the experts read in front of the last barrier (prepare).
struct Finish {
  float4 x, post, gate, next;

  __device__ __forceinline__ void load(const DecodeParams &p, int t, int c) {
    x = load4(p.x, p.x_dtype, t * p.ldx + c, fours(p.x, p.ldx, p.x_dtype));
    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
    post = p.post_w ? load4(p.post_w, p.norm_dtype, c, fours(p.post_w, 0, p.norm_dtype)) : one;
    next = p.next_w ? load4(p.next_w, p.norm_dtype, c, fours(p.next_w, 0, p.norm_dtype)) : one;
    gate = one;
    if (p.gate_kind == KNJ_GATE_NONE) return;
    if (p.gate_kind == KNJ_GATE_ROW) {
      const float g = load_as_f32(p.gate, p.gate_dtype, t * p.ldg);
      gate = make_float4(g, g, g, g);
    } else {
      const bool full = p.gate_kind == KNJ_GATE_FULL;
      gate = load4(p.gate, p.gate_dtype, full ? t * p.ldg + c : c, fours(p.gate, full ? p.ldg : 0, p.gate_dtype));
    }
    if (p.gate_sigmoid)
      gate = make_float4(1.0f / (1.0f + expf(-gate.x)), 1.0f / (1.0f + expf(-gate.y)), 1.0f / (1.0f + expf(-gate.z)), 1.0f / (1.0f + expf(-gate.w)));
  }
  __device__ __forceinline__ void prepare(const DecodeParams &p, int t) {
    if (4 * threadIdx.x < p.H) load(p, t, 4 * threadIdx.x);
  }
  // row: H values in shared memory, of which a thread reads only its own (e4m3 rows: all)
  __device__ __forceinline__ void run(const DecodeParams &p, Shared &s, int t, float *row) {
    const int first = 4 * threadIdx.x, H = p.H;
    constexpr int kStride = 4 * kThreads;
    float ss = 0.f;
    for (int c = first; c < H; c += kStride) {
      float4 v[kMaxK], y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kMaxK; ++j)
        if (j < p.k) v[j] = __ldcg(reinterpret_cast<const float4 *>(p.Y + ((int64_t)t * p.k + s.order[t][j]) * H + c));
#pragma unroll
      for (int j = 0; j < kMaxK; ++j)
        if (j < p.k) {
          const float weight = s.sel_w[t][s.order[t][j]];
          y.x = fmaf(weight, v[j].x, y.x);
          y.y = fmaf(weight, v[j].y, y.y);
          y.z = fmaf(weight, v[j].z, y.z);
          y.w = fmaf(weight, v[j].w, y.w);
        }
      *reinterpret_cast<float4 *>(row + c) = y;
      ss = fmaf(y.x, y.x, fmaf(y.y, y.y, fmaf(y.z, y.z, fmaf(y.w, y.w, ss))));
    }
    const float inv = p.post_w ? row_inverse(row, H, ss, p.eps, s.red) : 1.0f;
    const bool out4 = fours(p.out, p.ldo, p.out_dtype);
    ss = 0.f;
    for (int c = first; c < H; c += kStride) {
      if (c != first) load(p, t, c);
      float4 v = *reinterpret_cast<const float4 *>(row + c);
      v.x = fmaf(p.beta, x.x, p.alpha * gate.x * (v.x * inv * post.x));
      v.y = fmaf(p.beta, x.y, p.alpha * gate.y * (v.y * inv * post.y));
      v.z = fmaf(p.beta, x.z, p.alpha * gate.z * (v.z * inv * post.z));
      v.w = fmaf(p.beta, x.w, p.alpha * gate.w * (v.w * inv * post.w));
      store4(p.out, p.out_dtype, t * p.ldo + c, out4, v);
      *reinterpret_cast<float4 *>(row + c) = v;
      ss = fmaf(v.x, v.x, fmaf(v.y, v.y, fmaf(v.z, v.z, fmaf(v.w, v.w, ss))));
    }
    if (!p.next_w) return;
    const float inv2 = row_inverse(row, H, ss, p.eps, s.red + 2);
    const bool codes = p.h_dtype == KNJ_DT_E4M3, h4 = !codes && fours(p.h_next, p.ldh, p.h_dtype);
    for (int c = first; c < H; c += kStride) {   // 32 threads in a row hold a group of 128 values
      if (H > kStride) next = load4(p.next_w, p.norm_dtype, c, fours(p.next_w, 0, p.norm_dtype));
      float4 v = *reinterpret_cast<const float4 *>(row + c);
      v = make_float4(v.x * inv2 * next.x, v.y * inv2 * next.y, v.z * inv2 * next.z, v.w * inv2 * next.w);
      if (!codes) {
        store4(p.h_next, p.h_dtype, t * p.ldh + c, h4, v);
        continue;
      }
      float most = max3_abs_nan(max3_abs_nan(0.f, v.x, v.y), v.z, v.w);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
      const Fp8Scale sc = fp8_scale(most);
      const uint32_t lo = e4m3_pair(v.x * sc.inverse, v.y * sc.inverse), hi = e4m3_pair(v.z * sc.inverse, v.w * sc.inverse);
      uint8_t *at = static_cast<uint8_t *>(p.h_next) + t * p.ldh + c;
      if ((reinterpret_cast<uintptr_t>(p.h_next) | (uintptr_t)p.ldh) % 4 == 0) {
        *reinterpret_cast<uint32_t *>(at) = lo | hi << 16;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = (uint8_t)((lo | hi << 16) >> (8 * j));
      }
      if ((threadIdx.x & 31) == 0) p.h_next_scale[(int64_t)t * (H / kFp8Group) + c / kFp8Group] = sc.scale;
    }
  }
};

// A wait gave up: the others are told, and the rows that this CTA would have written are NaN. 
__device__ void give_up(const DecodeParams &p, Shared &s) {
  if (threadIdx.x == 0) {
    *reinterpret_cast<volatile int *>(&s.fail) = 1;
    atomicExch(p.sync + 1, 1u);
    atomicExch(p.status, 1);
  }
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

// Logits, and with the first experts' the statistics of the tokens' rows. The tokens x experts are dealt to the CTAs in squares of up to
// four by four, for which 4 + 4 rows are read; a thread takes runs of four channels, so that all its loads go out together (a warp
// per token over all of x in every CTA: 7 us at sixteen tokens).
template <int SIDE>
__global__ void __launch_bounds__(kThreads) moe_decode_front_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float part[kWarps][SIDE][2 + SIDE];   // of a token: squares, largest, dot products
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int token_tiles = (p.T + SIDE - 1) / SIDE;
  const bool x4 = fours(p.x, p.ldx, p.x_dtype);
  const int t0 = blockIdx.x % token_tiles * SIDE, e0 = blockIdx.x / token_tiles * SIDE;
  grid_dep_wait();   // x comes from an earlier launch, which may still use the workspace
  if (blockIdx.x == 0) {
    if (tid < 2) p.sync[tid] = 0u;
    if (tid == 2) *p.status = 0;
    if (tid < kMaxTokens * kMaxK) p.row_max[tid] = 0u;
    if (tid < kMaxExperts) p.ready[tid] = 0u;
  }
  float ss[SIDE], most[SIDE], dot[SIDE][SIDE];
#pragma unroll
  for (int i = 0; i < SIDE; ++i) {
    ss[i] = most[i] = 0.f;
#pragma unroll
    for (int k = 0; k < SIDE; ++k) dot[i][k] = 0.f;
  }
  for (int c = 4 * tid; c < p.H; c += 4 * kThreads) {
    float4 x[SIDE], n = make_float4(1.f, 1.f, 1.f, 1.f);
    uint2 r[SIDE];
#pragma unroll
    for (int k = 0; k < SIDE; ++k) r[k] = *reinterpret_cast<const uint2 *>(p.router + (int64_t)min(e0 + k, p.E - 1) * p.H + c);
#pragma unroll
    for (int i = 0; i < SIDE; ++i) x[i] = load4(p.x, p.x_dtype, min(t0 + i, p.T - 1) * p.ldx + c, x4);
    if (p.pre_w) n = load4(p.pre_w, p.norm_dtype, c, true);
#pragma unroll
    for (int i = 0; i < SIDE; ++i) {
      float4 &v = x[i];
      ss[i] = fmaf(v.x, v.x, fmaf(v.y, v.y, fmaf(v.z, v.z, fmaf(v.w, v.w, ss[i]))));
      v = make_float4(v.x * n.x, v.y * n.y, v.z * n.z, v.w * n.w);
      most[i] = max3_abs_nan(max3_abs_nan(most[i], v.x, v.y), v.z, v.w);
#pragma unroll
      for (int k = 0; k < SIDE; ++k)
        dot[i][k] = fmaf(v.x, __uint_as_float(r[k].x << 16), fmaf(v.y, __uint_as_float(r[k].x & 0xffff0000u),
                    fmaf(v.z, __uint_as_float(r[k].y << 16), fmaf(v.w, __uint_as_float(r[k].y & 0xffff0000u), dot[i][k]))));
    }
  }
#pragma unroll
  for (int i = 0; i < SIDE; ++i) {
    ss[i] = warp_sum(ss[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most[i] = max_nan(most[i], __shfl_xor_sync(0xffffffffu, most[i], o));
#pragma unroll
    for (int k = 0; k < SIDE; ++k) dot[i][k] = warp_sum(dot[i][k]);
  }
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < SIDE; ++i) {
      part[warp][i][0] = ss[i];
      part[warp][i][1] = most[i];
#pragma unroll
      for (int k = 0; k < SIDE; ++k) part[warp][i][2 + k] = dot[i][k];
    }
  }
  __syncthreads();
  const int i = warp, t = t0 + i;   // a warp per token, lane l the sum of value l
  if (i >= SIDE || t >= p.T) return;
  float v = 0.f;
  if (lane < 2 + SIDE)
    for (int w = 0; w < kWarps; ++w) v = lane == 1 ? max_nan(v, part[w][i][1]) : v + part[w][i][lane];
  const float tot = __shfl_sync(0xffffffffu, v, 0);
  float inv = 1.0f, scale = 1.0f;   // of the row's values; of the sums over it
  if (p.pre_w) {
    if (tot > 3.402823466e38f) {   // squares of a large row left the range, other sums may have: all from values * 2^-80, where eps does not count
      float q = 0.f, d[SIDE], far = 0.f;
#pragma unroll
      for (int k = 0; k < SIDE; ++k) d[k] = 0.f;
      for (int c = lane; c < p.H; c += 32) {
        const float f = load_as_f32(p.x, p.x_dtype, t * p.ldx + c) * kDown, g = f * load_as_f32(p.pre_w, p.norm_dtype, c);
        q = fmaf(f, f, q);
        far = max3_abs_nan(far, g, 0.f);
#pragma unroll
        for (int k = 0; k < SIDE; ++k) d[k] = fmaf(g, __uint_as_float((uint32_t)p.router[(int64_t)min(e0 + k, p.E - 1) * p.H + c] << 16), d[k]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) far = max_nan(far, __shfl_xor_sync(0xffffffffu, far, o));
      v = far;
#pragma unroll
      for (int k = 0; k < SIDE; ++k) {
        const float sum = warp_sum(d[k]);
        if (lane == 2 + k) v = sum;
      }
      scale = rsqrtf(warp_sum(q) * (1.0f / (float)p.H));
      inv = kDown * scale;
    } else {
      inv = scale = inverse_rms(tot, p.H, p.eps);
    }
  }
  const float m = __shfl_sync(0xffffffffu, v, 1);
  const int e = e0 + lane - 2;
  if (lane >= 2 && lane < 2 + SIDE && e < p.E) p.logits[t * p.E + e] = v * scale + (p.router_bias ? p.router_bias[e] : 0.f);
  if (e0 == 0 && lane == 0) p.stats[t] = make_float2(inv, m * scale);
}

template <int KIND>
__global__ void __launch_bounds__(kAll, 1) moe_decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Shared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid < kMaxExperts) s.mask[tid] = 0u;
  if (tid == 0) {
    for (int i = 0; i < kMaxSlots; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], kWarps);
    }
    s.fail = 0;
    mbar_init_fence();
  }
  __syncthreads();

  // ---- routing: a warp per token ----
  if (warp < p.T) {
    const float2 st = __ldcg(p.stats + warp);
    if (p.E <= 128) choose<4>(p.logits + warp * p.E, p.E, p.k, lane, s.sel_e[warp], s.sel_w[warp]);
    else choose<8>(p.logits + warp * p.E, p.E, p.k, lane, s.sel_e[warp], s.sel_w[warp]);
    if (lane < p.k) {
      const int e = s.sel_e[warp][lane];
      atomicOr(&s.mask[e], 1u << warp);
      if (blockIdx.x == 0 && p.tap_exp) p.tap_exp[warp * p.k + lane] = e;
      if (blockIdx.x == 0 && p.tap_w) p.tap_w[warp * p.k + lane] = s.sel_w[warp][lane];
      // in ascending order of the experts, in which their rows are added
      int rank = 0;
      for (int i = 0; i < p.k; ++i) rank += s.sel_e[warp][i] < e;
      s.order[warp][rank] = lane;
    }
    if (lane == 0) {
      s.inv[warp] = st.x;
      row_power(st.y, s.mult[warp], s.unmult[warp]);
    }
  }
  __syncthreads();
  if (warp < p.T && lane < p.k) {
    const int e = s.sel_e[warp][lane];
    s.pair_at[e][__popc(s.mask[e] & ((1u << warp) - 1u))] = (uint8_t)(warp * p.k + lane);
  }
  if (warp == 0) {
    // this lane's eight experts: which are active, and in one word their number and, from bit 8 on, their cost
    unsigned on = 0u, sum = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned m = s.mask[8 * lane + i];
      if (m == 0u) continue;
      on |= 1u << i;
      sum += 1u + ((unsigned)row_cost<KIND>(__popc(m)) << 8);
    }
    unsigned before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    if (lane == 31) {
      s.n_active = before & 255u;
      s.cost[before & 255u] = before >> 8;
    }
    before -= sum;
    for (; on; on &= on - 1u) {
      const int e = 8 * lane + __ffs(on) - 1;
      s.active[before & 255u] = e;
      s.cost[before & 255u] = before >> 8;
      before += 1u + ((unsigned)row_cost<KIND>(__popc(s.mask[e])) << 8);
    }
  }
  __syncthreads();
  if (warp < 2) {   // a warp for each product
    const int N = warp == 0 ? p.F : p.H, K = warp == 0 ? p.H : p.F;
    const Border from = border(p, s, N / 2, blockIdx.x), to = border(p, s, N / 2, blockIdx.x + 1);
    // a plan that is not whole is a wait that gave up
    if (lane == 0 && !make_plan(s.plan[warp], s, N, Geo<KIND>::pass(K), Geo<KIND>::cap(K), from, to, p.stall == 3 ? 1 : kMaxItems))
      *reinterpret_cast<volatile int *>(&s.fail) = 1;
  }
  __syncthreads();

  float *sums = reinterpret_cast<float *>(smem);
  uint8_t *panel = smem + kRed;
  const int held = max(s.plan[0].rows * p.shape[0].planes * Geo<KIND>::pitch(p.H), s.plan[1].rows * p.shape[1].planes * Geo<KIND>::pitch(p.F));
  const int at = kRed + (held + 127) / 128 * 128;
  uint8_t *slots = smem + at;
  Ring ring{0, min(kMaxSlots, (kSmem - at) / kSlot), 0u};
  if (warp == kWarps) {
    int copied = 0;
    if (!feed<KIND>(p, s, 0, ring, slots, copied) || !feed<KIND>(p, s, 1, ring, slots, copied)) {
      // the slots filled last may still be written: shared memory is not left before they are
      if (lane < ring.n && copied > lane) mbar_wait_for(&s.full[lane], (uint32_t)((copied - lane - 1) / ring.n) & 1u, p.wait_cycles, nullptr);
    }
    return;
  }
  if constexpr (KIND == kBf16Many) {   // rows of few bytes alone
    run_product<KIND, true, false>(p, s, ring, panel, sums, slots);
    run_product<KIND, false, false>(p, s, ring, panel, sums, slots);
  } else {
    if (p.shape[0].eight) run_product<KIND, true, true>(p, s, ring, panel, sums, slots);
    else run_product<KIND, true, false>(p, s, ring, panel, sums, slots);
    if (p.shape[1].eight) run_product<KIND, false, true>(p, s, ring, panel, sums, slots);
    else run_product<KIND, false, false>(p, s, ring, panel, sums, slots);
  }
  grid_arrive(p, s);
  const int t = blockIdx.x;
  Finish end;
  if (t < p.T) end.prepare(p, t);
  const bool ok = grid_wait(p, s);
  if (ok && t < p.T) end.run(p, s, t, reinterpret_cast<float *>(panel));
  if (!ok) give_up(p, s);   // ends the copying warp's waits, too
}

template <int KIND>
int launch(DecodeParams &p, cudaStream_t st) {
  for (int i = 0; i < 2; ++i) {
    Shape &sh = p.shape[i];
    sh.K = i == 0 ? p.H : p.F;
    sh.N = i == 0 ? p.F : p.H;
    sh.row_bytes = sh.K * Geo<KIND>::kElem;
    sh.planes = Geo<KIND>::planes(sh.K);
    sh.slices = (sh.row_bytes + kSlice - 1) / kSlice;
    sh.slice = sh.slices == 1 ? sh.row_bytes : ((sh.row_bytes + sh.slices - 1) / sh.slices + 127) / 128 * 128;
    sh.eight = sh.row_bytes > kSlice / 2;
    sh.subs = sh.row_bytes <= kSlice / 8 ? 4 : sh.row_bytes <= kSlice / 4 ? 2 : 1;
    sh.outs = (i == 0 ? 8 : 16) * sh.subs / (sh.eight ? 2 : 1);
  }
  int dev = 0;
  KNJ_CUDA(cudaGetDevice(&dev));
  auto kern = moe_decode_kernel<KIND>;
  static bool opted[64] = {false};
  if (dev >= 0 && dev < 64 && !opted[dev]) {
    KNJ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    opted[dev] = true;
  }
  const int side = p.T == 1 ? 1 : p.T <= 4 ? 2 : 4;
  const dim3 front((unsigned)(((p.T + side - 1) / side) * ((p.E + side - 1) / side)));
  if (side == 1) KNJ_CUDA(launch_chain(moe_decode_front_kernel<1>, front, dim3(kThreads), 0, st, p));
  else if (side == 2) KNJ_CUDA(launch_chain(moe_decode_front_kernel<2>, front, dim3(kThreads), 0, st, p));
  else KNJ_CUDA(launch_chain(moe_decode_front_kernel<4>, front, dim3(kThreads), 0, st, p));
  const int rc = launch_status("moe_decode_front_kernel");
  if (rc) return rc;
  void *args[] = {&p};
  KNJ_CUDA(cudaLaunchCooperativeKernel(reinterpret_cast<const void *>(kern), dim3(sm_count()), dim3(kAll), args, kSmem, st));
  return launch_status("moe_decode_kernel");
}

// bf16: passes of up to five tokens, or where experts have three and more on average and no row is in tiles of eight, of up to eight. us, by
// (experts, hidden, ffn, top_k, tokens), five and eight: (32, 1024, 512, 8, 12) 41.0, 37.8, (.., 16) 46.6, 40.0; (20, 512, 208, 8, 8) 28.3, 25.6,
// (.., 16) 37.8, 33.3; (8, 1024, 512, 2, 16) 33.3, 28.7. Fewer tokens an expert lose by it: (128, 1024, 512, 8, 16) 65.0, 69.7.
int launch_bf16(DecodeParams &p, cudaStream_t st) {
  const int longest = p.H > p.F ? p.H : p.F;
  return 2 * longest <= kSlice / 2 && p.T * p.k >= 3 * p.E ? launch<kBf16Many>(p, st) : launch<kBf16>(p, st);
}

}  // namespace

namespace knj {
size_t moe_decode_workspace(int T, int H, int F, int E, int k) {
  auto up256 = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const size_t P = (size_t)T * k;
  return kHead + up256((size_t)T * E * 4) + up256(P * F * 4) + up256(P * H * 4);
}

int moe_decode_launch(const knj_moe_block_args *a, int32_t *status, knj_stream_t stream) {
  auto up256 = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const int T = a->n_tokens, H = a->hidden, F = a->ffn, E = a->n_experts, k = a->top_k;
  KNJ_REQUIRE(T <= kMaxTokens, "knj_moe_block_decode: %d tokens, at most %d", T, kMaxTokens);
  KNJ_REQUIRE(F <= KNJ_MOE_DECODE_MAX_FFN, "knj_moe_block_decode: ffn=%d above %d", F, KNJ_MOE_DECODE_MAX_FFN);
  KNJ_REQUIRE(aligned16(a->pre_w), "knj_moe_block_decode: pre_w must be 16-byte aligned");
  KNJ_REQUIRE(a->w_dtype != KNJ_DT_I8 || (aligned16(a->gate_scale) && aligned16(a->up_scale) && aligned16(a->down_scale)),
              "knj_moe_block_decode: the scales of int8 matrices must be 16-byte aligned");
  // a CTA's items: its share of the cost and two experts at its borders, sixteen passes each, stay far below kMaxItems then
  KNJ_REQUIRE(sm_count() >= KNJ_MOE_DECODE_MIN_SMS, "knj_moe_block_decode: a device of %d SMs or more needed", KNJ_MOE_DECODE_MIN_SMS);
  DecodeParams p{};
  p.x = a->x; p.pre_w = a->pre_w; p.post_w = a->post_w; p.next_w = a->next_w; p.gate = a->gate; p.router = a->w_router; p.router_bias = a->router_bias;
  p.w_gate = static_cast<const uint8_t *>(a->w_gate); p.w_up = static_cast<const uint8_t *>(a->w_up); p.w_down = static_cast<const uint8_t *>(a->w_down);
  p.s_gate = a->gate_scale; p.s_up = a->up_scale; p.s_down = a->down_scale; p.out = a->out; p.h_next = a->h_next; p.h_next_scale = a->h_next_scale;
  p.tap_exp = a->tap_pair_exp; p.tap_w = a->tap_pair_w;
  uint8_t *ws = static_cast<uint8_t *>(a->workspace);
  p.sync = reinterpret_cast<unsigned *>(ws + kSyncAt);   // behind the status word of the whole block
  p.row_max = reinterpret_cast<unsigned *>(ws + kMaxAt);
  p.stats = reinterpret_cast<float2 *>(ws + kStatsAt);
  p.ready = reinterpret_cast<unsigned *>(ws + kReadyAt);
  ws += kHead;
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
  p.wait_cycles = decode_wait_cycles(); p.stall = t_stall; p.grid_inverse = (unsigned)((1ull << 32) / sm_count());
  const cudaStream_t st = as_stream(stream);
  switch (a->w_dtype) {
    case KNJ_DT_BF16: return launch_bf16(p, st);
    case KNJ_DT_F16: return launch<kF16>(p, st);
    case KNJ_DT_E4M3: return launch<kE4>(p, st);
    default: return launch<kS8>(p, st);
  }
}
}  // namespace knj

extern "C" void knj_moe_block_decode_test_stall(int what) { t_stall = what >= 1 && what <= 3 ? what : 0; }
