// knj_expert_tc.cu -- products of routed rows with expert matrices held in bf16, fp16 or e4m3 (one scale for each block of
// 128 x 128), grouped by expert, and the dense e4m3 product, which is the same with one expert and all rows.
//
//   out[p][n] = out_scale * x[row(p)] . w[e][n]     and     out_scale * silu(x . wg[e][n]) * (x . wu[e][n])
//   e4m3:  x . w = sum over blocks b of 128 k:  sx[row][b] * sw[n/128][b] * sum_{k in b} qx[k] qw[k]
//
// Few rows are bound by the matrices' bytes: every active expert's matrix is read once (512 rows x 8 of 128 experts, bf16: 806 MB, 131 us,
// 0.94 of the measured copy rate). Many rows are bound by the tensor core: 16384 rows, bf16, 1.38 PFLOP/s alone, 1.13 in a loop under
// the power limit. One kernel with three forms (enum Form; launch_rule says when) walks over (bucket, row tile) tiles; a bucket is up
// to kTok routed rows of one expert, and consecutive tiles share it, so that its rows stay in L2 while the matrices stream through
// once. Persistent CTAs. In all forms but one the MMA's M side is matrix rows and its N side the bucket, so that a ragged bucket wastes
// less than 16 (32 in a pair) columns and a single token less than a tile; e4m3 in pairs has it the other way round (see the epilogue).
// Warps:
//   epilogue   accumulators from tensor memory, scales, SiLU * up, stores
//   MMA        tcgen05; accumulators are double-buffered, so a tile's stores overlap the next tile's products
//   matrix     TMA boxes of 128 bytes of K: 128 rows, or for gate and up eight boxes of 16 rows in turn -- gate and up of one output
//              then lie 16 lanes apart in one warp and meet by a shuffle
//   rows       tile::gather4 TMA copies of four routed rows each; boxes where the rows are all rows in order
//   scales     e4m3: the rows' and the matrix blocks' scales, four blocks of K to a group, by asynchronous copies; 16 bits: finds
//              the tiles and their rows in the tables, a tile ahead (in e4m3 the matrix warp does)
// In 16 bits the tensor core adds over all of K. In e4m3 each block of K is one accumulator buffer, which the epilogue scales and
// adds to its registers in f32 while the tensor core fills the others.
//
// Every wait on an mbarrier is bounded (knj_decode_wait_limit); on give-up the kernel raises a status flag, stores NaN in place of the
// outputs it did not form, frees its tensor memory and returns. Barriers of a CTA or a cluster have no limit of their own: all their
// warps meet all of them, whichever gave up.
#include "knj_fp8.cuh"
#include "knj_tc.cuh"

#include <type_traits>

using namespace knj;

namespace {

constexpr int kMaxExperts = 256;
constexpr int64_t kMaxPairs = 1 << 30;   // sums of a count and a bucket's size stay in 32 bits

struct GemmParams {
  const uint8_t *x;
  int64_t x_row;              // bytes from row to row
  const float *xs, *ws0, *ws1;
  const int32_t *pair_idx, *pair_cnt, *row_map;  // pair_idx null: one expert, pair i is row i
  void *out;
  int *status;
  int64_t ldo, idx_stride;
  int out_dtype, N, K, E, row_div, n_rows, n_pairs, m_tiles;
  int part_bits;              // 2^part_bits CTAs share a tile's K
  uint32_t m_inverse;         // floor(2^32 / m_tiles), at most 2^32 - 1
  uint32_t idesc_format;
  int vec_out;                // bases and strides of the outputs allow 16-byte (lane = row form: 32-byte) stores
  int dense;                  // rows 0 .. n_pairs-1 in order: copied as boxes instead of gathered
  float out_scale;
  int stall;                  // test hook (knj_expert_tc_test_stall)
  long long wait_cycles;      // limit of the waits on mbarriers
  CUtensorMap map0, map1, mapx;
};
thread_local int t_stall = 0;

// kSingle: single SMs, two CTAs each, buckets of up to 64 rows. kPair: CTA pairs, buckets of up to 256. kSplit: as kSingle with
// buckets of up to 32, where the tiles are too few for the GPU: a cluster of CTAs shares each tile's K, and its first CTA adds the
// parts, in order, out of its shared memory.
enum Form { kSingle = 0, kPair = 1, kSplit = 2 };
constexpr int kMaxParts = 4;

template <bool FP8, bool GATEUP, int FORM>
struct Shape {
  static constexpr int CG = FORM == kPair ? 2 : 1;
  // e4m3 in pairs: the MMA's M side is the routed rows and its N side 256 matrix rows (of them 128 of gate and 128 of up)
  static constexpr bool kRowsM = FP8 && CG == 2;
  static constexpr int kTok = FORM == kPair ? 256 : FORM == kSplit ? 32 : 64;   // routed rows of a bucket
  static constexpr int kTokStep = kRowsM ? 8 : 16 * CG;  // bucket sizes are multiples of this
  static constexpr int kEpiWarps = CG == 2 ? 8 : 4;
  static constexpr int kMmaWarp = kEpiWarps, kMatWarp = kEpiWarps + 1, kScaleWarp = kEpiWarps + 2;
  static constexpr int kScaleWarps = CG == 2 ? 2 : 1;
  static constexpr int kRowWarps = CG == 2 ? (FP8 ? 4 : 8) : 1, kRowWarp = CG == 2 ? 12 : 7;
  static constexpr int kThreads = 32 * (kRowWarp + kRowWarps);
  static constexpr int kBlocksPerSm = CG == 2 ? 1 : 2;
  static constexpr int kSub = CG == 2 && !FP8 ? 2 : 1;   // slabs of 128 bytes of K per stage
  static constexpr int kStages = FORM == kPair ? 6 / kSub : FORM == kSplit ? 5 : 4;
  static constexpr int kATile = 128 * 128;               // bytes: 128 matrix rows x 128 bytes of K
  static constexpr int kBTile = kTok / CG * 128;
  static constexpr int kSlab = FP8 ? 128 : 64;           // elements of K per slab
  static constexpr int kOuts = GATEUP ? 64 : 128;        // outputs per CTA and tile (of a pair: kOuts * CG)
  static constexpr int kBoxRows = GATEUP && !kRowsM ? 16 : 128;
  static constexpr int kVecs = GATEUP || kRowsM ? 2 : 1; // matrix scales per block of K: gate and up, or two blocks of 128 outputs
  static constexpr int kVecRows = kRowsM ? 128 : kTok;   // the routed rows that this CTA's epilogue sees
  static constexpr int kAccCols = kRowsM ? 128 : kTok;   // columns of an accumulator buffer
  static constexpr int kAccs = CG == 2 && !kRowsM ? 2 : 4;
  static constexpr int kScaleGroups = FP8 ? 4 : 0;       // ring of scales, four blocks of K to a group
  static constexpr int kScaleGroup = 4 * kVecRows * 4 + 32;   // [4][kVecRows] of the rows, [4][2] of the matrix blocks
  static constexpr int kOffA = 0;
  static constexpr int kOffB = kOffA + kStages * kSub * kATile;
  static constexpr int kOffScale = kOffB + kStages * kSub * kBTile;
  // bytes per epilogue warp: 16 columns x 32 + 16 or 8 x 64 + 16; or 32 rows of 16 f32
  static constexpr int kStage = kRowsM ? 32 * 17 * 4 : 16 * 48;
  static constexpr int kOffStage = kOffScale + kScaleGroups * kScaleGroup;
  static constexpr int kOffPairs = kOffStage + kEpiWarps * kStage;    // [kTiles][kTok] pair of each column
  static constexpr int kTiles = 3;                       // ring of tile descriptions
  static constexpr int kOffRows = kOffPairs + kTiles * kTok * 4;            // [kTiles][kTok] row of each column
  static constexpr int kOffTile = kOffRows + kTiles * kTok * 4;             // [kTiles] Tile
  static constexpr int kOffPref = kOffTile + kTiles * 16;                   // [E + 1] buckets before expert e, [E] pairs of it
  static constexpr int kOffBars = kOffPref + (2 * kMaxExperts + 4) * 4;
  static constexpr int kBytes = kOffBars + 320 + 1024;
  // the sums of the other CTAs of a split tile wait in the first one's idle operand stages
  static_assert(FORM != kSplit || (kMaxParts - 1) * kTok * 128 * 4 <= kStages * kSub * kATile, "sums of a split tile");
};

struct Tile {
  int e, n0, ncol, tok0;   // expert, first output of the CTA, columns (routed rows, rounded up), first pair of the bucket
};

// (a0, a1) += (x0 * s0, x1 * s1): the pairs stay in 64-bit registers, packed and unpacked they would cost more than the product
__device__ __forceinline__ void fma2(unsigned long long &a, uint32_t x0, uint32_t x1, unsigned long long s) {
  asm("{\n\t.reg .b64 x;\n\tmov.b64 x, {%1, %2};\n\tfma.rn.f32x2 %0, x, %3, %0;\n\t}" : "+l"(a) : "r"(x0), "r"(x1), "l"(s));
}

// whether the phase is complete, without waiting and without ordering: who acts on it fences or waits
__device__ __forceinline__ bool mbar_ask(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity));
  return ok != 0;
}
__device__ __forceinline__ unsigned long long twice(float f) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "r"(__float_as_uint(f)));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// four bytes to shared memory by an asynchronous copy; cp_async_arrive: an arrival at the barrier once this thread's copies are there
__device__ __forceinline__ void cp_async4(const void *dst_smem, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst_smem)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void l2_line(const void *at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }
// 32 bytes, one whole sector
__device__ __forceinline__ void store_sector(float *at, const float *v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
// two values in the 16-bit type `dtype`
__device__ __forceinline__ uint32_t pack16(int dtype, float a, float b) {
  if (dtype == KNJ_DT_BF16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&x);
  }
  const __half2 x = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&x);
}

// Columns of PER 16-bit outputs from shared memory to rows at any address: a lane per output, so that an instruction touches one run
// of each row. A function of its own: inlined at each of its dozen places it cost the aligned stores' code 4 us of 29 (2772 x 4096 x 288).
template <int PER>
__device__ __noinline__ void store_any(uint16_t *out, int64_t ldo, int n0, int N, const uint8_t *stg, int pitch, const int32_t *pairs) {
  const int lane = threadIdx.x & 31, j = lane % PER;
  int pr[8];
  uint16_t v[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {   // all reads in front of the stores, which the compiler keeps them behind
    const int col = c * (32 / PER) + lane / PER;
    pr[c] = pairs[col];
    v[c] = *reinterpret_cast<const uint16_t *>(stg + col * pitch + 2 * j);
  }
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (pr[c] != -1 && n0 + j < N) out[(pr[c] < 0 ? -2 - pr[c] : pr[c]) * ldo + n0 + j] = pr[c] < 0 ? 0 : v[c];
}

// The same for 32 rows of 16 f32 values, kRowPitch apart, of which each lane knows its own row's pair.
constexpr int kRowPitch = 17;
__device__ __noinline__ void store_rows_any(void *out, int dtype, int64_t ldo, int n, int N, const float *stg, int pr) {
  const int lane = threadIdx.x & 31, j = lane & 15;
  int q[16];
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 2 * i + (lane >> 4);
    q[i] = __shfl_sync(0xffffffffu, pr, r);
    v[i] = stg[r * kRowPitch + j];
  }
  if (n + j >= N) return;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (q[i] != -1) store_from_f32(out, dtype, (q[i] < 0 ? -2 - q[i] : q[i]) * ldo + n + j, v[i]);
}

template <bool FP8, bool GATEUP, int FORM>
__global__ void __launch_bounds__(Shape<FP8, GATEUP, FORM>::kThreads, Shape<FP8, GATEUP, FORM>::kBlocksPerSm)
    expert_tc_kernel(const __grid_constant__ GemmParams p) {
  using S = Shape<FP8, GATEUP, FORM>;
  constexpr int CG = S::CG;
  constexpr bool SPLIT = FORM == kSplit;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = warp_index();
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;                       // in the pair
  const int part = SPLIT ? (int)cluster_rank() : 0, parts = SPLIT ? 1 << p.part_bits : 1;   // of K

  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kOffBars);
  uint64_t *full = bars;                        // [kStages] operands of both CTAs landed (the even CTA's are used)
  uint64_t *empty = full + S::kStages;          // [kStages] the stage's products are done
  uint64_t *acc_full = empty + S::kStages;      // [kAccs] accumulator buffer complete
  uint64_t *acc_empty = acc_full + S::kAccs;    // [kAccs] accumulator buffer read (the even CTA's are used)
  uint64_t *sc_full = acc_empty + S::kAccs;     // [kScaleGroups]
  uint64_t *sc_empty = sc_full + 4;
  uint64_t *tile_full = sc_empty + 4;           // [kTiles] the tile's description is there
  uint64_t *tile_empty = tile_full + S::kTiles; // [kTiles] every warp is done with it
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tile_empty + S::kTiles);
  volatile int *s_fail = reinterpret_cast<volatile int *>(tmem_slot + 1);  // raised by the first wait that gives up
  int32_t *s_pair = reinterpret_cast<int32_t *>(smem + S::kOffPairs);
  int32_t *s_row = reinterpret_cast<int32_t *>(smem + S::kOffRows);
  int4 *s_tile = reinterpret_cast<int4 *>(smem + S::kOffTile);
  int32_t *s_pref = reinterpret_cast<int32_t *>(smem + S::kOffPref), *s_cnt = s_pref + kMaxExperts + 1;

  if (warp == S::kMatWarp && lane < 3) {   // the maps' first use would wait for them
    const CUtensorMap *m = lane == 0 ? &p.map0 : lane == 1 ? &p.mapx : &p.map1;
    if (lane < 2 || GATEUP) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  if (tid == 0) {
    // a barrier that the hook stalls expects an arrival too many
    const bool first_cta = blockIdx.x == 0, last_of_cluster = (int)blockIdx.x == CG * parts - 1;
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], i == 0 && p.stall == 2 && first_cta ? 2 : 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < S::kAccs; ++i) {
      mbar_init(&acc_full[i], i == 0 && ((p.stall == 1 && first_cta) || (p.stall == 3 && last_of_cluster)) ? 2 : 1);
      mbar_init(&acc_empty[i], CG * (S::kRowsM ? S::kEpiWarps / 2 : S::kEpiWarps));
    }
    for (int i = 0; i < S::kScaleGroups; ++i) {
      mbar_init(&sc_full[i], 32 * S::kScaleWarps);
      mbar_init(&sc_empty[i], S::kEpiWarps);
    }
    for (int i = 0; i < S::kTiles; ++i) {
      mbar_init(&tile_full[i], 1);
      mbar_init(&tile_empty[i], S::kEpiWarps + S::kRowWarps + (FP8 ? S::kScaleWarps : 1) + (rank == 0 ? 1 : 0));
    }
    *s_fail = 0;
    mbar_init_fence();
  }
  __syncwarp();
  if (CG == 2 || SPLIT) cluster_arrive();
  constexpr uint32_t kTmemCols = S::kAccs * S::kAccCols;
  if (warp == S::kMmaWarp) {
    tmem_alloc<CG>(tmem_slot, kTmemCols);
    tmem_relinquish<CG>();
  }
  if constexpr (FORM != kPair) {
    // The tables' first entries and the first rows start for L2 while the counts are read: found one after the other, they are three
    // latencies of HBM. A line that an earlier launch still writes is brought there for it.
    if (tid < 8 && 32 * tid < p.E && p.pair_idx) l2_line(p.pair_cnt + 32 * tid);
    if (tid < p.E && p.pair_idx) l2_line(p.pair_idx + tid * p.idx_stride);
    const int per = (p.K * (FP8 ? 1 : 2) + 127) / 128, line = blockIdx.x * S::kThreads + tid, row = line / per;
    if (row < p.n_rows) l2_line(p.x + row * p.x_row + (line - row * per) * 128);
  }
  grid_dep_wait();  // the tables and the rows come from earlier launches
  if (warp == 0) {
    // lane l counts the buckets of experts 8l .. 8l+7; a warp scan gives every expert its first bucket
    int cnts[8], nb = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = lane * 8 + j;
      int c = 0;
      if (e < p.E) c = p.pair_idx ? (int)max((int64_t)0, min((int64_t)p.pair_cnt[e], p.idx_stride)) : p.n_pairs;
      cnts[j] = c;
      nb += (c + S::kTok - 1) / S::kTok;
    }
    int incl = nb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int at = incl - nb;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s_pref[lane * 8 + j] = at;
      s_cnt[lane * 8 + j] = cnts[j];
      at += (cnts[j] + S::kTok - 1) / S::kTok;
    }
    if (lane == 31) s_pref[kMaxExperts] = at;
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || SPLIT) cluster_wait();  // the peer's barriers are initialised before anything arrives on them
  tc_fence_after();
  // what comes out of shared memory and feeds issuing loops goes through a shuffle: the compiler then knows it is the same in all
  // lanes and keeps it, and what is derived from it, in uniform registers
  auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
  const uint32_t tmem_base = same(*tmem_slot);

  const int nslab = (p.K + S::kSlab - 1) / S::kSlab;
  const int n_tiles = same(s_pref[kMaxExperts]) * p.m_tiles;   // at most 2^30: checked on the host
  // As many CTAs (pairs) as take part in whole rounds: of 1536 tiles on 296 CTAs, 256 take six each instead of 56 a sixth; the matrices
  // stream as fast and no round is left to a few (gate and up of 512 rows, bf16: 172 -> 158 us).
  const int bits = SPLIT ? p.part_bits : 0, k_lo = (part * nslab) >> bits, k_hi = ((part + 1) * nslab) >> bits;   // this CTA's slabs
  const int avail = (int)(gridDim.x / CG) >> bits, mine = (int)(blockIdx.x / CG) >> bits;
  int step = max(n_tiles, 1);
  if (n_tiles > avail) {   // the divisions of a few tiles would be a tenth of the time to the first copy
    const int rounds = (n_tiles + avail - 1) / avail;
    step = (n_tiles + rounds - 1) / rounds;
  }
  const int first = mine < step ? mine : n_tiles;
  auto tile_at = [&](int t, int &ntok) {   // by a whole warp
    int b = (int)__umulhi((uint32_t)t, p.m_inverse);   // t / m_tiles or one less
    if (t - b * p.m_tiles >= p.m_tiles) ++b;
    const int mt = t - b * p.m_tiles;
    // the last expert whose first bucket is not behind b: of 32 groups of eight experts, then of the eight
    const int g = 8 * (__popc(__ballot_sync(0xffffffffu, s_pref[8 * lane] <= b)) - 1);
    const int e = g + __popc(__ballot_sync(0xffffffffu, s_pref[g + (lane & 7)] <= b) & 0xffu) - 1;
    const int b0 = same(s_pref[e]), nb = same(s_pref[e + 1]) - b0, cnt = same(s_cnt[e]);
    // an expert's pairs are spread evenly over its buckets: 256 + 14 pairs would stream the matrix twice for 14
    const int per = ((nb == 1 ? cnt : (cnt + nb - 1) / nb) + S::kTokStep - 1) / S::kTokStep * S::kTokStep;
    Tile r;
    r.e = e;
    r.n0 = (mt * CG + (S::kRowsM ? 0 : (int)rank)) * S::kOuts;
    r.tok0 = (b - b0) * per;
    ntok = min(per, cnt - r.tok0);
    r.ncol = (ntok + S::kTokStep - 1) / S::kTokStep * S::kTokStep;
    return r;
  };
  // pair and row of column c of a tile: pair -1: none; pair -2 - p: p's row lies outside x, its output is zero
  auto pair_at = [&](const Tile &tl, int ntok, int c) {
    return c < ntok ? (p.pair_idx ? p.pair_idx[tl.e * p.idx_stride + tl.tok0 + c] : tl.tok0 + c) : -1;
  };
  bool ok = true;  // once false this thread skips all work and waits but still meets every barrier
  // e4m3 in pairs: the epilogue's sums take 128 registers a thread. 512 threads x 128 registers at launch = 2 x 128 x 208 + 2 x 128 x 48
  if constexpr (FP8 && CG == 2) {
    if (warp < S::kEpiWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
  }

  // A warp waits, and goes on or gives up, as a whole. The loops of the issuing warps stay warp-uniform around the elected thread's
  // instructions: with the loop inside the elected branch a stage took ~480 cycles to issue, so ~60 and the wait.
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (ok && !mbar_wait_for(bar, parity, p.wait_cycles, s_fail)) ok = false;
    ok = __all_sync(0xffffffffu, ok);
    return ok;
  };

  // kSplit: a tile ends for all warps of the cluster together: every sum is formed and the operand stages are idle; the sums of
  // parts 1, 2, .. are in the first CTA's stages; and, where another tile follows, they are read.
  auto split_syncs = [&](int t) { return t + step < n_tiles ? 3 : 2; };
  auto split_end = [&](int t) {   // for the warps that take no part in it
    if constexpr (SPLIT)
      for (int i = 0; i < split_syncs(t); ++i) cluster_sync_all();
  };
  auto split_give_up = [&](int t, int done) {   // from the tile t on, of whose syncs `done` have been met
    if constexpr (SPLIT) {
      if (ok) return;
      // the first CTA is there as long as a sync is left; without one nobody would read it
      const bool left = t < n_tiles && (done < split_syncs(t) || t + step < n_tiles);
      if (left && lane == 0) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(const_cast<int *>(s_fail), 0)), "r"(1) : "memory");
      __syncwarp();
      for (; t < n_tiles; t += step, done = 0)
        for (int i = done; i < split_syncs(t); ++i) cluster_sync_all();
    }
  };

  // What a tile is, is found once per CTA, by one warp (look, publish), and handed on through a ring to all others (tile_take,
  // tile_done). Finding takes some 2000 cycles a tile. In 16 bits a warp of its own does it, so that the matrix warp leaves no stage
  // empty meanwhile (4096 tokens gate+up 211 -> 202 us); in e4m3, where the scales take that warp, the matrix
  // warp does (in front of the scales 1024 tokens gate+up took 108 us instead of 98).
  int tslot = 0;
  uint32_t tpar = 0;
  auto tile_take = [&](Tile &tl) {
    if (!wait(&tile_full[tslot], tpar)) return false;
    const int4 v = s_tile[tslot];
    tl = Tile{same(v.x), same(v.y), same(v.z), same(v.w)};
    return true;
  };
  auto tile_done = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&tile_empty[tslot]);
    if (++tslot == S::kTiles) {
      tslot = 0;
      tpar ^= 1u;
    }
  };

  // The tables of a tile are read a tile before it is handed on: behind a full memory queue such a load takes microseconds.
  constexpr int kPairs = S::kTok / 32;
  Tile found{};
  int pr[kPairs], fslot = 0;
  uint32_t fpar = 1;
  auto look = [&](int t) {
    int ntok;
    found = tile_at(t, ntok);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) pr[j] = pair_at(found, ntok, lane + 32 * j);
  };
  auto publish = [&] {
    int row[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      row[j] = 0;
      if (pr[j] < 0 || pr[j] >= p.n_pairs) {
        pr[j] = -1;
      } else {
        row[j] = p.row_map ? p.row_map[pr[j]] : p.row_div == 1 ? pr[j] : pr[j] / p.row_div;
        if (row[j] < 0 || row[j] >= p.n_rows) {
          pr[j] = -2 - pr[j];
          row[j] = 0;
        }
      }
    }
    if (!wait(&tile_empty[fslot], fpar)) return;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      s_pair[fslot * S::kTok + lane + 32 * j] = pr[j];
      s_row[fslot * S::kTok + lane + 32 * j] = row[j];
    }
    if (lane == 0) s_tile[fslot] = make_int4(found.e, found.n0, found.ncol, found.tok0);
    __syncwarp();
    if (lane == 0) mbar_arrive(&tile_full[fslot]);
    if (++fslot == S::kTiles) {
      fslot = 0;
      fpar ^= 1u;
    }
  };

  if (warp < S::kEpiWarps) {
    // =========================== epilogue ===========================
    // Chunks of 32 columns are dealt to the warp groups in turn. A thread holds, of each 8 columns, two columns of the rows t/4,
    // t/4 + 8 and (half 1) 16 further of its warp's 32 rows: for gate and up, half 0 is gate and half 1 up of the same outputs.
    const int group = warp >> 2, quad = warp & 3;
    constexpr int kGroups = S::kEpiWarps / 4, kChunks = S::kTok / 32 / kGroups;
    const uint32_t lanes = tmem_base + ((uint32_t)(quad * 32) << 16);
    constexpr int kBufStep = S::kRowsM ? 2 : 1;   // lane = routed row: each group has two of the four buffers
    int buf = S::kRowsM ? group : 0, sg = 0;
    uint32_t par = 0, sg_par = 0;
    int t = first;
    [[maybe_unused]] int synced = 0;   // syncs of the running tile that are met
    for (; t < n_tiles; t += step, tile_done()) {
      Tile tl;
      if (!tile_take(tl)) break;
      const int ncol = tl.ncol;
      const int32_t *pairs = s_pair + tslot * S::kTok;
      const int n0 = tl.n0 + quad * (GATEUP ? 16 : 32);   // the warp's first output
      // 16 columns from c0 on, f32: the eight lanes of a column write one 32-byte sector of its row
      auto finish_f32 = [&](float *out, const float (&v)[2][8], int c0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int2 pp = *reinterpret_cast<const int2 *>(pairs + c0 + 8 * i + 2 * (lane & 3));
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const int pr = cc ? pp.y : pp.x;
            if (pr == -1) continue;
            float *row = out + (pr < 0 ? -2 - pr : pr) * p.ldo + n0 + (lane >> 2);
#pragma unroll
            for (int h = 0; h < (GATEUP ? 1 : 2); ++h)
#pragma unroll
              for (int rr = 0; rr < 2; ++rr) {
                float f = v[h][4 * i + 2 * rr + cc];
                if (pr < 0) f = 0.f;
                if (n0 + (lane >> 2) + 8 * rr + 16 * h < p.N) row[8 * rr + 16 * h] = f;
              }
          }
        }
      };
      // 16 bits: transposed through shared memory (stmatrix), so that whole sectors are written -- 16-byte pieces of a row from
      // two instructions made the stores of a tile of 256 columns take 28,000 cycles
      auto finish_16 = [&](const float (&v)[2][8], int c0) {
        constexpr int kRow = GATEUP ? 32 : 64, kPitch = kRow + 16;          // bytes of a column's outputs
        constexpr int kCols = GATEUP ? 16 : 8;                              // columns per store of the warp
        uint8_t *stg = smem + S::kOffStage + warp * S::kStage;
#pragma unroll
        for (int i = 0; i < 16 / kCols; ++i) {
          uint32_t m[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // matrix q: 8 outputs x 8 columns
            const int g = GATEUP ? q >> 1 : i, h = GATEUP ? 0 : q >> 1, rr = q & 1;
            m[q] = pack16(p.out_dtype, v[h][4 * g + 2 * rr], v[h][4 * g + 2 * rr + 1]);
          }
          const int q = lane >> 3, c = (GATEUP ? 8 * (q >> 1) : 0) + (lane & 7);
          __syncwarp();
          asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                           smem_u32(stg + c * kPitch + (GATEUP ? q & 1 : q) * 16)),
                       "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3])
                       : "memory");
          __syncwarp();
          uint16_t *out = static_cast<uint16_t *>(p.out);
          if (p.vec_out && n0 + kRow / 2 <= p.N) {
            const int col = lane / (kRow / 16), part = lane % (kRow / 16);
            uint4 u = *reinterpret_cast<const uint4 *>(stg + col * kPitch + part * 16);
            const int pr = pairs[c0 + i * kCols + col];
            if (pr < 0) u = make_uint4(0, 0, 0, 0);
            if (pr != -1) *reinterpret_cast<uint4 *>(out + (pr < 0 ? -2 - pr : pr) * p.ldo + n0 + 8 * part) = u;
          } else {
            store_any<kRow / 2>(out, p.ldo, n0, p.N, stg, kPitch, pairs + c0 + i * kCols);
          }
        }
      };
      auto finish = [&](const uint32_t (&lo)[8], const uint32_t (&hi)[8], int c0) {
        float v[2][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = __uint_as_float(lo[j]), b = __uint_as_float(hi[j]);
          v[0][j] = (GATEUP ? __fdividef(a, 1.0f + __expf(-a)) * b : a) * p.out_scale;
          v[1][j] = b * p.out_scale;
        }
        if (p.out_dtype == KNJ_DT_F32) finish_f32(static_cast<float *>(p.out), v, c0);
        else finish_16(v, c0);
      };
      auto load = [&](uint32_t (&lo)[8], uint32_t (&hi)[8], int col) {
        tmem_ld_16x16(lanes + buf * S::kAccCols + col, lo);
        tmem_ld_16x16(lanes + (16u << 16) + buf * S::kAccCols + col, hi);
      };
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) mbar_arrive_cluster(cluster_addr(&acc_empty[buf], 0));
          else mbar_arrive(&acc_empty[buf]);
        }
        buf += kBufStep;
        if (buf >= S::kAccs) {
          buf -= S::kAccs;
          par ^= 1u;
        }
      };
      // kSplit: this thread's sixteen sums of a step of 16 columns, to the first CTA or out of its stages
      auto part_at = [&](int from, int c, int i) { return (uint32_t)((((from - 1) * (S::kTok / 16) + c) * 4 + i) * 128 + tid) * 16u; };
      auto part_send = [&](const uint32_t (&lo)[8], const uint32_t (&hi)[8], int c) {
        const uint32_t base = cluster_addr(smem, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t *v = i < 2 ? lo + 4 * i : hi + 4 * (i - 2);
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + part_at(part, c, i)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                       : "memory");
        }
      };
      auto part_add = [&](uint32_t (&lo)[8], uint32_t (&hi)[8], int c) {
        for (int from = 1; from < parts; ++from)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = *reinterpret_cast<const float4 *>(smem + part_at(from, c, i));
            uint32_t *v = i < 2 ? lo + 4 * i : hi + 4 * (i - 2);
            v[0] = __float_as_uint(__uint_as_float(v[0]) + f.x);
            v[1] = __float_as_uint(__uint_as_float(v[1]) + f.y);
            v[2] = __float_as_uint(__uint_as_float(v[2]) + f.z);
            v[3] = __float_as_uint(__uint_as_float(v[3]) + f.w);
          }
      };
      // every thread of the warp: meets sync `i` of the tile; after the second, whether all parts are there
      auto part_sync = [&](int i) {
        fence_proxy_async();   // the stages go over between copies and ordinary accesses
        cluster_sync_all();
        synced = i;
        if (i == 2 && __any_sync(0xffffffffu, *s_fail != 0)) ok = false;
        return ok;
      };
      if constexpr (!FP8) {
        if (!wait(&acc_full[buf], par)) break;
        tc_fence_after();
        if constexpr (SPLIT) {
          // one chunk of 32 columns
          uint32_t r[4][8];
          load(r[0], r[1], 0);
          load(r[2], r[3], 16);
          tmem_ld_wait(r[0], r[1]);
          tmem_ld_wait(r[2], r[3]);
          part_sync(1);
          if (part != 0) {
            part_send(r[0], r[1], 0);
            if (ncol > 16) part_send(r[2], r[3], 1);
          }
          if (!part_sync(2)) break;
          if (part == 0) {
            part_add(r[0], r[1], 0);
            finish(r[0], r[1], 0);
            if (ncol > 16) {
              part_add(r[2], r[3], 1);
              finish(r[2], r[3], 16);
            }
          }
          if (split_syncs(t) == 3) part_sync(3);
          synced = 0;
        } else {
#pragma unroll 1
          for (int ch = group; ch * 32 < ncol; ch += kGroups) {
            uint32_t r[4][8];
            load(r[0], r[1], ch * 32);
            load(r[2], r[3], ch * 32 + 16);
            tmem_ld_wait(r[0], r[1]);
            tmem_ld_wait(r[2], r[3]);
            finish(r[0], r[1], ch * 32);
            finish(r[2], r[3], ch * 32 + 16);
          }
        }
        release();
      } else if constexpr (S::kRowsM) {
        // Lane = routed row, so that a block's scale is one register and the loads take the 32-lane form, 935 bytes a cycle; with lane
        // = matrix row every thread has to fetch a scale for each of its columns, 1024 cycles of shared memory a block, or load in
        // the 16-lane form, 524 cycles of tensor memory (the products take 512). A product is issued as two of 128 columns, 64 rows
        // of each CTA's matrix tile, into buffers of their own: group g reads the buffers of half g, outputs 64 g .. + 63 of gate and
        // of up, or of both blocks of 128 outputs. Whole products in two buffers left the tensor core waiting for the hand-offs, which
        // still bound it: 8192 x 4096 x 4096 154 us, tensor pipe 41 % busy (copies and products alone: 101 us). The loads run one step
        // of 16 columns ahead of the sums, across blocks of K too, and whether the next buffer is complete is asked two steps before it
        // is needed; the next block's scales are read after the first step (4096 tokens gate+up 203 -> 196 us; at the block's start, or
        // late in it, 203 to 208). Sixteen warps with 64 sums a thread and one load under way each took 175 us.
        constexpr int kSteps = 8;
        auto col_of = [&](int c) { return c * 16; };
        const int local = quad * 32 + lane;
        unsigned long long acc[kSteps][8];   // pairs of f32 sums
        uint32_t r[2][16];
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[c][j] = 0ull;
        unsigned long long next0 = 0, next1 = 0;
        auto scales = [&](int ks) {   // of the next block, read while this one's loads are under way
          const float *sc = reinterpret_cast<const float *>(smem + S::kOffScale + sg * S::kScaleGroup);
          const float sx = sc[(ks & 3) * S::kVecRows + local];
          const float2 sw = *reinterpret_cast<const float2 *>(sc + 4 * S::kVecRows + 2 * (ks & 3));
          next0 = twice(sx * sw.x);
          next1 = twice(sx * sw.y);
        };
        auto scales_done = [&] {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_empty[sg]);
          if (++sg == S::kScaleGroups) {
            sg = 0;
            sg_par ^= 1u;
          }
        };
        if (!wait(&sc_full[sg], sg_par)) break;
        scales(0);
        if (!wait(&acc_full[buf], par)) break;
        tc_fence_after();
        tmem_ld_32x16(lanes + buf * S::kAccCols + col_of(0), r[0]);
        for (int ks = 0; ks < nslab; ++ks) {
          const unsigned long long s0 = next0, s1 = next1;
          bool ready = false;
#pragma unroll
          for (int c = 0; c < kSteps; ++c) {
            tmem_ld_wait(r[c & 1]);
            if (c + 2 == kSteps) {
              const int nb = buf + kBufStep < S::kAccs ? buf + kBufStep : buf + kBufStep - S::kAccs;
              ready = mbar_ask(&acc_full[nb], nb < buf ? par ^ 1u : par);
            }
            if (c + 1 < kSteps) {
              tmem_ld_32x16(lanes + buf * S::kAccCols + col_of(c + 1), r[(c + 1) & 1]);
            } else {
              release();
              if (ks + 1 < nslab) {
                if (!__all_sync(0xffffffffu, ready) && !wait(&acc_full[buf], par)) break;
                tc_fence_after();
                tmem_ld_32x16(lanes + buf * S::kAccCols + col_of(0), r[0]);
              }
            }
            if (c == 1 && ks + 1 < nslab) {
              if ((ks & 3) == 3) {
                scales_done();
                if (!wait(&sc_full[sg], sg_par)) break;
              }
              scales(ks + 1);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) fma2(acc[c][j], r[c & 1][2 * j], r[c & 1][2 * j + 1], c >= 4 ? s1 : s0);
          }
          if (!ok) break;
        }
        if (!ok) {
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");   // a load may be under way, and tensor memory is freed soon
          break;
        }
        scales_done();
        const int n_cta = ncol / CG;
        const int pr = local < n_cta ? pairs[(int)rank * n_cta + local] : -1;
        const bool none = pr < -1;
        const int64_t row = (int64_t)(none ? -2 - pr : pr) * p.ldo;
        auto value = [&](int c, int j) {   // output 16 c + j of this thread's row
          const unsigned long long w = acc[c][j >> 1];
          return __uint_as_float((uint32_t)((j & 1) ? w >> 32 : w));
        };
        constexpr int kOut16 = GATEUP ? 4 : 8;   // runs of 16 outputs
#pragma unroll
        for (int c = 0; c < kOut16; ++c) {
          float f[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            f[j] = value(c, j);
            if constexpr (GATEUP) f[j] = __fdividef(f[j], 1.0f + __expf(-f[j])) * value(c + 4, j);
            f[j] = none ? 0.f : f[j] * p.out_scale;
          }
          const int n = tl.n0 + group * 64 + (c & 3) * 16 + (c >> 2) * 128;
          if (n >= p.N) continue;
          if (p.vec_out && n + 16 <= p.N) {
            if (pr == -1) continue;
            if (p.out_dtype == KNJ_DT_F32) {
              store_sector(static_cast<float *>(p.out) + row + n, f);
              store_sector(static_cast<float *>(p.out) + row + n + 8, f + 8);
            } else {
              float w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) w[j] = __uint_as_float(pack16(p.out_dtype, f[2 * j], f[2 * j + 1]));
              store_sector(reinterpret_cast<float *>(static_cast<uint16_t *>(p.out) + row + n), w);
            }
          } else {
            float *stg = reinterpret_cast<float *>(smem + S::kOffStage + warp * S::kStage);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) stg[lane * kRowPitch + j] = f[j];
            __syncwarp();
            store_rows_any(p.out, p.out_dtype, p.ldo, n, p.N, stg, pr);
          }
        }
      } else {
        // One straight run of code for each number of chunks: with a branch around every chunk their loads could not be started in
        // front of each other's sums.
        auto blocks = [&](auto chunks) {
          constexpr int kSteps = 2 * decltype(chunks)::value;   // of 16 columns
          auto col_of = [&](int c) { return c * 16; };
          unsigned long long acc[kSteps][2][4];   // pairs of f32 sums: steps, halves, (8 columns, rows)
#pragma unroll
          for (int c = 0; c < kSteps; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[c][h][j] = 0ull;
          for (int ks = 0; ks < k_hi - k_lo; ++ks) {
            if ((ks & 3) == 0) wait(&sc_full[sg], sg_par);
            if (!wait(&acc_full[buf], par)) return;
            tc_fence_after();
            const float *sg_at = reinterpret_cast<const float *>(smem + S::kOffScale + sg * S::kScaleGroup);
            const float *sc = sg_at + (ks & 3) * S::kVecRows + 2 * (lane & 3);
            const float2 sw = *reinterpret_cast<const float2 *>(sg_at + 4 * S::kVecRows + 2 * (ks & 3));
            const unsigned long long w0 = twice(sw.x), w1 = twice(sw.y);
            uint32_t r[2][2][8];
            load(r[0][0], r[0][1], col_of(0));
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
              tmem_ld_wait(r[c & 1][0], r[c & 1][1]);
              if (c + 1 < kSteps) load(r[(c + 1) & 1][0], r[(c + 1) & 1][1], col_of(c + 1));
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const unsigned long long sx = *reinterpret_cast<const unsigned long long *>(sc + col_of(c) + 8 * i);
                const unsigned long long s0 = mul2(sx, w0), s1 = GATEUP ? mul2(sx, w1) : s0;
#pragma unroll
                for (int rr = 0; rr < 2; ++rr) {
                  fma2(acc[c][0][2 * i + rr], r[c & 1][0][4 * i + 2 * rr], r[c & 1][0][4 * i + 2 * rr + 1], s0);
                  fma2(acc[c][1][2 * i + rr], r[c & 1][1][4 * i + 2 * rr], r[c & 1][1][4 * i + 2 * rr + 1], s1);
                }
              }
            }
            release();
            if ((ks & 3) == 3 || ks + 1 == k_hi - k_lo) {
              if (lane == 0) mbar_arrive(&sc_empty[sg]);   // behind release()'s __syncwarp
              if (++sg == S::kScaleGroups) {
                sg = 0;
                sg_par ^= 1u;
              }
            }
          }
          if constexpr (SPLIT) {
            uint32_t v[kSteps][2][8];
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                v[c][0][j] = (uint32_t)(acc[c][0][j >> 1] >> (32 * (j & 1)));
                v[c][1][j] = (uint32_t)(acc[c][1][j >> 1] >> (32 * (j & 1)));
              }
            part_sync(1);
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
              if (part != 0 && 16 * c < ncol) part_send(v[c][0], v[c][1], c);
            if (!part_sync(2)) return;
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
              if (part == 0 && 16 * c < ncol) {
                part_add(v[c][0], v[c][1], c);
                finish(v[c][0], v[c][1], 16 * c);
              }
            if (split_syncs(t) == 3) part_sync(3);
            synced = 0;
          } else {
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
              uint32_t lo[8], hi[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                lo[j] = (uint32_t)(acc[c][0][j >> 1] >> (32 * (j & 1)));
                hi[j] = (uint32_t)(acc[c][1][j >> 1] >> (32 * (j & 1)));
              }
              finish(lo, hi, col_of(c));
            }
          }
        };
        static_assert(kGroups == 1 && kChunks <= 2, "one case for each number of chunks, and no bucket is empty");
        if (kChunks == 1 || ncol <= 32) blocks(std::integral_constant<int, 1>{});
        else if constexpr (kChunks > 1) blocks(std::integral_constant<int, 2>{});
        if (!ok) break;
      }
    }
    // a wait gave up: NaN for what this warp has not stored, its tile at that moment and those behind it
    split_give_up(t, synced);
    for (; !ok && part == 0 && t < n_tiles; t += step) {
      int ntok;
      const Tile tl = tile_at(t, ntok);
      if constexpr (S::kRowsM) {
        const int n_cta = tl.ncol / CG, local = quad * 32 + lane, pr = local < n_cta ? pair_at(tl, ntok, (int)rank * n_cta + local) : -1;
        for (int j = 0; j < S::kOuts; ++j) {
          const int n = tl.n0 + group * 64 + (j & 63) + (j >> 6) * 128;
          if (n < p.N && pr >= 0 && pr < p.n_pairs) store_from_f32(p.out, p.out_dtype, pr * p.ldo + n, __int_as_float(0x7fffffff));
        }
      } else {
        const int n = tl.n0 + quad * (GATEUP ? 16 : 32) + lane;
        for (int c = 0; c < ntok; ++c) {
          if ((c / 32) % kGroups != group || n >= p.N || lane >= (GATEUP ? 16 : 32)) continue;
          const int pr = pair_at(tl, ntok, c);
          if (pr >= 0 && pr < p.n_pairs) store_from_f32(p.out, p.out_dtype, pr * p.ldo + n, __int_as_float(0x7fffffff));
        }
      }
    }
  } else if (warp == S::kMmaWarp) {
    // =========================== MMA issue ===========================
    if (rank == 0) {
      const uint64_t a_desc0 = smem_desc_sw128(smem_u32(smem + S::kOffA)), b_desc0 = smem_desc_sw128(smem_u32(smem + S::kOffB));
      int st = 0, buf = 0;
      uint32_t par = 0, acc_par = 1;  // a fresh barrier passes a wait for parity 1
      int t = first;
      for (; t < n_tiles; tile_done(), split_end(t), t += step) {
        Tile tl;
        if (!tile_take(tl)) break;
        const uint32_t idesc = instr_desc_f16(128 * CG, S::kRowsM ? 128 : tl.ncol) | p.idesc_format;
        for (int ks = k_lo; ks < k_hi; ks += S::kSub) {
          if (!S::kRowsM && (FP8 || ks == k_lo) && !wait(&acc_empty[buf], acc_par)) break;
          if (!wait(&full[st], par)) break;
          tc_fence_after();
          const uint64_t mat = a_desc0 + (uint32_t)(st * S::kSub * S::kATile) / 16, rows = b_desc0 + (uint32_t)(st * S::kSub * S::kBTile) / 16;
          auto commit = [&](uint64_t *bar) {
            if (CG == 2) tc_commit_pair(smem_u32(bar));
            else tc_commit_addr<CG>(smem_u32(bar));
          };
          auto next_buf = [&] {
            if (++buf == S::kAccs) { buf = 0; acc_par ^= 1u; }
          };
          if constexpr (S::kRowsM) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!wait(&acc_empty[buf], acc_par)) break;
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma<FP8, CG>(tmem_base + buf * S::kAccCols, rows + 2 * k, mat + h * 512 + 2 * k, idesc, k > 0 ? 1u : 0u);
                commit(&acc_full[buf]);
                if (h == 1) commit(&empty[st]);
              }
              __syncwarp();
              next_buf();
            }
            if (!ok) break;
          } else {
            const bool last = FP8 || ks + S::kSub >= k_hi;
            if (elect_one()) {
#pragma unroll
              for (int u = 0; u < S::kSub; ++u) {
                if (u > 0 && ks + u >= k_hi) break;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  tc_mma<FP8, CG>(tmem_base + buf * S::kAccCols, mat + u * (S::kATile / 16) + 2 * k, rows + u * (S::kBTile / 16) + 2 * k, idesc,
                               (u > 0 || k > 0 || (!FP8 && ks > k_lo)) ? 1u : 0u);
              }
              commit(&empty[st]);
              if (last) commit(&acc_full[buf]);
            }
            __syncwarp();
            if (last) next_buf();
          }
          if (++st == S::kStages) { st = 0; par ^= 1u; }
        }
        if (!ok) break;
      }
      split_give_up(t, 0);
    }
  } else if (warp == S::kMatWarp) {
    // =========================== matrix rows (e4m3: and tiles) ===========================
    int st = 0;
    uint32_t par = 1;
    // one stage of the matrix, and the announcement of the bytes of both CTAs' copies into it
    auto issue = [&](const Tile &tl, int ks) {
      const int y = tl.e * p.N + tl.n0 + (S::kRowsM && !GATEUP ? 128 * (int)rank : 0);
      const uint32_t bar = CG == 2 ? cluster_addr(&full[st], 0) : smem_u32(&full[st]);
      if (elect_one()) {
        const uint32_t bytes = (uint32_t)(CG * S::kATile + (p.dense ? CG * S::kBTile : tl.ncol * 128));
        if (rank == 0) mbar_expect_tx(&full[st], bytes * min(S::kSub, k_hi - ks));
#pragma unroll
        for (int u = 0; u < S::kSub; ++u) {
          if (u > 0 && ks + u >= k_hi) break;
          const uint32_t dst = smem_u32(smem + S::kOffA + (st * S::kSub + u) * S::kATile);
          const int x = (ks + u) * S::kSlab;
          if (S::kRowsM) {
            tma_load_box<CG>(dst, GATEUP && rank ? &p.map1 : &p.map0, x, y, bar);
          } else if (GATEUP) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              tma_load_box<CG>(dst + j * 4096, &p.map0, x, y + 16 * j, bar);
              tma_load_box<CG>(dst + j * 4096 + 2048, &p.map1, x, y + 16 * j, bar);
            }
          } else {
            tma_load_box<CG>(dst, &p.map0, x, y, bar);
          }
        }
      }
      __syncwarp();
      if (++st == S::kStages) { st = 0; par ^= 1u; }
    };
    int ahead = k_lo;
    if (first < n_tiles) {
      int ntok;
      if constexpr (FP8) look(first);
      else found = tile_at(first, ntok);
      // the first stages are empty and the matrix depends on no table entry: it travels while those are read
      for (int i = 0; i < S::kStages && ahead < k_hi; ++i, ahead += S::kSub) issue(found, ahead);
    }
    int t = first;
    for (; t < n_tiles; split_end(t), t += step) {
      Tile tl = found;
      if constexpr (FP8) {
        publish();
        if (!ok) break;
        if (t + step < n_tiles) look(t + step);
      } else {
        if (!tile_take(tl)) break;
      }
      for (int ks = ahead; ks < k_hi; ks += S::kSub) {
        if (!wait(&empty[st], par)) break;
        issue(tl, ks);
      }
      ahead = k_lo;
      if (!ok) break;
      if (!FP8) tile_done();
    }
    split_give_up(t, 0);
  } else if (!FP8 && warp == S::kScaleWarp) {
    // =========================== tiles ===========================
    int t = first;
    if (first < n_tiles) {
      look(first);
      publish();
    }
    for (; ok && t < n_tiles; split_end(t), t += step) {
      if (t + step < n_tiles) {
        look(t + step);
        publish();
        if (!ok) break;
      }
    }
    split_give_up(t, 0);
  } else if (FP8 && warp >= S::kScaleWarp && warp < S::kScaleWarp + S::kScaleWarps) {
    // =========================== scales ===========================
    // Asynchronous copies of four bytes, four blocks of K to a group: this warp never waits for a load, only for a free group of the
    // ring. (Loads into registers a group ahead were as fast where HBM or L2 is quiet, 8192 x 4096 x 4096: 166 and 171 us.)
    constexpr int kPer = S::kVecRows / 32 / S::kScaleWarps;   // rows per lane
    const int nb_n = (p.N + 127) / 128, c0 = (warp - S::kScaleWarp) * 32 * kPer + lane;
    int sg = 0;
    uint32_t par = 1;
    int t = first;
    for (; t < n_tiles; tile_done(), split_end(t), t += step) {
      Tile tl;
      if (!tile_take(tl)) break;
      // scales of block `blk` of matrix 0 and, for two, of matrix 1 or of the next block; behind the last output there is no block:
      // any one's scales do. Lanes 0..3: the first, lanes 4..7 the second, block of K lane % 4.
      const int blk = min(tl.n0 / 128, nb_n - 1), second = lane >> 2 & 1;
      const float *ws = (GATEUP && second ? p.ws1 : p.ws0) + ((int64_t)tl.e * nb_n + (GATEUP || !second ? blk : min(blk + 1, nb_n - 1))) * nslab + (lane & 3);
      const int n_cta = tl.ncol / CG;
      const float *xs[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int c = c0 + 32 * j;   // of the bucket, or in lane = row form of this CTA's part of it
        const int at = S::kRowsM ? (c < n_cta ? (int)rank * n_cta + c : 0) : c;
        xs[j] = p.xs + (int64_t)s_row[tslot * S::kTok + at] * nslab;
      }
      for (int k0 = k_lo; k0 < k_hi; k0 += 4) {
        if (!wait(&sc_empty[sg], par)) break;
        float *dst = reinterpret_cast<float *>(smem + S::kOffScale + sg * S::kScaleGroup);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k0 + i < k_hi) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) cp_async4(dst + i * S::kVecRows + c0 + 32 * j, xs[j] + k0 + i);
          }
        if (warp == S::kScaleWarp && lane < 4 * S::kVecs && k0 + (lane & 3) < k_hi) cp_async4(dst + 4 * S::kVecRows + 2 * (lane & 3) + second, ws + k0);
        cp_async_arrive(&sc_full[sg]);
        if (++sg == S::kScaleGroups) {
          sg = 0;
          par ^= 1u;
        }
      }
      if (!ok) break;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    split_give_up(t, 0);
  } else if (warp >= S::kRowWarp && warp < S::kRowWarp + S::kRowWarps) {
    // =========================== routed rows ===========================
    const int w = warp - S::kRowWarp;
    constexpr int kQuads = S::kTok / CG / (4 * S::kRowWarps);   // copies of four rows per warp and slab
    int st = 0;
    uint32_t par = 1;
    int t = first;
    for (; t < n_tiles; tile_done(), split_end(t), t += step) {
      Tile tl;
      if (!tile_take(tl)) break;
      const int n_cta = tl.ncol / CG;
      int4 rows[kQuads];
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const int r = 4 * (w + S::kRowWarps * q);
        rows[q] = *reinterpret_cast<const int4 *>(s_row + tslot * S::kTok + (r < n_cta ? (int)rank * n_cta + r : 0));
      }
      for (int ks = k_lo; ks < k_hi; ks += S::kSub) {
        if (!wait(&empty[st], par)) break;
        const uint32_t bar = CG == 2 ? cluster_addr(&full[st], 0) : smem_u32(&full[st]);
        if (elect_one()) {
#pragma unroll
          for (int u = 0; u < S::kSub; ++u) {
            if (u > 0 && ks + u >= k_hi) break;
            const uint32_t dst = smem_u32(smem + S::kOffB + (st * S::kSub + u) * S::kBTile);
            const int x = (ks + u) * S::kSlab;
            if (p.dense) {
              if (w == 0) tma_load_box<CG>(dst, &p.mapx, x, tl.tok0 + (int)rank * n_cta, bar);
            } else if constexpr (S::kRowWarps == 1) {
              // buckets are multiples of 16 rows: one branch for four copies (with one for each, skipped or not, a stage took this
              // warp 1000 cycles whatever the bucket)
#pragma unroll
              for (int q = 0; q < kQuads; q += 4) {
                if (4 * q >= n_cta) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) tma_gather4<CG>(dst + (q + i) * 512, &p.mapx, x, rows[q + i], bar);
              }
            } else {
#pragma unroll
              for (int q = 0; q < kQuads; ++q) {
                const int r = 4 * (w + S::kRowWarps * q);
                if (r < n_cta) tma_gather4<CG>(dst + r * 128, &p.mapx, x, rows[q], bar);
              }
            }
          }
        }
        __syncwarp();
        if (++st == S::kStages) { st = 0; par ^= 1u; }
      }
      if (!ok) break;
    }
    split_give_up(t, 0);
  }
  static_assert(!SPLIT || S::kThreads == 32 * (S::kEpiWarps + 4), "every warp of a split tile meets its syncs");

  if (!ok) {
    // a wait gave up: let the copies that are in flight land before this CTA's shared memory is handed on
    if (p.status) atomicExch(p.status, 1);
    const long long t0 = clock64();
    while (clock64() - t0 < (1ll << 20)) __nanosleep(1000);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // a CTA of a pair may neither free tensor memory nor leave while the peer still uses its shared memory or its barriers
  if (CG == 2) cluster_sync_all();
  if (warp == S::kMmaWarp) tmem_dealloc<CG>(tmem_base, kTmemCols);
}

int g_form = 0;  // 0 = by the rule below, 1 = single SMs, 2 = pairs, 3 = K split over a cluster (knj_expert_tc_form)

struct Operands {
  const void *x, *w0, *w1;
  int64_t ldx;
  bool fp8;
};

// the tiles that these pairs can make; a table that names pairs more than once makes more, which the same grid walks over
template <class S>
int64_t most_tiles(const GemmParams &p) {
  const int64_t rows = S::kOuts * S::CG, buckets = p.dense ? (p.n_pairs + S::kTok - 1) / S::kTok : p.n_pairs / S::kTok + (p.E < p.n_pairs ? p.E : p.n_pairs);
  return buckets * ((p.N + rows - 1) / rows);
}

template <bool FP8, bool GATEUP, int FORM>
int launch_form(GemmParams p, const Operands &o, cudaStream_t st) {
  using S = Shape<FP8, GATEUP, FORM>;
  constexpr int CG = S::CG;
  int dev = 0;
  KNJ_CUDA(cudaGetDevice(&dev));
  auto kern = expert_tc_kernel<FP8, GATEUP, FORM>;
  static bool opted[64] = {false};
  if (dev >= 0 && dev < 64 && !opted[dev]) {
    KNJ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    opted[dev] = true;
  }
  constexpr int esz = FP8 ? 1 : 2;
  const uint64_t w_rows = (uint64_t)p.E * p.N;
  int rc = make_operand_tensor_map(&p.map0, o.w0, esz, p.K, p.K, w_rows, S::kBoxRows);
  if (!rc && GATEUP) rc = make_operand_tensor_map(&p.map1, o.w1, esz, p.K, p.K, w_rows, S::kBoxRows);
  if (!rc) rc = make_operand_tensor_map(&p.mapx, o.x, esz, p.K, o.ldx, p.n_rows, p.dense ? S::kTok / CG : 1);
  if (rc) return rc;
  p.m_tiles = (p.N + S::kOuts * CG - 1) / (S::kOuts * CG);
  p.m_inverse = (uint32_t)((1ull << 32) / p.m_tiles - (p.m_tiles == 1));
  const int out_esz = p.out_dtype == KNJ_DT_F32 ? 4 : 2, unit = S::kRowsM ? 32 : 16;
  p.vec_out = reinterpret_cast<uintptr_t>(p.out) % unit == 0 && p.ldo * out_esz % unit == 0;
  p.stall = t_stall;
  p.wait_cycles = decode_wait_cycles();
  const int64_t most = p.pair_idx ? p.E * ((p.idx_stride + S::kTok - 1) / S::kTok) : (p.n_pairs + S::kTok - 1) / S::kTok;
  KNJ_REQUIRE(most * p.m_tiles <= (1ll << 30) && (int64_t)w_rows + 256 < (1ll << 31), "expert product: %lld buckets of %d row tiles are too many",
              (long long)most, p.m_tiles);
  const int64_t tiles = most_tiles<S>(p), cap = (int64_t)sm_count() * S::kBlocksPerSm / (CG << p.part_bits);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((tiles < cap ? tiles : cap) * (CG << p.part_bits)));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG << p.part_bits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_chain_overlap ? 2 : 1;
  KNJ_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return launch_status("expert_tc_kernel");
}

template <bool FP8, bool GATEUP>
int launch_rule(GemmParams p, const Operands &o, cudaStream_t st) {
  const int64_t experts = p.E < p.n_pairs ? p.E : p.n_pairs;
  const int nslab = (p.K + Shape<FP8, GATEUP, kSplit>::kSlab - 1) / Shape<FP8, GATEUP, kSplit>::kSlab;
  // K is split where even the smallest tiles leave half of the CTAs' places free, into parts of two slabs or more: one row times
  // 4096 x 4096 e4m3, rows in 16 bits, 15.1 -> 9.7 us, 64 rows 19.1 -> 13.0 (parts of one slab, K = 512, cost 2 us more than none). Clusters of two and
  // four fill a GPC's SMs; of clusters of three, 96 did not fit at once (22.6 us where two took 16.4).
  const int64_t places = 2ll * sm_count() / most_tiles<Shape<FP8, GATEUP, kSplit>>(p);
  int bits = places >= kMaxParts ? 2 : places >= 2 ? 1 : 0;
  while (bits > 0 && (2 << bits) > nslab) --bits;
  p.part_bits = 0;
  if (g_form == 3 || (g_form == 0 && bits > 0)) {
    p.part_bits = bits;
    return launch_form<FP8, GATEUP, kSplit>(p, o, st);
  }
  // Single SMs or pairs, us each, by (rows per expert; experts), matrices from HBM. 16 bits, gate and up, hidden 2048, ffn 768: 81, 80
  // (1; 128), 132, 129 (32; 128), 134, 131 (32, Zipf; 128), 187, 146 (128; 128), 336, 205 (256; 128); hidden 1024, ffn 512: 15.3, 15.4
  // (1; 32), 17.4, 17.6 (32; 32), 19.3, 18.4 (64; 32) -- pairs where the buckets fill them or the tiles take four rounds of pairs anyway.
  // e4m3, whose pairs always multiply 256 rows and whose stores no product overlaps: 49, 85 (1; 128), 77, 130 (32; 128), 95, 139 (64;
  // 128), 149, 133 (128; 128), 282, 191 (256; 128), down 104, 97 (128; 128); dense with its rows' quantiser, rows x outputs x K:
  // 4096 x 4096 x 4096 155, 99, 1024 x 4096 x 1024 (64 tiles of pairs) 18.1, 14.8, 1024 x 2048 x 2048 (32 tiles) 17.5, 18.7,
  // 2048 x 4096 x 512 21.4, 17.2, 2772 x 4091 x 288 (outputs at any address) 38, 49.
  const int64_t pair_tiles = most_tiles<Shape<FP8, GATEUP, kPair>>(p), round = sm_count() / 2;
  bool pairs = FP8 ? p.n_pairs >= 128 * experts && nslab >= 4 && 4 * pair_tiles >= 3 * round : p.n_pairs > 32 * experts || pair_tiles >= 4 * round;
  if (g_form) pairs = g_form == 2;
  return pairs ? launch_form<FP8, GATEUP, kPair>(p, o, st) : launch_form<FP8, GATEUP, kSingle>(p, o, st);
}
template <bool GATEUP>
int launch_gemm(const GemmParams &p, const Operands &o, cudaStream_t st) {
  return o.fp8 ? launch_rule<true, GATEUP>(p, o, st) : launch_rule<false, GATEUP>(p, o, st);
}

}  // namespace

namespace knj {
int expert_product_check(const knj_expert_gemm_args *a, bool gateup, const char *who) {
  KNJ_REQUIRE(a, "%s: null argument block", who);
  KNJ_REQUIRE(a->n_pairs >= 0 && a->n_rows >= 0 && a->N > 0 && a->K > 0 && a->n_experts >= 1 && a->n_experts <= kMaxExperts, "%s: bad sizes", who);
  if (a->n_pairs == 0) return KNJ_OK;
  KNJ_REQUIRE(a->n_pairs <= kMaxPairs && a->idx_stride <= kMaxPairs, "%s: tables of more than 2^30 pairs", who);
  KNJ_REQUIRE(a->n_rows >= 1, "%s: pairs without a row of x", who);
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
}  // namespace knj

namespace {

int run_expert(const knj_expert_gemm_args *a, bool gateup, const char *who, knj_stream_t s) {
  const int rc = expert_product_check(a, gateup, who);
  if (rc || a->n_pairs == 0) return rc;
  GemmParams p{};
  p.xs = a->x_scale; p.ws0 = a->w0_scale; p.ws1 = a->w1_scale; p.pair_idx = a->pair_idx; p.pair_cnt = a->pair_cnt; p.row_map = a->row_map;
  p.out = a->out; p.status = a->status; p.ldo = a->ldo; p.idx_stride = a->idx_stride; p.out_dtype = a->out_dtype; p.N = a->N; p.K = a->K;
  p.E = a->n_experts; p.row_div = a->row_div > 0 ? a->row_div : 1; p.n_rows = a->n_rows; p.n_pairs = a->n_pairs; p.out_scale = a->out_scale;
  p.idesc_format = a->w_dtype == KNJ_DT_BF16 ? (1u << 7) | (1u << 10) : 0u;
  p.x = static_cast<const uint8_t *>(a->x); p.x_row = a->ldx * (a->w_dtype == KNJ_DT_E4M3 ? 1 : 2);
  const Operands o{a->x, a->w0, a->w1, a->ldx, a->w_dtype == KNJ_DT_E4M3};
  return gateup ? launch_gemm<true>(p, o, as_stream(s)) : launch_gemm<false>(p, o, as_stream(s));
}

inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

extern "C" {

int knj_expert_gateup_launch(const knj_expert_gemm_args *a, knj_stream_t s) { return run_expert(a, true, "knj_expert_gateup", s); }

int knj_expert_proj_launch(const knj_expert_gemm_args *a, knj_stream_t s) { return run_expert(a, false, "knj_expert_proj", s); }

void knj_expert_tc_test_stall(int what) { t_stall = what >= 1 && what <= 3 ? what : 0; }

void knj_expert_tc_form(int form) { g_form = form >= 1 && form <= 3 ? form : 0; }

size_t knj_fp8_matmul_workspace_bytes(int m, int n_in) {
  if (m <= 0 || n_in <= 0) return 0;
  return up256((size_t)m * n_in) + up256((size_t)m * ((n_in + 127) / 128) * 4);
}

int knj_fp8_matmul_launch(const void *W, const float *W_scale, int n_in, int n_out, const void *x, int x_dtype, int64_t ldx, int m, void *y,
                          int y_dtype, int64_t ldy, void *workspace, size_t workspace_bytes, int *status, knj_stream_t s) {
  KNJ_REQUIRE(m >= 0 && n_in > 0 && n_out > 0, "knj_fp8_matmul: bad sizes");
  if (m == 0) return KNJ_OK;
  KNJ_REQUIRE(W && W_scale && x && y, "knj_fp8_matmul: null pointer");
  KNJ_REQUIRE(m <= kMaxPairs, "knj_fp8_matmul: more than 2^30 rows");
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
  p.x = q; p.x_row = n_in; p.xs = qs; p.ws0 = W_scale; p.out = y; p.status = status; p.ldo = ldy; p.out_dtype = y_dtype; p.N = n_out; p.K = n_in; p.E = 1;
  p.row_div = 1; p.n_rows = m; p.n_pairs = m; p.out_scale = 1.0f; p.dense = 1;
  return launch_gemm<false>(p, Operands{q, W, nullptr, n_in, true}, as_stream(s));
}

}  // extern "C"
