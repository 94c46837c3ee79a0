// knj_expert_tc.cu -- products of routed rows with expert matrices held in bf16, fp16 or e4m3 (one scale for each block of
// 128 x 128), grouped by expert, and the dense e4m3 product, which is the same with one expert and all rows.
//
//   out[p][n] = out_scale * x[row(p)] . w[e][n]     and     out_scale * silu(x . wg[e][n]) * (x . wu[e][n])
//   e4m3:  x . w = sum over blocks b of 128 k:  sx[row][b] * sw[n/128][b] * sum_{k in b} qx[k] qw[k]
//
// The MMA's M side is matrix rows, its N side a bucket of up to kTok routed rows of one expert, so that a ragged bucket wastes
// less than 16 (32 in a pair) columns and a single token less than a tile. One CTA (CG = 1) or a pair (CG = 2: tcgen05
// cta_group::2, 128 matrix rows and half of the bucket's rows each) walks over (bucket, row tile) tiles; consecutive tiles share a
// bucket, so its rows stay in L2 while the matrices stream through once. Warps:
//   epilogue   accumulators from tensor memory, scales, SiLU * up, stores. Lane = matrix row, column = routed row.
//   MMA        one elected thread; accumulators are double-buffered, so a tile's stores overlap the next tile's products
//   matrix     one elected thread, TMA boxes of 128 bytes of K: 128 rows, or for gate and up eight boxes of 16 rows in turn --
//              gate and up of one output then lie 16 lanes apart in one warp and meet by a shuffle
//   rows       tile::gather4 TMA copies of four routed rows each
//   scales     e4m3: sx * sw of each block of K as vectors in shared memory, a few blocks ahead
// In 16 bits the tensor core adds over all of K. In e4m3 each block of K is one accumulator buffer, which the epilogue scales and
// adds to its registers in f32 while the tensor core fills the other.
//
// Every wait on an mbarrier is bounded; on give-up the kernel raises a status flag, stores NaN in place of the outputs it did not
// form, frees its tensor memory and returns.
#include "knj_fp8.cuh"
#include "knj_tc.cuh"

using namespace knj;

namespace {

constexpr int kMaxExperts = 256;

struct GemmParams {
  const float *xs, *ws0, *ws1;
  const int32_t *pair_idx, *pair_cnt, *row_map;  // pair_idx null: one expert, pair i is row i
  void *out;
  int *status;
  int64_t ldo, idx_stride;
  int out_dtype, N, K, E, row_div, n_rows, n_pairs, m_tiles;
  uint32_t idesc_format;
  float out_scale;
  CUtensorMap map0, map1, mapx;
};

template <bool FP8, bool GATEUP, int CG>
struct Shape {
  static constexpr int kTok = CG == 2 ? 256 : 64;        // routed rows of a bucket (MMA N upper bound)
  static constexpr int kTokStep = 16 * CG;               // bucket sizes are multiples of this
  static constexpr int kEpiWarps = CG == 2 ? 8 : 4;
  static constexpr int kMmaWarp = kEpiWarps, kMatWarp = kEpiWarps + 1, kScaleWarp = kEpiWarps + 2;
  static constexpr int kRowWarps = CG == 2 ? 4 : 1, kRowWarp = CG == 2 ? 12 : 7;
  static constexpr int kThreads = 32 * (kRowWarp + kRowWarps);
  static constexpr int kBlocksPerSm = CG == 2 ? 1 : 2;
  static constexpr int kStages = CG == 2 ? 6 : 4;
  static constexpr int kATile = 128 * 128;               // bytes: 128 matrix rows x 128 bytes of K
  static constexpr int kBTile = kTok / CG * 128;
  static constexpr int kSlab = FP8 ? 128 : 64;           // elements of K per stage
  static constexpr int kOuts = GATEUP ? 64 : 128;        // outputs per CTA and tile
  static constexpr int kVecs = GATEUP ? 2 : 1;
  static constexpr int kScaleSlots = FP8 ? 4 : 0;
  static constexpr int kScaleSlot = kVecs * kTok * 4 + (GATEUP ? 64 : 0);   // the second vector starts 16 banks on
  static constexpr int kOffA = 0;
  static constexpr int kOffB = kOffA + kStages * kATile;
  static constexpr int kOffScale = kOffB + kStages * kBTile;
  static constexpr int kOffPairs = kOffScale + kScaleSlots * kScaleSlot;    // [2][kTok] pair of each column
  static constexpr int kOffPref = kOffPairs + 2 * kTok * 4;                 // [E + 1] buckets before expert e, [E] pairs of it
  static constexpr int kOffBars = kOffPref + (2 * kMaxExperts + 4) * 4;
  static constexpr int kBytes = kOffBars + 256 + 1024;
};

struct Tile {
  int e, tok0, ntok, mt;
};

// one MMA's K step is 32 bytes of every operand row in both element sizes
template <bool FP8, int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (FP8) tc_mma_f8<CG>(d, a, b, idesc, acc);
  else tc_mma_f16<CG>(d, a, b, idesc, acc);
}

__device__ __forceinline__ void fma2(float &a0, float &a1, uint32_t x0, uint32_t x1, float s0, float s1) {
  asm("{\n\t.reg .b64 x, s, a;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 s, {%4, %5};\n\tmov.b64 a, {%0, %1};\n\t"
      "fma.rn.f32x2 a, x, s, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(x0), "r"(x1), "f"(s0), "f"(s1));
}

template <bool FP8, bool GATEUP, int CG>
__global__ void __launch_bounds__(Shape<FP8, GATEUP, CG>::kThreads, Shape<FP8, GATEUP, CG>::kBlocksPerSm)
    expert_tc_kernel(const __grid_constant__ GemmParams p) {
  using S = Shape<FP8, GATEUP, CG>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = warp_index();
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;

  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kOffBars);
  uint64_t *full = bars;                        // [kStages] operands of both CTAs landed (the even CTA's are used)
  uint64_t *empty = full + S::kStages;          // [kStages] the stage's products are done
  uint64_t *acc_full = empty + S::kStages;      // [2] accumulator buffer complete
  uint64_t *acc_empty = acc_full + 2;           // [2] accumulator buffer read (the even CTA's are used)
  uint64_t *sc_full = acc_empty + 2;            // [kScaleSlots]
  uint64_t *sc_empty = sc_full + 4;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sc_empty + 4);
  volatile int *s_fail = reinterpret_cast<volatile int *>(tmem_slot + 1);  // raised by the first wait that gives up
  int32_t *s_pair = reinterpret_cast<int32_t *>(smem + S::kOffPairs);
  int32_t *s_pref = reinterpret_cast<int32_t *>(smem + S::kOffPref), *s_cnt = s_pref + kMaxExperts + 1;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], CG * S::kEpiWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sc_full[i], 1);
      mbar_init(&sc_empty[i], S::kEpiWarps);
    }
    *s_fail = 0;
    mbar_init_fence();
  }
  constexpr uint32_t kTmemCols = 2 * S::kTok;
  if (warp == S::kMmaWarp) {
    tmem_alloc<CG>(tmem_slot, kTmemCols);
    tmem_relinquish<CG>();
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
  if (CG == 2) cluster_sync_all();  // the peer's barriers are initialised before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int nslab = (p.K + S::kSlab - 1) / S::kSlab;
  const int n_tiles = s_pref[kMaxExperts] * p.m_tiles;   // < 2^31: checked on the host
  const int step = gridDim.x / CG;
  auto tile_at = [&](int t) {
    Tile r;
    const int b = t / p.m_tiles;
    r.mt = t - b * p.m_tiles;
    int lo = 0;  // the last expert whose first bucket is not behind b
#pragma unroll
    for (int h = kMaxExperts / 2; h > 0; h >>= 1)
      if (s_pref[lo + h] <= b) lo += h;
    r.e = lo;
    const int nb = s_pref[lo + 1] - s_pref[lo], cnt = s_cnt[lo];
    // an expert's pairs are spread evenly over its buckets: 256 + 14 pairs would stream the matrix twice for 14
    const int per = ((cnt + nb - 1) / nb + S::kTokStep - 1) / S::kTokStep * S::kTokStep;
    r.tok0 = (b - s_pref[lo]) * per;
    r.ntok = min(per, cnt - r.tok0);
    return r;
  };
  auto columns = [&](const Tile &t) { return (t.ntok + S::kTokStep - 1) / S::kTokStep * S::kTokStep; };
  // pair of column c (-1: none) and its row of x; pair -2 - p: p's row lies outside x, its output is zero
  auto resolve = [&](const Tile &t, int c, int &pr, int &row) {
    pr = -1;
    row = 0;
    if (c >= t.ntok) return;
    pr = p.pair_idx ? p.pair_idx[t.e * p.idx_stride + t.tok0 + c] : t.tok0 + c;
    if (pr < 0 || pr >= p.n_pairs) {
      pr = -1;
      return;
    }
    row = p.row_map ? p.row_map[pr] : pr / p.row_div;
    if (row < 0 || row >= p.n_rows) {
      pr = -2 - pr;
      row = 0;
    }
  };
  bool ok = true;  // once false this thread skips all work and waits but still meets every barrier
  // e4m3 in pairs: the epilogue's sums take 128 registers a thread. 512 threads x 128 registers at launch = 2 x 128 x 192 + 2 x 128 x 64
  if constexpr (FP8 && CG == 2) {
    if (warp < S::kEpiWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  }

  if (warp < S::kEpiWarps) {
    // =========================== epilogue ===========================
    const int group = warp >> 2, quad = warp & 3;     // chunks of 32 columns are dealt to the warp groups in turn
    constexpr int kGroups = S::kEpiWarps / 4, kChunks = S::kTok / 32 / kGroups;
    const uint32_t lanes = tmem_base + ((uint32_t)(quad * 32) << 16);
    auto wait_all = [&](uint64_t *bar, uint32_t parity) {
      if (ok && !mbar_wait(bar, parity, s_fail)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
    };
    int buf = 0, slot = 0, pb = 0;
    uint32_t par = 0, sc_par = 0;
    for (int t = blockIdx.x / CG; t < n_tiles; t += step, pb ^= 1) {
      const Tile tl = tile_at(t);
      const int ncol = columns(tl);
      if (tid < S::kTok) {
        int pr, row;
        resolve(tl, tid, pr, row);
        s_pair[pb * S::kTok + tid] = pr;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kEpiWarps) : "memory");
      const int32_t *pairs = s_pair + pb * S::kTok;
      const int n0 = tl.mt * S::kOuts * CG + (int)rank * S::kOuts;
      const int n = n0 + (GATEUP ? quad * 16 + (lane & 15) : quad * 32 + lane);
      auto put = [&](int pr, float v) {
        if (pr == -1 || n >= p.N) return;
        if (!ok) v = __int_as_float(0x7fffffff);
        else v *= p.out_scale;
        if (pr < 0) {
          pr = -2 - pr;
          if (ok) v = 0.f;
        }
        store_from_f32(p.out, p.out_dtype, pr * p.ldo + n, v);
      };
      // 32 columns from c0 on: one output per lane and column, or for gate and up one per lane and pair of columns
      auto finish = [&](const float (&v)[32], int c0) {
        if constexpr (GATEUP) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[j + 1] : v[j], 16);
            const float g = lane < 16 ? v[j] : got, u = lane < 16 ? got : v[j + 1];
            put(pairs[c0 + j + (lane >> 4)], __fdividef(g, 1.0f + __expf(-g)) * u);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) put(pairs[c0 + j], v[j]);
        }
      };
      if constexpr (!FP8) {
        wait_all(&acc_full[buf], par);
        tc_fence_after();
#pragma unroll 1
        for (int ch = group; ch * 32 < ncol; ch += kGroups) {
          uint32_t r[32] = {};
          if (ok) {
            tmem_ld32(lanes + buf * S::kTok + ch * 32, r);
            tmem_ld_wait();
          }
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          finish(v, ch * 32);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) mbar_arrive_cluster(cluster_addr(&acc_empty[buf], 0));
          else mbar_arrive(&acc_empty[buf]);
        }
        buf ^= 1;
        if (buf == 0) par ^= 1u;
      } else {
        float acc[kChunks][32];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c][j] = 0.f;
        for (int ks = 0; ks < nslab; ++ks) {
          wait_all(&sc_full[slot], sc_par);
          wait_all(&acc_full[buf], par);
          if (!ok) break;
          tc_fence_after();
          const float *sc = reinterpret_cast<const float *>(smem + S::kOffScale + slot * S::kScaleSlot) +
                            (GATEUP && lane >= 16 ? S::kTok + 16 : 0);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const int c0 = (c * kGroups + group) * 32;
            if (c0 < ncol) {
              uint32_t r[32];
              tmem_ld32(lanes + buf * S::kTok + c0, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(sc + c0 + j);
                fma2(acc[c][j], acc[c][j + 1], r[j], r[j + 1], f.x, f.y);
                fma2(acc[c][j + 2], acc[c][j + 3], r[j + 2], r[j + 3], f.z, f.w);
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) mbar_arrive_cluster(cluster_addr(&acc_empty[buf], 0));
            else mbar_arrive(&acc_empty[buf]);
            mbar_arrive(&sc_empty[slot]);
          }
          buf ^= 1;
          if (buf == 0) par ^= 1u;
          if (++slot == S::kScaleSlots) {
            slot = 0;
            sc_par ^= 1u;
          }
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int c0 = (c * kGroups + group) * 32;
          if (c0 < ncol) finish(acc[c], c0);
        }
      }
    }
  } else if (warp == S::kMmaWarp) {
    // =========================== MMA issue ===========================
    if (rank == 0 && elect_one()) {
      const uint64_t a_desc0 = smem_desc_sw128(smem_u32(smem + S::kOffA)), b_desc0 = smem_desc_sw128(smem_u32(smem + S::kOffB));
      int st = 0, buf = 0;
      uint32_t par = 0, acc_par = 1;  // a fresh barrier passes a wait for parity 1
      for (int t = blockIdx.x / CG; t < n_tiles && ok; t += step) {
        const uint32_t idesc = instr_desc_f16(128 * CG, columns(tile_at(t))) | p.idesc_format;
        if (!FP8 && !mbar_spin(&acc_empty[buf], acc_par, s_fail)) { ok = false; break; }
        for (int ks = 0; ks < nslab; ++ks) {
          if (FP8 && !mbar_spin(&acc_empty[buf], acc_par, s_fail)) { ok = false; break; }
          if (!mbar_spin(&full[st], par, s_fail)) { ok = false; break; }
          tc_fence_after();
          const uint64_t a = a_desc0 + (uint32_t)(st * S::kATile) / 16, b = b_desc0 + (uint32_t)(st * S::kBTile) / 16;
#pragma unroll
          for (int k = 0; k < 4; ++k) mma<FP8, CG>(tmem_base + buf * S::kTok, a + 2 * k, b + 2 * k, idesc, (k > 0 || (!FP8 && ks > 0)) ? 1u : 0u);
          if (CG == 2) tc_commit_pair(smem_u32(&empty[st]));
          else tc_commit_addr<CG>(smem_u32(&empty[st]));
          if (FP8 || ks + 1 == nslab) {
            if (CG == 2) tc_commit_pair(smem_u32(&acc_full[buf]));
            else tc_commit_addr<CG>(smem_u32(&acc_full[buf]));
            buf ^= 1;
            if (buf == 0) acc_par ^= 1u;
          }
          if (++st == S::kStages) { st = 0; par ^= 1u; }
        }
      }
    }
  } else if (warp == S::kMatWarp) {
    // =========================== matrix rows ===========================
    if (elect_one()) {
      int st = 0;
      uint32_t par = 1;
      for (int t = blockIdx.x / CG; t < n_tiles && ok; t += step) {
        const Tile tl = tile_at(t);
        const int y = tl.e * p.N + tl.mt * S::kOuts * CG + (int)rank * S::kOuts;
        const uint32_t bytes = (uint32_t)(CG * S::kATile + columns(tl) * 128);  // of both CTAs, matrix and rows
        for (int ks = 0; ks < nslab; ++ks) {
          if (!mbar_spin(&empty[st], par, s_fail)) { ok = false; break; }
          if (rank == 0) mbar_expect_tx(&full[st], bytes);
          const uint32_t bar = CG == 2 ? cluster_addr(&full[st], 0) : smem_u32(&full[st]);
          const uint32_t dst = smem_u32(smem + S::kOffA + st * S::kATile);
          if (GATEUP) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              tma_load_box<CG>(dst + j * 4096, &p.map0, ks * S::kSlab, y + 16 * j, bar);
              tma_load_box<CG>(dst + j * 4096 + 2048, &p.map1, ks * S::kSlab, y + 16 * j, bar);
            }
          } else {
            tma_load_box<CG>(dst, &p.map0, ks * S::kSlab, y, bar);
          }
          if (++st == S::kStages) { st = 0; par ^= 1u; }
        }
      }
    }
  } else if (FP8 && warp == S::kScaleWarp) {
    // =========================== scales ===========================
    constexpr int kPer = S::kTok / 32, kAhead = 4;   // columns per lane, blocks of K read at once
    const int nb_n = (p.N + 127) / 128;
    int slot = 0;
    uint32_t par = 1;
    for (int t = blockIdx.x / CG; t < n_tiles && ok; t += step) {
      const Tile tl = tile_at(t);
      const int n0 = tl.mt * S::kOuts * CG + (int)rank * S::kOuts;
      // a CTA behind the last output of a pair's tile has no block of its own: any block's scales do
      const int64_t blk = ((int64_t)tl.e * nb_n + min(n0 / 128, nb_n - 1)) * nslab;
      const float *xs[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        int pr, row;
        resolve(tl, lane + 32 * j, pr, row);
        xs[j] = p.xs + (int64_t)row * nslab;
      }
      for (int k0 = 0; k0 < nslab && ok; k0 += kAhead) {
        float v[kAhead][kPer], w0[kAhead], w1[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int kb = min(k0 + i, nslab - 1);
          w0[i] = p.ws0[blk + kb];
          if (GATEUP) w1[i] = p.ws1[blk + kb];
#pragma unroll
          for (int j = 0; j < kPer; ++j) v[i][j] = xs[j][kb];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (k0 + i < nslab && ok) {
            if (!mbar_wait(&sc_empty[slot], par, s_fail)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              float *dst = reinterpret_cast<float *>(smem + S::kOffScale + slot * S::kScaleSlot);
#pragma unroll
              for (int j = 0; j < kPer; ++j) {
                dst[lane + 32 * j] = v[i][j] * w0[i];
                if (GATEUP) dst[S::kTok + 16 + lane + 32 * j] = v[i][j] * w1[i];
              }
              __syncwarp();
              if (lane == 0) mbar_arrive(&sc_full[slot]);
              if (++slot == S::kScaleSlots) {
                slot = 0;
                par ^= 1u;
              }
            }
          }
        }
      }
    }
  } else if (warp >= S::kRowWarp && warp < S::kRowWarp + S::kRowWarps) {
    // =========================== routed rows ===========================
    const int w = warp - S::kRowWarp;
    constexpr int kQuads = S::kTok / CG / (4 * S::kRowWarps);   // copies of four rows per warp and stage
    int st = 0;
    uint32_t par = 1;
    for (int t = blockIdx.x / CG; t < n_tiles; t += step) {
      const Tile tl = tile_at(t);
      const int n_cta = columns(tl) / CG;
      int4 rows[kQuads];
#pragma unroll
      for (int g = 0; g < kQuads / 8; ++g) {
        // lane 4q + i finds row i of the warp's quad 8g + q
        const int r = 4 * (w + S::kRowWarps * (8 * g + (lane >> 2))) + (lane & 3);
        int pr, row = 0;
        if (r < n_cta) resolve(tl, (int)rank * n_cta + r, pr, row);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          rows[8 * g + q].x = __shfl_sync(0xffffffffu, row, 4 * q);
          rows[8 * g + q].y = __shfl_sync(0xffffffffu, row, 4 * q + 1);
          rows[8 * g + q].z = __shfl_sync(0xffffffffu, row, 4 * q + 2);
          rows[8 * g + q].w = __shfl_sync(0xffffffffu, row, 4 * q + 3);
        }
      }
      if (elect_one()) {
        int s = st;
        uint32_t sp = par;
        for (int ks = 0; ks < nslab; ++ks) {
          if (!mbar_spin(&empty[s], sp, s_fail)) { ok = false; break; }
          const uint32_t bar = CG == 2 ? cluster_addr(&full[s], 0) : smem_u32(&full[s]);
          const uint32_t dst = smem_u32(smem + S::kOffB + s * S::kBTile);
#pragma unroll
          for (int q = 0; q < kQuads; ++q) {
            const int r = 4 * (w + S::kRowWarps * q);
            if (r < n_cta) tma_gather4<CG>(dst + r * 128, &p.mapx, ks * S::kSlab, rows[q], bar);
          }
          if (++s == S::kStages) { s = 0; sp ^= 1u; }
        }
      }
      par ^= (uint32_t)((st + nslab) / S::kStages) & 1u;
      st = (st + nslab) % S::kStages;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
  }

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

int g_form = 0;  // 0 = by the rule below, 1 = single SMs, 2 = pairs (knj_expert_tc_form)

struct Operands {
  const void *x, *w0, *w1;
  int64_t ldx;
  bool fp8;
};

template <bool FP8, bool GATEUP, int CG>
int launch_form(GemmParams p, const Operands &o, cudaStream_t st) {
  using S = Shape<FP8, GATEUP, CG>;
  int dev = 0;
  KNJ_CUDA(cudaGetDevice(&dev));
  auto kern = expert_tc_kernel<FP8, GATEUP, CG>;
  static bool opted[64] = {false};
  if (dev >= 0 && dev < 64 && !opted[dev]) {
    KNJ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    opted[dev] = true;
  }
  constexpr int esz = FP8 ? 1 : 2;
  const uint64_t w_rows = (uint64_t)p.E * p.N;
  int rc = make_operand_tensor_map(&p.map0, o.w0, esz, p.K, p.K, w_rows, GATEUP ? 16 : 128);
  if (!rc && GATEUP) rc = make_operand_tensor_map(&p.map1, o.w1, esz, p.K, p.K, w_rows, 16);
  if (!rc) rc = make_operand_tensor_map(&p.mapx, o.x, esz, p.K, o.ldx, p.n_rows, 1);
  if (rc) return rc;
  p.m_tiles = (p.N + S::kOuts * CG - 1) / (S::kOuts * CG);
  const int64_t most = p.pair_idx ? p.E * ((p.idx_stride + S::kTok - 1) / S::kTok) : (p.n_pairs + S::kTok - 1) / S::kTok;
  KNJ_REQUIRE(most * p.m_tiles < (1ll << 31) && (int64_t)w_rows + 256 < (1ll << 31), "expert product: %lld buckets of %d row tiles are too many",
              (long long)most, p.m_tiles);
  // the tiles that these pairs can make; a table that names pairs more than once makes more, which the same grid walks over
  const int64_t tiles = ((int64_t)p.n_pairs / S::kTok + (p.E < p.n_pairs ? p.E : p.n_pairs)) * p.m_tiles;
  const int64_t cap = (int64_t)sm_count() * S::kBlocksPerSm / CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((tiles < cap ? tiles : cap) * CG));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_chain_overlap ? 2 : 1;
  KNJ_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return launch_status("expert_tc_kernel");
}

template <bool GATEUP>
int launch_gemm(const GemmParams &p, const Operands &o, cudaStream_t st) {
  const int experts = p.E < p.n_pairs ? p.E : p.n_pairs;
  const bool pairs = g_form ? g_form == 2 : (int64_t)p.n_pairs > 32ll * experts;
  if (o.fp8) return pairs ? launch_form<true, GATEUP, 2>(p, o, st) : launch_form<true, GATEUP, 1>(p, o, st);
  return pairs ? launch_form<false, GATEUP, 2>(p, o, st) : launch_form<false, GATEUP, 1>(p, o, st);
}

int check_expert(const knj_expert_gemm_args *a, bool gateup, const char *who) {
  KNJ_REQUIRE(a, "%s: null argument block", who);
  KNJ_REQUIRE(a->n_pairs >= 0 && a->n_rows >= 0 && a->N > 0 && a->K > 0 && a->n_experts >= 1 && a->n_experts <= kMaxExperts, "%s: bad sizes", who);
  if (a->n_pairs == 0) return KNJ_OK;
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

int run_expert(const knj_expert_gemm_args *a, bool gateup, const char *who, knj_stream_t s) {
  const int rc = check_expert(a, gateup, who);
  if (rc || a->n_pairs == 0) return rc;
  GemmParams p{};
  p.xs = a->x_scale; p.ws0 = a->w0_scale; p.ws1 = a->w1_scale; p.pair_idx = a->pair_idx; p.pair_cnt = a->pair_cnt; p.row_map = a->row_map;
  p.out = a->out; p.status = a->status; p.ldo = a->ldo; p.idx_stride = a->idx_stride; p.out_dtype = a->out_dtype; p.N = a->N; p.K = a->K;
  p.E = a->n_experts; p.row_div = a->row_div > 0 ? a->row_div : 1; p.n_rows = a->n_rows; p.n_pairs = a->n_pairs; p.out_scale = a->out_scale;
  p.idesc_format = a->w_dtype == KNJ_DT_BF16 ? (1u << 7) | (1u << 10) : 0u;
  const Operands o{a->x, a->w0, a->w1, a->ldx, a->w_dtype == KNJ_DT_E4M3};
  return gateup ? launch_gemm<true>(p, o, as_stream(s)) : launch_gemm<false>(p, o, as_stream(s));
}

inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

extern "C" {

int knj_expert_gateup_launch(const knj_expert_gemm_args *a, knj_stream_t s) { return run_expert(a, true, "knj_expert_gateup", s); }

int knj_expert_proj_launch(const knj_expert_gemm_args *a, knj_stream_t s) { return run_expert(a, false, "knj_expert_proj", s); }

void knj_expert_tc_form(int form) { g_form = form == 1 || form == 2 ? form : 0; }

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
  p.xs = qs; p.ws0 = W_scale; p.out = y; p.status = status; p.ldo = ldy; p.out_dtype = y_dtype; p.N = n_out; p.K = n_in; p.E = 1;
  p.row_div = 1; p.n_rows = m; p.n_pairs = m; p.out_scale = 1.0f;
  return launch_gemm<false>(p, Operands{q, W, nullptr, n_in, true}, as_stream(s));
}

}  // extern "C"
