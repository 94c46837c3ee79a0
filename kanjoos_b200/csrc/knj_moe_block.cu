// knj_moe_block.cu -- a whole MoE block with experts in bf16, fp16 or e4m3 as one C-ABI call: the stage sequence of the CPU
// branch (src/model/model.cpp:631-652) with a norm, a gate and scales around the residual add, every intermediate in a
// caller-provided workspace.
#include "knj_common.cuh"

using namespace knj;

namespace {

constexpr float kF16Prescale = 0.015625f;  // 2^-6: room for products of gate and up in fp16

inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

struct BlockWs {
  uint8_t *h, *hq, *act, *aq;
  float *hs, *as, *logits, *pair_w, *Y, *sum;
  int32_t *pair_exp, *pair_idx, *pair_cnt, *status;
  size_t bytes;
};

BlockWs carve(void *base, int T, int H, int F, int E, int k, int w_dtype) {
  BlockWs w{};
  size_t used = 0;
  auto take = [&](size_t n) {
    uint8_t *r = base ? static_cast<uint8_t *>(base) + used : nullptr;
    used += up256(n);
    return r;
  };
  const size_t P = (size_t)T * k;
  const bool q = w_dtype == KNJ_DT_E4M3;
  w.status = reinterpret_cast<int32_t *>(take(16));   // the first word, whatever the sizes
  w.h = take((size_t)T * H * 2);
  w.hq = q ? take((size_t)T * H) : nullptr;
  w.hs = reinterpret_cast<float *>(q ? take((size_t)T * ((H + 127) / 128) * 4) : nullptr);
  w.logits = reinterpret_cast<float *>(take((size_t)T * E * 4));
  w.pair_exp = reinterpret_cast<int32_t *>(take(P * 4));
  w.pair_w = reinterpret_cast<float *>(take(P * 4));
  w.pair_idx = reinterpret_cast<int32_t *>(take((size_t)E * T * 4));
  w.pair_cnt = reinterpret_cast<int32_t *>(take((size_t)E * 4));
  w.act = take(P * F * 2);
  w.aq = q ? take(P * F) : nullptr;
  w.as = reinterpret_cast<float *>(q ? take(P * ((F + 127) / 128) * 4) : nullptr);
  w.Y = reinterpret_cast<float *>(take(P * H * 4));
  w.sum = reinterpret_cast<float *>(take((size_t)T * H * 4));
  w.bytes = used;
  return w;
}

struct StageSpan {
  int h;
  knj_stream_t s;
  StageSpan(const char *name, knj_stream_t st) : h(knj_spans_active() ? knj_span_begin(name, st) : -1), s(st) {}
  ~StageSpan() { if (h >= 0) knj_span_end(h, s); }
};

int check(const knj_moe_block_args *a, const char *who) {
  KNJ_REQUIRE(a, "%s: null argument block", who);
  KNJ_REQUIRE(a->n_tokens >= 0 && a->hidden > 0 && a->ffn > 0 && a->n_experts > 0, "%s: bad sizes", who);
  if (a->n_tokens == 0) return KNJ_OK;
  KNJ_REQUIRE(a->hidden % 256 == 0 && a->ffn % 16 == 0, "%s: hidden=%d must be a multiple of 256, ffn=%d of 16", who, a->hidden, a->ffn);
  KNJ_REQUIRE(a->hidden <= KNJ_BLOCK_NORM_MAX_HIDDEN, "%s: hidden=%d above %d", who, a->hidden, KNJ_BLOCK_NORM_MAX_HIDDEN);
  KNJ_REQUIRE(a->n_experts <= 256 && a->top_k >= 1 && a->top_k <= 8 && a->top_k <= a->n_experts, "%s: %d experts, top_k=%d out of range", who,
              a->n_experts, a->top_k);
  KNJ_REQUIRE(a->w_dtype >= KNJ_DT_BF16 && a->w_dtype <= KNJ_DT_E4M3, "%s: experts are bf16, f16 or e4m3", who);
  KNJ_REQUIRE(a->x && a->out && a->w_router && a->w_gate && a->w_up && a->w_down, "%s: null tensor pointer", who);
  KNJ_REQUIRE(a->w_dtype != KNJ_DT_E4M3 || (a->gate_scale && a->up_scale && a->down_scale), "%s: e4m3 experts need their scales", who);
  KNJ_REQUIRE(aligned16(a->w_router), "%s: the router's weights must be 16-byte aligned", who);
  KNJ_REQUIRE((int64_t)a->n_tokens * a->top_k <= (1ll << 30), "%s: more than 2^30 pairs of a token and an expert", who);
  KNJ_REQUIRE((a->next_w != nullptr) == (a->h_next != nullptr), "%s: next_w and h_next go together", who);
  const size_t need = knj_moe_block_workspace_bytes(a->n_tokens, a->hidden, a->ffn, a->n_experts, a->top_k, a->w_dtype);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("%s: workspace of %zu bytes needed, %zu given", who, need, a->workspace_bytes);
    return KNJ_E_WORKSPACE;
  }
  KNJ_REQUIRE((reinterpret_cast<uintptr_t>(a->workspace) & 255u) == 0, "%s: workspace must be 256-byte aligned", who);
  return KNJ_OK;
}

}  // namespace

extern "C" {

size_t knj_moe_block_workspace_bytes(int n_tokens, int hidden, int ffn, int n_experts, int top_k, int w_dtype) {
  if (n_tokens <= 0) return 256;
  return carve(nullptr, n_tokens, hidden, ffn, n_experts, top_k, w_dtype).bytes;
}

int knj_moe_block_launch(const knj_moe_block_args *a, knj_stream_t s) {
  int rc = check(a, "knj_moe_block");
  if (rc || a->n_tokens == 0) return rc;
  const int T = a->n_tokens, H = a->hidden, F = a->ffn, E = a->n_experts, k = a->top_k, P = T * k;
  const bool q = a->w_dtype == KNJ_DT_E4M3;
  const int act = a->w_dtype == KNJ_DT_F16 ? KNJ_DT_F16 : KNJ_DT_BF16;   // 16-bit rows
  const BlockWs w = carve(a->workspace, T, H, F, E, k, a->w_dtype);
  int32_t *pair_exp = a->tap_pair_exp ? a->tap_pair_exp : w.pair_exp;
  float *pair_w = a->tap_pair_w ? a->tap_pair_w : w.pair_w;
  int32_t *status = a->status ? a->status : w.status;

  // what the launches check of the caller's operands is checked before the first runs
  knj_block_norm_args after{};
  after.n_tokens = T; after.hidden = H; after.x = a->x; after.ldx = a->ldx; after.y = w.sum; after.ldy = H; after.post_w = a->post_w;
  after.pre_w = a->next_w; after.gate = a->gate; after.ldg = a->ldg; after.stream_out = a->out; after.ld_stream = a->ldo; after.h = a->h_next;
  after.ldh = a->ld_h_next; after.h_scale = a->h_next_scale; after.x_dtype = a->x_dtype; after.y_dtype = KNJ_DT_F32; after.w_dtype = a->w_norm_dtype;
  after.gate_dtype = a->gate_dtype; after.stream_dtype = a->out_dtype; after.h_dtype = a->h_next_dtype; after.gate_kind = a->gate_kind;
  after.gate_sigmoid = a->gate_sigmoid; after.alpha = a->alpha; after.beta = a->beta; after.eps = a->eps; after.status = status;
  rc = block_norm_check(&after);
  if (rc) return rc;
  // the rows of x in the experts' 16-bit type, normalised or as they are
  knj_block_norm_args before{};
  before.n_tokens = T; before.hidden = H; before.x = a->x; before.ldx = a->ldx; before.x_dtype = a->x_dtype; before.w_dtype = a->w_norm_dtype;
  before.beta = 1.0f; before.alpha = 1.0f; before.eps = a->eps; before.status = status;
  if (a->pre_w) {
    before.pre_w = a->pre_w; before.h = w.h; before.ldh = H; before.h_dtype = act;
  } else {
    before.stream_out = w.h; before.ld_stream = H; before.stream_dtype = act;
  }
  knj_expert_gemm_args gateup{};
  gateup.pair_idx = w.pair_idx; gateup.pair_cnt = w.pair_cnt; gateup.idx_stride = T; gateup.n_pairs = P; gateup.n_experts = E;
  gateup.x_dtype = gateup.w_dtype = a->w_dtype; gateup.status = status;
  knj_expert_gemm_args down = gateup;
  gateup.x = q ? w.hq : w.h; gateup.x_scale = w.hs; gateup.ldx = H; gateup.n_rows = T; gateup.row_div = k; gateup.w0 = a->w_gate; gateup.w1 = a->w_up;
  gateup.w0_scale = a->gate_scale; gateup.w1_scale = a->up_scale; gateup.N = F; gateup.K = H; gateup.out = w.act; gateup.ldo = F; gateup.out_dtype = act;
  gateup.out_scale = act == KNJ_DT_F16 ? kF16Prescale : 1.0f;
  down.x = q ? w.aq : w.act; down.x_scale = w.as; down.ldx = F; down.n_rows = P; down.row_div = 1; down.w0 = a->w_down; down.w0_scale = a->down_scale;
  down.N = H; down.K = F; down.out = w.Y; down.ldo = H; down.out_dtype = KNJ_DT_F32; down.out_scale = act == KNJ_DT_F16 ? 1.0f / kF16Prescale : 1.0f;
  rc = block_norm_check(&before);
  if (!rc) rc = expert_product_check(&gateup, true, "knj_moe_block, gate and up");
  if (!rc) rc = expert_product_check(&down, false, "knj_moe_block, down");
  if (rc) return rc;
  KNJ_CUDA(cudaMemsetAsync(status, 0, 4, as_stream(s)));  // raised when a bounded wait of a norm or a product gives up
  {
    StageSpan sp("moe-router", s);
    rc = knj_block_norm_launch(&before, s);
    if (rc) return rc;
    rc = knj_router_topk_launch(w.h, act, H, a->w_router, a->router_bias, T, H, E, k, w.logits, pair_exp, pair_w, s);
    if (rc) return rc;
  }
  {
    StageSpan sp("moe-gather", s);
    // long pair lists take the counting-sort form; its scratch is the activation buffer, which is written later
    rc = moe_permute_tables(pair_exp, P, E, T, w.pair_idx, w.pair_cnt, w.act, (size_t)P * F * 2, as_stream(s));
    if (rc) return rc;
    if (q) rc = knj_fp8_rows_launch(w.h, act, H, T, H, w.hq, w.hs, s);
    if (rc) return rc;
  }
  {
    StageSpan sp("moe-gate", s);
    rc = knj_expert_gateup_launch(&gateup, s);
    if (rc) return rc;
  }
  {
    StageSpan sp("moe-down", s);
    if (q) rc = knj_fp8_rows_launch(w.act, act, F, P, F, w.aq, w.as, s);
    if (rc) return rc;
    rc = knj_expert_proj_launch(&down, s);
    if (rc) return rc;
  }
  StageSpan sp("moe-scatter", s);
  rc = knj_moe_combine_launch(w.Y, nullptr, pair_exp, pair_w, nullptr, 0, 0, w.sum, KNJ_DT_F32, H, T, H, k, s);
  if (rc) return rc;
  return knj_block_norm_launch(&after, s);
}

int knj_moe_block_status(const knj_moe_block_args *a, knj_stream_t s) {
  const int rc = check(a, "knj_moe_block_status");
  if (rc || a->n_tokens == 0) return rc;
  const int32_t *status = a->status ? a->status : static_cast<const int32_t *>(a->workspace);
  int32_t word = 0;
  KNJ_CUDA(cudaMemcpyAsync(&word, status, sizeof(word), cudaMemcpyDeviceToHost, as_stream(s)));
  KNJ_CUDA(cudaStreamSynchronize(as_stream(s)));
  if (word != 0) {
    set_error("knj_moe_block: a bounded device wait of the norms or the expert products gave up");
    return KNJ_E_TIMEOUT;
  }
  return KNJ_OK;
}

}  // extern "C"
