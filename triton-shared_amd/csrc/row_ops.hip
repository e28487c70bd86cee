// The C entries of the operators whose weights are picked per row: what include/tts_hip.h says about their arguments is checked
// here, on the host, before anything is launched.
#include "op_args.h"
#include "row_ops.h"

using namespace tts;

namespace {

constexpr int64_t MOST_WIDTH = (int64_t)1 << 24;  // of a layer: its tiles fit 32 bits, and a token's sums a grid

ExpertMatrix matrix_of(const Arg &w) {
  ExpertMatrix m = {};
  m.w = w.t->ptr, m.w_expert = w.stride(0), m.w_k = w.stride(1), m.w_n = w.stride(2);
  if (m.w_k != 1 && m.w_n != 1) invalid(w.name + ": neither its inputs (dimension 1) nor its outputs (dimension 2) have stride 1");
  // the kernels' offsets within an expert are 32-bit: to a column's inputs, or to eight rows of them
  const int64_t item = item_size(w.t->dtype), most = m.w_k == 1 ? w.size(2) * m.w_n + 64 : 32 * m.w_k + w.size(2);
  if (most * item > 0xffffffffll) unsupported(w.name + ": strides of " + std::to_string(m.w_k) + " and " + std::to_string(m.w_n) + " reach past 4 GiB in one expert");
  return m;
}

// what sizes, types and orders alone say, for the workspace and for the call
ExpertsParams experts_sizes(const tts_tensor *x_, const tts_tensor *ids_, const tts_tensor *w_up_, const tts_tensor *w_down_, int gated) {
  Arg x(x_, "x"), ids(ids_, "ids"), w_up(w_up_, "w_up"), w_down(w_down_, "w_down");
  x.rank(2), ids.rank(2).type(TTS_I32).shape(0, x.size(0), "x").some(1), w_up.rank(3).shape(1, x.size(1), "x").some(0), w_down.rank(3).shape(0, w_up.size(0), "w_up");
  half_type(x);
  if (w_up.t->dtype != TTS_I8 && w_up.t->dtype != x.t->dtype) invalid("w_up is " + std::string(type_name(w_up.t->dtype)) + ", not i8 or x's type");
  w_down.type(w_up.t->dtype);
  if (gated && w_up.size(2) % 2) invalid("w_up: dimension 2 is " + std::to_string(w_up.size(2)) + ", and a gated layer has two halves there");
  ExpertsParams p = {};
  p.tokens = x.size(0), p.hidden = x.size(1), p.inner = gated ? w_up.size(2) / 2 : w_up.size(2), p.outputs = w_down.size(2);
  w_down.shape(1, p.inner, "w_up");
  p.experts = (int)w_up.size(0), p.gated = gated != 0, p.bf16 = x.t->dtype == TTS_BF16, p.int8 = w_up.t->dtype == TTS_I8;
  const int least = p.int8 ? 16 : 8;  // 16 bytes of a row of weights
  if (p.hidden < least || p.inner < least || p.outputs < least) unsupported("a layer narrower than " + std::to_string(least) + " (" + std::to_string(p.hidden) + " x " + std::to_string(p.inner) + " x " + std::to_string(p.outputs) + ")");
  if (p.inner > MOST_WIDTH || p.outputs > MOST_WIDTH) unsupported("a layer wider than " + std::to_string(MOST_WIDTH) + " (" + std::to_string(p.inner) + ", " + std::to_string(p.outputs) + ")");
  if (ids.size(1) > EXPERTS_MAX_SLOTS || p.tokens * ids.size(1) > EXPERTS_MAX_SLOTS)
    unsupported(std::to_string(p.tokens) + " tokens of " + std::to_string(ids.size(1)) + " experts: more than " + std::to_string(EXPERTS_MAX_SLOTS) + " in all");
  p.top = (int)ids.size(1);
  p.up = matrix_of(w_up), p.down = matrix_of(w_down);
  if (!experts_fit_a_grid(p)) unsupported(std::to_string(p.tokens * p.top) + " slots of " + std::to_string(p.inner) + " and " + std::to_string(p.outputs) + " columns: more workgroups than a launch has");
  return p;
}

LoraParams lora_sizes(const tts_tensor *x_, const tts_tensor *b_) {
  Arg x(x_, "x"), b(b_, "b");
  x.rank(2).some(1), b.rank(3).some(0).some(1).some(2);
  half_type(x);
  b.type(x.t->dtype);
  LoraParams p = {};
  p.tokens = x.size(0), p.inputs = x.size(1), p.adapters = (int)b.size(0), p.outputs = b.size(1);
  if (b.size(2) > LORA_MAX_RANK) unsupported("b: a rank of " + std::to_string(b.size(2)) + ", more than " + std::to_string(LORA_MAX_RANK));
  if (p.tokens > 32 * 65535) unsupported("x: " + std::to_string(p.tokens) + " rows");
  p.rank = (int)b.size(2), p.bf16 = x.t->dtype == TTS_BF16;
  return p;
}

}  // namespace

extern "C" {

tts_status tts_moe_route(const tts_tensor *logits_, const tts_tensor *bias_, int scoring, int renormalize, double scale, const tts_tensor *ids_, const tts_tensor *weights_,
                         void *stream) {
  return guarded("tts_moe_route", [&]() -> hipError_t {
    Arg logits(logits_, "logits"), ids(ids_, "ids"), weights(weights_, "weights");
    logits.rank(2).some(1).neighbours();
    if (logits.t->dtype != TTS_F32 && logits.t->dtype != TTS_F16 && logits.t->dtype != TTS_BF16) invalid("logits are " + std::string(type_name(logits.t->dtype)) + ", not f32, f16 or bf16");
    if (scoring != TTS_SOFTMAX && scoring != TTS_SIGMOID) invalid("unknown scoring " + std::to_string(scoring));
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    if (experts > ROUTE_MAX_EXPERTS) unsupported(std::to_string(experts) + " experts, more than " + std::to_string(ROUTE_MAX_EXPERTS));
    ids.rank(2).type(TTS_I32).shape(0, tokens, "logits").some(1).neighbours().distinct();
    const int64_t top = ids.size(1);
    if (top > experts) invalid("ids: " + std::to_string(top) + " of " + std::to_string(experts) + " experts");
    if (top > ROUTE_MAX_TOP) unsupported("ids: " + std::to_string(top) + " experts of a token, more than " + std::to_string(ROUTE_MAX_TOP));
    weights.rank(2).type(TTS_F32).shape(0, tokens, "logits").shape(1, top, "ids").neighbours().distinct();
    RouteParams p = {};
    if (bias_) {
      Arg bias(bias_, "bias");
      bias.rank(1).type(TTS_F32).shape(0, experts, "logits").neighbours().present();
      apart(ids, bias), apart(weights, bias);
      p.bias = (const float *)bias.t->ptr;
    }
    logits.present(), ids.present(), weights.present();
    apart(ids, logits), apart(weights, logits), apart(ids, weights);
    if (!tokens) return hipSuccess;
    p.logits = logits.t->ptr, p.ids = (int *)ids.t->ptr, p.weights = (float *)weights.t->ptr;
    p.tokens = tokens, p.ld = logits.stride(0), p.ld_ids = ids.stride(0), p.ld_weights = weights.stride(0);
    p.experts = (int)experts, p.top = (int)top;
    p.elem = logits.t->dtype, p.sigmoid = scoring == TTS_SIGMOID, p.renormalize = renormalize != 0, p.scale = (float)scale;
    return launch_route(p, (hipStream_t)stream);
  });
}

tts_status tts_moe_experts_workspace(const tts_tensor *x, const tts_tensor *ids, const tts_tensor *w_up, const tts_tensor *w_down, int gated, size_t *bytes) {
  return guarded("tts_moe_experts_workspace", [&]() -> hipError_t {
    if (!bytes) invalid("bytes is missing");
    *bytes = experts_workspace_bytes(experts_sizes(x, ids, w_up, w_down, gated));
    return hipSuccess;
  });
}

tts_status tts_moe_experts(const tts_tensor *x_, const tts_tensor *ids_, const tts_tensor *weights_, const tts_tensor *w_up_, const tts_tensor *s_up_, const tts_tensor *w_down_,
                           const tts_tensor *s_down_, int activation, int gated, const tts_tensor *out_, void *workspace, size_t bytes, void *stream) {
  return guarded("tts_moe_experts", [&]() -> hipError_t {
    ExpertsParams p = experts_sizes(x_, ids_, w_up_, w_down_, gated);
    Arg x(x_, "x"), ids(ids_, "ids"), weights(weights_, "weights"), w_up(w_up_, "w_up"), w_down(w_down_, "w_down"), out(out_, "out");
    if (activation < TTS_SILU || activation > TTS_RELU) invalid("unknown activation " + std::to_string(activation));
    x.neighbours(), ids.neighbours();
    weights.rank(2).type(TTS_F32).shape(0, p.tokens, "x").shape(1, p.top, "ids").neighbours();
    out.rank(2).type(x.t->dtype).shape(0, p.tokens, "x").shape(1, p.outputs, "w_down").neighbours().distinct();
    x.present(), ids.present(), weights.present(), w_up.present(), w_down.present(), out.present();
    if (p.int8) {
      Arg s_up(s_up_, "s_up"), s_down(s_down_, "s_down");
      s_up.rank(2).type(TTS_F32).shape(0, p.experts, "w_up").shape(1, w_up.size(2), "w_up").neighbours().present();
      s_down.rank(2).type(TTS_F32).shape(0, p.experts, "w_down").shape(1, p.outputs, "w_down").neighbours().present();
      apart(out, s_up), apart(out, s_down);
      p.up.scale = (const float *)s_up.t->ptr, p.up.scale_expert = s_up.stride(0);
      p.down.scale = (const float *)s_down.t->ptr, p.down.scale_expert = s_down.stride(0);
    } else if (s_up_ || s_down_)
      invalid("scales belong to i8 weights, and these are " + std::string(type_name(w_up.t->dtype)));
    apart(out, ids), apart(out, weights), apart(out, w_up), apart(out, w_down);
    check_workspace(workspace, bytes, experts_workspace_bytes(p));
    if (!p.tokens) return hipSuccess;
    p.x = x.t->ptr, p.ids = (const int *)ids.t->ptr, p.weights = (const float *)weights.t->ptr, p.out = out.t->ptr;
    p.ld_x = x.stride(0), p.ld_ids = ids.stride(0), p.ld_weights = weights.stride(0), p.ld_out = out.stride(0);
    p.activation = activation, p.workspace = workspace;
    return launch_experts(p, (hipStream_t)stream);
  });
}

tts_status tts_lora_add_workspace(const tts_tensor *x, const tts_tensor *b, size_t *bytes) {
  return guarded("tts_lora_add_workspace", [&]() -> hipError_t {
    if (!bytes) invalid("bytes is missing");
    *bytes = lora_workspace_bytes(lora_sizes(x, b));
    return hipSuccess;
  });
}

tts_status tts_lora_add(const tts_tensor *base_, const tts_tensor *x_, const tts_tensor *a_, const tts_tensor *b_, const tts_tensor *ids_, const tts_tensor *scales_,
                        const tts_tensor *out_, void *workspace, size_t bytes, void *stream) {
  return guarded("tts_lora_add", [&]() -> hipError_t {
    LoraParams p = lora_sizes(x_, b_);
    Arg base(base_, "base"), x(x_, "x"), a(a_, "a"), b(b_, "b"), ids(ids_, "ids"), out(out_, "out");
    x.neighbours(), b.neighbours();
    base.rank(2).type(x.t->dtype).shape(0, p.tokens, "x").shape(1, p.outputs, "b").neighbours();
    out.rank(2).type(x.t->dtype).shape(0, p.tokens, "x").shape(1, p.outputs, "b").neighbours().distinct();
    a.rank(3).type(x.t->dtype).shape(0, p.adapters, "b").shape(1, p.rank, "b").shape(2, p.inputs, "x").neighbours();
    ids.rank(1).type(TTS_I32).shape(0, p.tokens, "x");
    if (2 * (a.size(1) * a.stride(1) + 64) > 0xffffffffll) unsupported("a: rows " + std::to_string(a.stride(1)) + " apart reach past 4 GiB in one adapter");
    base.present(), x.present(), a.present(), b.present(), ids.present(), out.present();
    if (scales_) {
      Arg scales(scales_, "scales");
      scales.rank(1).type(TTS_F32).shape(0, p.adapters, "b").neighbours().present();
      apart(out, scales);
      p.scales = (const float *)scales.t->ptr;
    }
    const bool in_place = out.first() == base.first() && (out.stride(0) == base.stride(0) || p.tokens <= 1);
    if (!in_place) apart(out, base);
    apart(out, x), apart(out, a), apart(out, b), apart(out, ids);
    check_workspace(workspace, bytes, lora_workspace_bytes(p));
    if (!p.tokens) return hipSuccess;
    p.base = base.t->ptr, p.x = x.t->ptr, p.a = a.t->ptr, p.b = b.t->ptr, p.ids = (const int *)ids.t->ptr, p.out = out.t->ptr;
    p.ld_base = base.stride(0), p.ld_x = x.stride(0), p.ld_out = out.stride(0), p.stride_ids = ids.stride(0);
    p.a_adapter = a.stride(0), p.a_rank = a.stride(1), p.b_adapter = b.stride(0), p.b_col = b.stride(1);
    p.workspace = workspace;
    return launch_lora(p, (hipStream_t)stream);
  });
}

}  // extern "C"
