// The C entries of the operators whose weights are picked per row: what include/tts_hip.h says about their arguments is checked
// here, on the host, before anything is launched.
#include "row_ops.h"

#include <stdexcept>
#include <string>

#include "../../include/tts_hip.h"

namespace tts {
tts_status report(tts_status st, const std::string &msg);  // runtime.hip: sets tts_last_error
}

using namespace tts;

namespace {

struct Refused : std::runtime_error {
  tts_status status;
  Refused(tts_status st, const std::string &msg) : std::runtime_error(msg), status(st) {}
};

[[noreturn]] void invalid(const std::string &msg) { throw Refused(TTS_INVALID, msg); }
[[noreturn]] void unsupported(const std::string &msg) { throw Refused(TTS_UNSUPPORTED, msg); }

int64_t item_size(int dtype) { return dtype == TTS_I8 ? 1 : dtype == TTS_F16 || dtype == TTS_BF16 ? 2 : 4; }
const char *type_name(int dtype) {
  static const char *names[] = {"f32", "f16", "bf16", "i8", "i32"};
  return dtype >= 0 && dtype < 5 ? names[dtype] : "an unknown type";
}

constexpr int64_t MOST_SIZE = (int64_t)1 << 30;  // of a dimension: sums of two fit 32 bits

constexpr int64_t MOST_WIDTH = (int64_t)1 << 24;  // of a layer: its tiles fit 32 bits, and a token's sums a grid

// one argument of a call, by its name
struct Arg {
  const tts_tensor *t;
  std::string name;
  Arg(const tts_tensor *tensor, const char *n) : t(tensor), name(n) {
    if (!t) invalid(name + " is missing");
    if (t->dtype < TTS_F32 || t->dtype > TTS_I32) invalid(name + " has an unknown type");
    if (t->rank < 1 || t->rank > 3) invalid(name + " has " + std::to_string(t->rank) + " dimensions");
    for (int d = 0; d < t->rank; d++) {
      if (t->shape[d] < 0 || t->shape[d] > MOST_SIZE) invalid(name + ": dimension " + std::to_string(d) + " is " + std::to_string(t->shape[d]));
      if (t->stride[d] < 0 || t->stride[d] > ((int64_t)1 << 48)) invalid(name + ": stride " + std::to_string(d) + " is " + std::to_string(t->stride[d]));
    }
    if ((uintptr_t)t->ptr % item_size(t->dtype)) invalid(name + " is not aligned to its elements");
  }
  int64_t size(int d) const { return t->shape[d]; }
  int64_t stride(int d) const { return t->stride[d]; }
  Arg &rank(int n) {
    if (t->rank != n) invalid(name + " has " + std::to_string(t->rank) + " dimensions, not " + std::to_string(n));
    return *this;
  }
  Arg &type(int want) {
    if (t->dtype != want) invalid(name + " is " + type_name(t->dtype) + ", not " + type_name(want));
    return *this;
  }
  Arg &shape(int d, int64_t want, const char *like) {
    if (size(d) != want) invalid(name + ": dimension " + std::to_string(d) + " is " + std::to_string(size(d)) + ", but " + like + " says " + std::to_string(want));
    return *this;
  }
  Arg &neighbours() {  // the elements of a row
    const int d = t->rank - 1;
    if (stride(d) != 1 && size(d) > 1) invalid(name + ": its last dimension has stride " + std::to_string(stride(d)) + ", not 1");
    return *this;
  }
  Arg &some(int d) {
    if (size(d) < 1) invalid(name + ": dimension " + std::to_string(d) + " is empty");
    return *this;
  }
  // nothing in it is there twice (for what is written)
  Arg &distinct() {
    if (t->rank == 2 && size(0) > 1 && stride(0) < size(1)) invalid(name + ": its rows overlap");
    return *this;
  }
  bool empty() const {
    for (int d = 0; d < t->rank; d++)
      if (size(d) == 0) return true;
    return false;
  }
  void present() const {
    if (!t->ptr && !empty()) invalid(name + " is a null pointer");
  }
  uintptr_t first() const { return (uintptr_t)t->ptr; }
  uintptr_t end() const {  // the byte behind its last element
    int64_t last = 0;
    for (int d = 0; d < t->rank; d++) last += (size(d) - 1) * stride(d);
    return first() + (uintptr_t)(last + 1) * item_size(t->dtype);
  }
};

// whether they share memory: by their extents, except that columns of one buffer with rows of the same distance are told apart
bool overlap(const Arg &a, const Arg &b) {
  if (a.empty() || b.empty() || a.end() <= b.first() || b.end() <= a.first()) return false;
  if (a.t->rank == 2 && b.t->rank == 2 && item_size(a.t->dtype) == item_size(b.t->dtype) && a.stride(0) == b.stride(0) && a.stride(0) > 0 && a.stride(1) == 1 && b.stride(1) == 1) {
    const int64_t item = item_size(a.t->dtype), pitch = a.stride(0) * item;
    const int64_t apart = ((int64_t)(b.first() - a.first()) % pitch + pitch) % pitch;
    if (apart >= a.size(1) * item && apart + b.size(1) * item <= pitch) return false;
  }
  return true;
}
void apart(const Arg &out, const Arg &in) {
  if (overlap(out, in)) invalid(out.name + " shares memory with " + in.name);
}

void half_type(const Arg &a) {
  if (a.t->dtype == TTS_F32) unsupported(a.name + " is f32: the operator takes f16 and bf16");
  if (a.t->dtype != TTS_F16 && a.t->dtype != TTS_BF16) invalid(a.name + " is " + std::string(type_name(a.t->dtype)) + ", not f16 or bf16");
}

void check_workspace(void *workspace, size_t bytes, size_t need) {
  if (bytes < need) invalid("the workspace has " + std::to_string(bytes) + " bytes, and " + std::to_string(need) + " are needed");
  if (need && !workspace) invalid("the workspace is a null pointer");
  if ((uintptr_t)workspace % 256) invalid("the workspace is not aligned to 256 bytes");
}

template <class F>
tts_status guarded(const char *who, F &&f) {
  try {
    const hipError_t e = f();
    return e == hipSuccess ? TTS_OK : report(TTS_HIP_ERROR, std::string(who) + ": " + hipGetErrorString(e));
  } catch (const Refused &e) {
    return report(e.status, std::string(who) + ": " + e.what());
  } catch (const std::exception &e) {
    return report(TTS_INVALID, std::string(who) + ": " + e.what());
  }
}

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
