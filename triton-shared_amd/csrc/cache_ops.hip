// The C entries of the attention part of a decode step over a cache held in 4 bits: what include/tts_hip.h says about their arguments is
// checked here, on the host, before anything is launched.
#include "cache_ops.h"

#include <algorithm>
#include <climits>
#include <cmath>

#include "op_args.h"

using namespace tts;

namespace {

Kv4Cache cache_of(const Arg &a, int64_t dim) {
  if (a.t->rank != 3) invalid(a.name + " has " + std::to_string(a.t->rank) + " dimensions, not 3");
  half_type(a);
  if (dim < 32 || dim > 256 || dim % 32) unsupported(a.name + ": heads of " + std::to_string(dim) + " elements, not a multiple of 32 up to 256");
  const int64_t bytes = a.size(2) * 2, page = bytes / (dim + 8);
  if (page < 1 || bytes % (dim + 8)) invalid(a.name + ": dimension 2 is " + std::to_string(a.size(2)) + ", not a number of tokens times " + std::to_string((dim + 8) / 2) + " for heads of " + std::to_string(dim));
  if (page % 16) unsupported(a.name + ": pages of " + std::to_string(page) + " tokens, not a multiple of 16");
  if (a.t->stride[2] != 1) invalid(a.name + ": its last dimension has stride " + std::to_string(a.stride(2)) + ", not 1");
  if (a.size(0) < 1 || a.size(1) < 1) invalid(a.name + " is empty");
  if (a.size(0) * page > INT_MAX) unsupported(a.name + ": " + std::to_string(a.size(0) * page) + " slots, more than 32 bits number");
  if (a.size(1) > 65535) unsupported(a.name + ": " + std::to_string(a.size(1)) + " heads");
  if (a.first() % 16 || (a.size(0) > 1 && a.stride(0) % 8) || (a.size(1) > 1 && a.stride(1) % 8)) invalid(a.name + ": its pages and heads do not begin at multiples of 16 bytes");
  a.present();
  Kv4Cache c = {};
  c.base = a.t->ptr, c.page_bytes = a.stride(0) * 2, c.head_bytes = a.stride(1) * 2;
  c.pages = (int)a.size(0), c.heads = (int)a.size(1), c.page = (int)page, c.dim = (int)dim, c.bf16 = a.t->dtype == TTS_BF16, c.by_page = fast_div((uint32_t)page);
  return c;
}

// keys and values, or what is to hold them
Kv4RowsParams rows_of(Arg &cache, Arg &k, Arg &v, Arg &slots) {
  k.rank(3).neighbours();
  Kv4RowsParams p = {};
  p.cache = cache_of(cache, k.size(2));
  k.type(cache.t->dtype).shape(1, p.cache.heads, "cache").present();
  v.rank(3).type(cache.t->dtype).shape(0, k.size(0), "k").shape(1, p.cache.heads, "cache").shape(2, k.size(2), "k").neighbours().present();
  slots.rank(1).type(TTS_I32).shape(0, k.size(0), "k").neighbours().present();
  p.k = k.t->ptr, p.v = v.t->ptr, p.slots = (const int *)slots.t->ptr;
  p.k_token = k.stride(0), p.k_head = k.stride(1), p.v_token = v.stride(0), p.v_head = v.stride(1), p.tokens = k.size(0);
  return p;
}

// out in the place of x itself, or apart from it
void same_or_apart(const Arg &out, const Arg &x) {
  const bool same = out.first() == x.first() && (out.stride(0) == x.stride(0) || x.size(0) <= 1) && (out.stride(1) == x.stride(1) || x.size(1) <= 1);
  if (!same) apart(out, x);
}

struct Attend {
  Arg q, cache, table;
  AttendParams p = {};
  Attend(const tts_tensor *q_, const tts_tensor *cache_, const tts_tensor *table_, int window, int64_t longest) : q(q_, "q"), cache(cache_, "cache"), table(table_, "table") {
    q.rank(3).neighbours();
    p.cache = cache_of(cache, q.size(2));
    q.type(cache.t->dtype);
    table.rank(2).type(TTS_I32).neighbours();
    p.tokens = q.size(0), p.heads = (int)q.size(1), p.requests = (int)table.size(0), p.window = window;
    if (p.heads < 1 || p.heads % p.cache.heads) invalid("q: " + std::to_string(p.heads) + " heads, not a multiple of the cache's " + std::to_string(p.cache.heads));
    p.group = p.heads / p.cache.heads;
    if (window < 0) invalid("the window is " + std::to_string(window));
    if (longest < 0) invalid("longest is " + std::to_string(longest));
    if (p.tokens * p.heads > ((int64_t)1 << 26)) unsupported("q: " + std::to_string(p.tokens) + " rows of " + std::to_string(p.heads) + " heads");
    if (p.requests > (1 << 20)) unsupported("table: " + std::to_string(p.requests) + " requests");
    const int64_t most = table.size(1) * p.cache.page;
    if (most > INT_MAX / 2) unsupported("table: places for " + std::to_string(most) + " tokens, 2^30 and more");  // (what is added to a token's number stays in 32 bits)
    p.places = (int)most;
    p.by_group = fast_div(p.group), p.by_heads = fast_div(p.heads);
    p.plan = plan_attend(p.tokens, p.requests, p.heads, p.cache.heads, p.cache.dim, longest ? std::min(longest, most) : most, window);
    // (a launch of 2^32 lanes and more starts only their remainder; the rows of no request have 8 workgroups besides)
    if ((p.plan.items + p.plan.extra) * p.cache.heads + 8 >= (1 << 24)) unsupported(std::to_string(p.requests) + " requests of " + std::to_string(p.cache.heads) + " heads: more workgroups than a launch has");
  }
};

}  // namespace

extern "C" {

tts_status tts_page_slots(const tts_tensor *table_, const tts_tensor *lengths_, const tts_tensor *fresh_, const tts_tensor *free_, const tts_tensor *count_, int page,
                          const tts_tensor *slots_, const tts_tensor *positions_, const tts_tensor *owners_, const tts_tensor *starts_, const tts_tensor *left_, void *stream) {
  return guarded("tts_page_slots", [&]() -> hipError_t {
    Arg table(table_, "table"), lengths(lengths_, "lengths"), fresh(fresh_, "fresh"), free(free_, "free"), count(count_, "count");
    Arg slots(slots_, "slots"), positions(positions_, "positions"), owners(owners_, "owners"), starts(starts_, "starts"), left(left_, "left");
    table.rank(2).type(TTS_I32).neighbours().distinct();
    if (table.size(0) > SLOTS_MAX_REQUESTS) unsupported("table: " + std::to_string(table.size(0)) + " requests, more than " + std::to_string(SLOTS_MAX_REQUESTS));
    if (page < 1) invalid("a page of " + std::to_string(page) + " tokens");
    lengths.rank(1).type(TTS_I32).shape(0, table.size(0), "table").neighbours();
    fresh.rank(1).type(TTS_I32).shape(0, table.size(0), "table").neighbours();
    free.rank(1).type(TTS_I32).neighbours();
    count.rank(1).type(TTS_I32).shape(0, 1, "one number");
    slots.rank(1).type(TTS_I32).neighbours();
    positions.rank(1).type(TTS_I32).shape(0, slots.size(0), "slots").neighbours();
    owners.rank(1).type(TTS_I32).shape(0, slots.size(0), "slots").neighbours();
    starts.rank(1).type(TTS_I32).shape(0, table.size(0) + 1, "table").neighbours();
    left.rank(1).type(TTS_I32).shape(0, 1, "one number");
    const Arg *in[] = {&lengths, &fresh, &free, &count}, *out[] = {&table, &slots, &positions, &owners, &starts, &left};
    for (const Arg *a : in) a->present();
    for (const Arg *a : out) a->present();
    // (every workgroup reads all of the inputs, and others may have written by then)
    for (const Arg *o : out)
      for (const Arg *i : in) apart(*o, *i);
    for (int i = 0; i < 6; i++)
      for (int j = 0; j < i; j++) apart(*out[i], *out[j]);
    SlotsParams p = {};
    p.table = (int *)table.t->ptr, p.lengths = (const int *)lengths.t->ptr, p.fresh = (const int *)fresh.t->ptr, p.free = (const int *)free.t->ptr, p.count = (const int *)count.t->ptr;
    p.slots = (int *)slots.t->ptr, p.positions = (int *)positions.t->ptr, p.owners = (int *)owners.t->ptr, p.starts = (int *)starts.t->ptr, p.left = (int *)left.t->ptr;
    p.ld_table = table.stride(0), p.rows = slots.size(0), p.requests = (int)table.size(0), p.columns = (int)table.size(1), p.stack = (int)free.size(0), p.page = page;
    return launch_slots(p, (hipStream_t)stream);
  });
}

tts_status tts_qk_norm_rope(const tts_tensor *q_, const tts_tensor *k_, const tts_tensor *positions_, const tts_tensor *cos_sin_, const tts_tensor *w_q_, const tts_tensor *w_k_, double eps,
                            int interleaved, int clear, const tts_tensor *q_out_, const tts_tensor *k_out_, void *stream) {
  return guarded("tts_qk_norm_rope", [&]() -> hipError_t {
    Arg q(q_, "q"), k(k_, "k"), positions(positions_, "positions"), cos_sin(cos_sin_, "cos_sin"), q_out(q_out_, "q_out"), k_out(k_out_, "k_out");
    q.rank(3).neighbours();
    const int type = q.t->dtype;
    if (type != TTS_F32 && type != TTS_F16 && type != TTS_BF16) invalid("q is " + std::string(type_name(type)) + ", not f32, f16 or bf16");
    const int64_t tokens = q.size(0), dim = q.size(2);
    if (dim < 2 || dim % 2) invalid("q: heads of " + std::to_string(dim) + " elements, not an even number");
    if (dim > ROPE_MAX_DIM) unsupported("q: heads of " + std::to_string(dim) + " elements, more than " + std::to_string(ROPE_MAX_DIM));
    if (q.size(1) > 65535) unsupported("q: " + std::to_string(q.size(1)) + " heads");
    k.rank(3).type(type).shape(0, tokens, "q").shape(2, dim, "q").neighbours();
    if (k.size(1) > 65535) unsupported("k: " + std::to_string(k.size(1)) + " heads");
    q_out.rank(3).type(type).shape(0, tokens, "q").shape(1, q.size(1), "q").shape(2, dim, "q").neighbours().distinct();
    k_out.rank(3).type(type).shape(0, tokens, "q").shape(1, k.size(1), "k").shape(2, dim, "q").neighbours().distinct();
    positions.rank(1).type(TTS_I32).shape(0, tokens, "q").neighbours();
    cos_sin.rank(2).type(TTS_F32).neighbours();
    const int64_t rotary = cos_sin.size(1);
    if (rotary < 2 || rotary % 2 || rotary > dim) invalid("cos_sin: dimension 1 is " + std::to_string(rotary) + ", not an even number up to q's " + std::to_string(dim));
    if (!(eps >= 0.0) || !std::isfinite((float)eps)) invalid("eps is " + std::to_string(eps));
    RopeParams p = {};
    p.w_f32 = 0;
    if (!w_q_ != !w_k_) invalid(std::string(w_q_ ? "w_k" : "w_q") + " is missing");
    if (w_q_) {
      Arg w_q(w_q_, "w_q"), w_k(w_k_, "w_k");
      if (w_q.t->dtype != TTS_F32) w_q.type(type);
      w_q.rank(1).shape(0, dim, "q").neighbours().present();
      w_k.rank(1).type(w_q.t->dtype).shape(0, dim, "q").neighbours().present();
      for (const Arg *w : {&w_q, &w_k}) apart(q_out, *w), apart(k_out, *w);
      p.w_q = w_q.t->ptr, p.w_k = w_k.t->ptr, p.w_f32 = w_q.t->dtype == TTS_F32;
    }
    for (const Arg *a : {&q, &k, &positions, &cos_sin, &q_out, &k_out}) a->present();
    same_or_apart(q_out, q), same_or_apart(k_out, k);
    apart(q_out, k), apart(k_out, q), apart(q_out, k_out);
    for (const Arg *out : {&q_out, &k_out}) apart(*out, positions), apart(*out, cos_sin);
    if (!tokens || q.size(1) + k.size(1) == 0) return hipSuccess;
    if (!cos_sin.size(0) && !clear) return hipSuccess;  // no position is in the table
    p.q = q.t->ptr, p.k = k.t->ptr, p.q_out = q_out.t->ptr, p.k_out = k_out.t->ptr, p.positions = (const int *)positions.t->ptr, p.cos_sin = (const float *)cos_sin.t->ptr;
    p.q_token = q.stride(0), p.q_head = q.stride(1), p.k_token = k.stride(0), p.k_head = k.stride(1);
    p.qo_token = q_out.stride(0), p.qo_head = q_out.stride(1), p.ko_token = k_out.stride(0), p.ko_head = k_out.stride(1), p.ld_cos_sin = cos_sin.stride(0);
    p.tokens = tokens, p.heads = (int)q.size(1), p.kv_heads = (int)k.size(1), p.dim = (int)dim, p.rotary = (int)rotary, p.places = (int)cos_sin.size(0);
    p.eps = (float)eps, p.elem = type, p.interleaved = interleaved != 0, p.clear = clear != 0;
    return launch_rope(p, (hipStream_t)stream);
  });
}

tts_status tts_kv4_write(const tts_tensor *cache_, const tts_tensor *k_, const tts_tensor *v_, const tts_tensor *slots_, void *stream) {
  return guarded("tts_kv4_write", [&]() -> hipError_t {
    Arg cache(cache_, "cache"), k(k_, "k"), v(v_, "v"), slots(slots_, "slots");
    const Kv4RowsParams p = rows_of(cache, k, v, slots);
    cache.distinct();
    apart(cache, k), apart(cache, v), apart(cache, slots);
    return p.tokens ? launch_kv4_write(p, (hipStream_t)stream) : hipSuccess;
  });
}

tts_status tts_kv4_read(const tts_tensor *cache_, const tts_tensor *slots_, const tts_tensor *k_, const tts_tensor *v_, void *stream) {
  return guarded("tts_kv4_read", [&]() -> hipError_t {
    Arg cache(cache_, "cache"), k(k_, "k"), v(v_, "v"), slots(slots_, "slots");
    const Kv4RowsParams p = rows_of(cache, k, v, slots);
    k.distinct(), v.distinct();
    apart(k, cache), apart(v, cache), apart(k, slots), apart(v, slots), apart(k, v);
    return p.tokens ? launch_kv4_read(p, (hipStream_t)stream) : hipSuccess;
  });
}

tts_status tts_kv4_attention_workspace(const tts_tensor *q, const tts_tensor *cache, const tts_tensor *table, int window, int64_t longest, size_t *bytes) {
  return guarded("tts_kv4_attention_workspace", [&]() -> hipError_t {
    if (!bytes) invalid("bytes is missing");
    const Attend a(q, cache, table, window, longest);
    *bytes = attend_workspace_bytes(a.p.plan, a.p.cache.heads, a.p.cache.dim);
    return hipSuccess;
  });
}

tts_status tts_kv4_attention(const tts_tensor *q_, const tts_tensor *cache_, const tts_tensor *table_, const tts_tensor *lengths_, const tts_tensor *starts_, double scale, int window,
                             int64_t longest, int clear, const tts_tensor *out_, void *workspace, size_t bytes, void *stream) {
  return guarded("tts_kv4_attention", [&]() -> hipError_t {
    Attend a(q_, cache_, table_, window, longest);
    Arg lengths(lengths_, "lengths"), starts(starts_, "starts"), out(out_, "out");
    AttendParams &p = a.p;
    lengths.rank(1).type(TTS_I32).shape(0, p.requests, "table").neighbours();
    starts.rank(1).type(TTS_I32).shape(0, (int64_t)p.requests + 1, "table").neighbours();
    out.rank(3).type(a.q.t->dtype).shape(0, p.tokens, "q").shape(1, p.heads, "q").shape(2, p.cache.dim, "q").neighbours().distinct();
    if (!std::isfinite((float)scale)) invalid("the scale is " + std::to_string(scale));
    for (const Arg *x : {&a.q, &a.table, &lengths, &starts, &out}) x->present();
    same_or_apart(out, a.q);
    apart(out, a.cache), apart(out, a.table), apart(out, lengths), apart(out, starts);
    const size_t need = attend_workspace_bytes(p.plan, p.cache.heads, p.cache.dim);
    check_workspace(workspace, bytes, need);
    if (!p.tokens || (!p.requests && !clear)) return hipSuccess;
    p.q = a.q.t->ptr, p.out = out.t->ptr, p.table = (const int *)a.table.t->ptr, p.lengths = (const int *)lengths.t->ptr, p.starts = (const int *)starts.t->ptr;
    p.q_token = a.q.stride(0), p.q_head = a.q.stride(1), p.o_token = out.stride(0), p.o_head = out.stride(1), p.ld_table = a.table.stride(0);
    p.scale = (float)scale, p.clear = clear != 0;
    p.parts = (float *)workspace, p.stats = p.parts + ((p.plan.items + p.plan.extra) * p.cache.heads << p.plan.tile_log) * p.cache.dim;
    return launch_attend(p, (hipStream_t)stream);
  });
}

}  // extern "C"
