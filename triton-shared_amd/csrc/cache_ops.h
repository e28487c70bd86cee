// The attention part of a decode step over a paged cache held in 4 bits: slots from lengths, norms with the rotation by position, the
// cache's writing and reading, and the attention.  Parameter blocks are plain data that the C entries (cache_ops.hip) have checked.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tts {

// n / divisor for 0 <= n < 2^31 is n * mul >> shift
struct FastDiv {
  uint32_t mul;
  int shift;
};
inline FastDiv fast_div(uint32_t divisor) {
  int up = 0;
  while (((uint64_t)1 << up) < divisor) up++;
  return {(uint32_t)((((uint64_t)1 << (31 + up)) + divisor - 1) / divisor), 31 + up};
}

__device__ __forceinline__ int divided(int n, FastDiv by) { return (int)(((uint64_t)(uint32_t)n * by.mul) >> by.shift); }

constexpr int SLOTS_MAX_REQUESTS = 4096;

struct SlotsParams {
  int *table;           // [requests, columns]
  const int *lengths, *fresh;
  const int *free, *count;
  int *slots, *positions, *owners;  // [rows]
  int *starts;          // [requests + 1]
  int *left;            // [1]
  int64_t ld_table, rows;
  int requests, columns, stack, page;
};
hipError_t launch_slots(const SlotsParams &p, hipStream_t s);

constexpr int ROPE_MAX_DIM = 512;

struct RopeParams {
  const void *q, *k;    // [tokens, heads, dim], [tokens, kv_heads, dim]
  void *q_out, *k_out;
  const int *positions; // [tokens]
  const float *cos_sin; // [places, rotary]: cosines of rotary / 2 angles, and their sines
  const void *w_q, *w_k;  // [dim] or null
  int64_t q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head, ld_cos_sin;
  int64_t tokens;
  int heads, kv_heads, dim, rotary, places;
  float eps;
  int elem;             // ElemKind of q and k
  int w_f32, interleaved, clear;
  FastDiv by_all_heads; // (the launch's own)
};
hipError_t launch_rope(const RopeParams &p, hipStream_t s);

// The cache: of a page and a head, KV4_... bytes in this order, `page` tokens each:
//   keys' codes      page rows of dim / 2 bytes: 32-bit words of 8 neighbouring elements, element 2 i in bits 4 i .. 4 i + 3, element 2 i + 1 in bits 16 + 4 i ..
//   values' codes    the same, element i in bits 4 i ..
//   keys' pairs      page words: the step in the lower half, the lowest value in the upper one, both of the cache's type
//   values' pairs
// An element is code * step + lowest.  (The order of a word's codes is the one in which the attention's operands come out of it.)
struct Kv4Cache {
  void *base;
  int64_t page_bytes, head_bytes;  // from page to page, from head to head
  int pages, heads, page, dim, bf16;
  FastDiv by_page;
};

struct Kv4RowsParams {
  Kv4Cache cache;
  void *k, *v;          // [tokens, heads, dim]
  const int *slots;     // [tokens]
  int64_t k_token, k_head, v_token, v_head, tokens;
  FastDiv by_heads;     // of keys and of values (the launch's own)
};
hipError_t launch_kv4_write(const Kv4RowsParams &p, hipStream_t s);
hipError_t launch_kv4_read(const Kv4RowsParams &p, hipStream_t s);

// How a call's rows and lengths are dealt to workgroups (kernels_kv4_attend.hip)
enum AttendOwn { OWN_BLOCKS = 0, OWN_ROWS = 1, OWN_HEADS = 2 };
struct AttendPlan {
  int own;              // AttendOwn: what a workgroup's four wavefronts have of their own
  int tile_log;         // log2 of a workgroup's rows
  int64_t items;        // tiles of rows per head of the cache, at most
  int64_t extra;        // workgroups beyond one for each of them: slices of their tokens (0: none are sliced)
  float over_extra;     // 1 / extra
};

struct AttendParams {
  Kv4Cache cache;
  const void *q;        // [tokens, heads, dim]
  void *out;
  const int *table;     // [requests, columns]
  const int *lengths;   // [requests]
  const int *starts;    // [requests + 1]
  int64_t q_token, q_head, o_token, o_head, ld_table, tokens;
  int requests, heads, group;
  int places;           // tokens that a request's row of the table has places for
  FastDiv by_group, by_heads, by_per_item;  // (the last: workgroups per tile or slice, the launch's own)
  int window;           // 0: none
  int clear;            // rows of no request get zeros
  float scale;
  AttendPlan plan;
  float *parts;         // [workgroups, tile, dim] of what is sliced
  float *stats;         // [workgroups, tile, 2]
};
AttendPlan plan_attend(int64_t tokens, int requests, int heads, int kv_heads, int dim, int64_t longest, int window);
size_t attend_workspace_bytes(const AttendPlan &plan, int kv_heads, int dim);
hipError_t launch_attend(const AttendParams &p, hipStream_t s);

}  // namespace tts
