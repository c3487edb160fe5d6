// A call of rotary positions, with or without norms of the heads: what the kernels get, and the checks on the host.
#pragma once

#include "rows.cuh"

struct ShahdRope {
  int head_dim, rotary, layout;
  float magnitude;
  double turns[128];  // f_i / 2pi
};

namespace shahd {

struct RopeOperand {
  const void* in;
  void* out;
  long long in_row, in_head, out_row, out_head;
  int heads;
};

struct RopeArgs {
  RopeOperand q, k, v;  // v.out is never set: values only go to the cache
  const int* positions;
  const int* offsets;  // null: every row counts
  int n, rows, d, half, interleaved, pieces;
  float magnitude;
  uint16_t* pool;  // null: no cache
  long long page_stride;
  const int* table;
  int max_blocks, pages;
  double turns[128];
};

// Whether 16-byte pieces of 8 values can be used: every address and stride in use is a multiple of 16 bytes; and whether pieces are
// whole: none lies across the rotated part's end or across the halves of the pairs, so that a lane holds both values of its pairs.
struct RopePieces {
  bool vec, whole;
};

// More of a call's pointers than ShahdRopeCall has.
struct MoreBuffer {
  const char* name;
  const void* p;
  size_t align;
};

// The checks of a call, and the kernel's arguments from it. SHAHD_OK with call->rows == 0: there is nothing to do, nothing is set.
inline int PrepareRope(const char* op, const ShahdRope* rope, const ShahdRopeCall* c, const MoreBuffer* more, int count, RopeArgs* out, RopePieces* pieces,
                       DeviceInfo* info, int* device) {
  if (!CheckType(op, c->dtype, true)) return SHAHD_EINVAL;
  const bool q = c->num_heads > 0, k = c->kv_heads > 0, cache = c->cache.pool != nullptr;
  const int d = rope->head_dim;
  if (c->rows < 0 || c->num_heads < 0 || c->kv_heads < 0 || c->num_heads > (1 << 16) || c->kv_heads > (1 << 16) || !(q || k)) {
    SetError("%s: need rows >= 0 and num_heads or kv_heads (got rows=%d num_heads=%d kv_heads=%d)", op, c->rows, c->num_heads,
             c->kv_heads);
    return SHAHD_EINVAL;
  }
  if (c->n > kOpsMaxRows) {
    SetError("%s: too many sequences: %d, at most 2^30", op, c->n);
    return SHAHD_EINVAL;
  }
  if (c->n < 0 || (cache && (c->n < 1 || !c->offsets)) || (c->offsets && c->n < 1)) {
    SetError("%s: offsets, and so a cache, need n >= 1 sequences (got n=%d)", op, c->n);
    return SHAHD_EINVAL;
  }
  if (cache && (!k || !CheckCache(op, c->cache, c->kv_heads, d))) {
    if (!k) SetError("%s: a cache needs kv_heads", op);
    return SHAHD_EINVAL;
  }
  if (k && !cache && !c->k_out.data) {
    SetError("%s: keys need k_out or a cache", op);
    return SHAHD_EINVAL;
  }
  if ((q && (!CheckRows(op, "q", c->q, c->rows, c->num_heads, d, 1) || !CheckRows(op, "q_out", c->q_out, c->rows, c->num_heads, d, 1, true))) ||
      (k && !CheckRows(op, "k", c->k, c->rows, c->kv_heads, d, 1)) ||
      (k && c->k_out.data && !CheckRows(op, "k_out", c->k_out, c->rows, c->kv_heads, d, 1, true)) ||
      (cache && !CheckRows(op, "v", c->v, c->rows, c->kv_heads, d, 1)))
    return SHAHD_EINVAL;
  if (c->rows == 0) return SHAHD_OK;
  const size_t size = TypeBytes(c->dtype);
  BufferCheck b(op);
  b.Add("positions", c->positions, 4);
  if (c->offsets) b.Add("offsets", c->offsets, 4);
  if (q) {
    b.Add("q", c->q.data, size);
    b.Add("q_out", c->q_out.data, size);
  }
  if (k) b.Add("k", c->k.data, size);
  if (k && c->k_out.data) b.Add("k_out", c->k_out.data, size);
  if (cache) {
    b.Add("v", c->v.data, size);
    b.Add("cache.pool", c->cache.pool, 16);
    b.Add("cache.block_table", c->cache.block_table, 4);
  }
  for (int i = 0; i < count; i++) b.Add(more[i].name, more[i].p, more[i].align);
  if (b.rc != SHAHD_OK) return b.rc;
  *device = b.device;
  *info = InfoOf(b.device);
  if (!info->usable) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  RopeArgs a = {};
  // With whole pieces on both sides of the rotated part's end and of the pairs' halves a lane holds both values of its pairs; otherwise
  // shared memory brings them together (57344 f16 rows of 32 + 8 heads of 128 with 126 values turned: 227 us, value by value 862;
  // with 54 243 and 1363).
  bool vec = d % 8 == 0;
  const bool whole = rope->layout == SHAHD_ROPE_HALF ? d % 16 == 0 && rope->rotary % 16 == 0 : rope->rotary % 8 == 0;
  const auto operand = [&](const ShahdRows& in, const ShahdRows& out_rows, int heads) {
    for (const ShahdRows* r : {&in, &out_rows})
      if (r->data)
        vec = vec && reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->row_stride * size % 16 == 0 && r->head_stride * size % 16 == 0;
    return RopeOperand{in.data, out_rows.data, in.row_stride, in.head_stride, out_rows.row_stride, out_rows.head_stride, heads};
  };
  if (q) a.q = operand(c->q, c->q_out, c->num_heads);
  if (k) a.k = operand(c->k, c->k_out, c->kv_heads);
  if (cache) a.v = operand(c->v, ShahdRows{}, c->kv_heads);
  a.positions = c->positions;
  a.offsets = c->offsets;
  a.n = c->n;
  a.rows = c->rows;
  a.d = d;
  a.half = rope->rotary / 2;
  a.interleaved = rope->layout == SHAHD_ROPE_INTERLEAVED;
  a.magnitude = rope->magnitude;
  if (cache) {
    a.pool = static_cast<uint16_t*>(c->cache.pool);
    a.page_stride = c->cache.page_stride;
    a.table = c->cache.block_table;
    a.max_blocks = c->cache.max_blocks;
    a.pages = c->cache.pages;
  }
  std::copy(rope->turns, rope->turns + a.half, a.turns);
  *out = a;
  *pieces = {vec, whole};
  return SHAHD_OK;
}

}  // namespace shahd
