// Rotary positions on packed rows (ApplyRope, Brain/Ops/RotaryEmbedding.ts:63-75, for prompts of different lengths
// and for the layouts and scalings that the session's fused RoPE does not have), with the append of the rotated keys
// and the values to a paged cache.
//
// The first r of a head's d values are r/2 pairs; pair i of a row at position p is turned by p * f_i:
//   (a, b) -> m (a cos - b sin, a sin + b cos),   f_i = base^(-2i/r), scaled as the plan says, m the plan's magnitude,
// with pairs (2i, 2i+1) or (i, i + r/2). Angles: the turn p * f_i / 2pi is formed in 64 bits and only its fraction is
// rounded to 32, so a position of 10^6 loses nothing (in 32 bits the angle alone would be off by 0.03).
//
// Bound by memory: each value is read once and written once. A block takes a few rows: it first writes the rows'
// (cos, sin) table to shared memory, one sincospi per (row, pair) for all heads together, then its threads go
// over 8-value pieces of all heads of q, k and v with 16-byte accesses. Operands whose address, strides or pair count
// do not allow 16-byte pieces go through one pair per thread.
#pragma once

#include "ops_common.cuh"

struct ShahdRope {
  int head_dim, rotary, layout;
  float magnitude;
  double turns[128];  // f_i / 2pi
};

namespace shahd {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxRows = 16;   // rows of a block
constexpr int kRopeTable = 512;    // (row, pair) entries of a block's table

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
  int n, rows, d, half, interleaved, rows_per_block, pieces, shift;
  float magnitude;
  uint16_t* pool;  // null: no cache
  long long page_stride;
  const int* table;
  int max_blocks, pages;
  double turns[128];
};

template <class T>
__device__ __forceinline__ float ToFloat(T x) {
  return float(x);
}
template <class T>
__device__ __forceinline__ T FromFloat(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <class T>
__device__ __forceinline__ void Load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = ToFloat(h[i]);
  }
}
template <class T>
__device__ __forceinline__ void Store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 u;
    T* h = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = FromFloat<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// The sequence that holds packed row `row`: the last s with offsets[s] <= row (empty sequences before it share its start).
__device__ __forceinline__ int SequenceOf(const int* offsets, int n, int row) {
  int lo = 0, hi = n;  // offsets[lo] <= row < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// T: the operands' type, C: the cache's. VEC: 16-byte pieces.
template <class T, class C, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) RopeKernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 turn[kRopeTable];
  __shared__ int pos[kRopeMaxRows];
  __shared__ long long at[kRopeMaxRows];  // the row's place in the cache (kv head 0, K), or -1
  GridDepWait();
  GridDepLaunch();
  const int r0 = blockIdx.x * a.rows_per_block, nr = min(a.rows_per_block, a.rows - r0);
  if (threadIdx.x < nr) {
    const int row = r0 + threadIdx.x;
    int p = a.positions[row];
    if (a.offsets && (row < a.offsets[0] || row >= a.offsets[a.n])) p = -1;
    long long c = -1;
    if (a.pool && p >= 0 && (p >> 6) < a.max_blocks) {
      const int page = a.table[(long long)SequenceOf(a.offsets, a.n, row) * a.max_blocks + (p >> 6)];
      if (page >= 0 && page < a.pages) c = page * a.page_stride + (long long)(p & 63) * a.d;
    }
    pos[threadIdx.x] = p;
    at[threadIdx.x] = c;
  }
  for (int e = threadIdx.x; e < nr * a.half; e += kRopeThreads) {
    const int r = e / a.half, i = e - r * a.half;
    const double t = (double)max(a.positions[r0 + r], 0) * a.turns[i];
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    turn[e] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int per_row = heads * a.pieces;
  const int d = a.d, half = a.half;
  for (int e = threadIdx.x; e < nr * per_row; e += kRopeThreads) {
    const int r = e / per_row;
    const int rest = e - r * per_row;
    int h = a.shift >= 0 ? rest >> a.shift : rest / a.pieces;
    const int piece = rest - h * a.pieces;
    if (pos[r] < 0) continue;
    const RopeOperand* o = &a.q;
    int kv = -1;
    if (h >= a.q.heads) {
      h -= a.q.heads;
      o = &a.k;
      kv = 0;
      if (h >= a.k.heads) {
        h -= a.k.heads;
        o = &a.v;
        kv = 1;
      }
    }
    const int row = r0 + r;
    const T* in = static_cast<const T*>(o->in) + row * o->in_row + h * o->in_head;
    T* out = o->out ? static_cast<T*>(o->out) + row * o->out_row + h * o->out_head : nullptr;
    C* cache = kv >= 0 && at[r] >= 0 ? reinterpret_cast<C*>(a.pool) + at[r] + (long long)(2 * h + kv) * kOpsPage * d : nullptr;
    const float2* tr = turn + r * half;
    if constexpr (VEC) {
      float x[8], y[8];
      const bool paired = !a.interleaved && piece * 8 < half;  // this piece stands for the one at + half as well
      if (kv == 1 || !(paired || (a.interleaved && piece * 8 < 2 * half))) {  // values, or behind the rotated part
        const int j = a.interleaved || paired ? piece * 8 : piece * 8 + half;
        Load8(in + j, x);
        if (paired) Load8(in + j + half, y);
        if (out) Store8(out + j, x);
        if (cache) {
          Store8(cache + j, x);
          if (paired) Store8(cache + j + half, y);
        }
        continue;
      }
      if (a.interleaved) {
        const int j = piece * 8;
        Load8(in + j, x);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 t = tr[j / 2 + i];
          y[2 * i] = x[2 * i] * t.x - x[2 * i + 1] * t.y;
          y[2 * i + 1] = x[2 * i] * t.y + x[2 * i + 1] * t.x;
        }
        if (out) Store8(out + j, y);
        if (cache) Store8(cache + j, y);
      } else {
        const int j = piece * 8;
        float b[8], z[8];
        Load8(in + j, x);
        Load8(in + j + half, b);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float2 t = tr[j + i];
          y[i] = x[i] * t.x - b[i] * t.y;
          z[i] = x[i] * t.y + b[i] * t.x;
        }
        if (out) {
          Store8(out + j, y);
          Store8(out + j + half, z);
        }
        if (cache) {
          Store8(cache + j, y);
          Store8(cache + j + half, z);
        }
      }
    } else {  // piece: a pair, or one value behind the rotated part
      int j0 = piece, j1 = -1;
      float x, y = 0.f;
      if (piece < half) {
        j0 = a.interleaved ? 2 * piece : piece;
        j1 = a.interleaved ? j0 + 1 : piece + half;
      } else {
        j0 = piece + half;
      }
      x = ToFloat(in[j0]);
      if (j1 >= 0) {
        y = ToFloat(in[j1]);
        if (kv != 1) {
          const float2 t = tr[piece];
          const float u = x * t.x - y * t.y;
          y = x * t.y + y * t.x;
          x = u;
        }
      }
      if (out) {
        out[j0] = FromFloat<T>(x);
        if (j1 >= 0) out[j1] = FromFloat<T>(y);
      }
      if (cache) {
        cache[j0] = FromFloat<C>(x);
        if (j1 >= 0) cache[j1] = FromFloat<C>(y);
      }
    }
  }
}

template <class T, class C>
void LaunchRope(const RopeArgs& a, bool vec, int blocks, cudaStream_t st) {
  if (vec) LaunchPdl(RopeKernel<T, C, true>, dim3(blocks), dim3(kRopeThreads), 0, st, a);
  else LaunchPdl(RopeKernel<T, C, false>, dim3(blocks), dim3(kRopeThreads), 0, st, a);
}

}  // namespace shahd

extern "C" {

int shahd_rope_create(const ShahdRopeCfg* cfg, ShahdRope** out) {
  using namespace shahd;
  const char* op = "shahd_rope_create";
  ClearError();
  if (!cfg || !out) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  *out = nullptr;
  const int r = cfg->rotary_dim;
  if (cfg->head_dim < 2 || cfg->head_dim > 256 || r < 2 || r > cfg->head_dim || r % 2 != 0) {
    SetError("%s: need 2 <= head_dim <= 256 and an even rotary_dim in 2 .. head_dim (got %d and %d)", op, cfg->head_dim, r);
    return SHAHD_EINVAL;
  }
  if (cfg->layout != SHAHD_ROPE_INTERLEAVED && cfg->layout != SHAHD_ROPE_HALF) {
    SetError("%s: unknown layout %d", op, cfg->layout);
    return SHAHD_EINVAL;
  }
  const bool scaled = cfg->scaling != SHAHD_ROPE_UNSCALED;
  if (!(cfg->base > 1) || !std::isfinite(cfg->base) || !std::isfinite(cfg->magnitude) || cfg->magnitude == 0 ||
      (scaled && (!(cfg->factor >= 1) || !std::isfinite(cfg->factor)))) {
    SetError("%s: need a finite base > 1, a finite magnitude other than 0 and, for a scaling, a finite factor >= 1 (got "
             "base=%g magnitude=%g factor=%g)", op, cfg->base, cfg->magnitude, cfg->factor);
    return SHAHD_EINVAL;
  }
  double low = 0, high = 0;
  switch (cfg->scaling) {
    case SHAHD_ROPE_UNSCALED:
    case SHAHD_ROPE_LINEAR:
      break;
    case SHAHD_ROPE_STRETCHED:
      if (r < 4) {
        SetError("%s: SHAHD_ROPE_STRETCHED needs rotary_dim >= 4, got %d", op, r);
        return SHAHD_EINVAL;
      }
      break;
    case SHAHD_ROPE_BY_PARTS: {
      if (cfg->original_positions < 1 || !(cfg->beta_slow > 0) || !(cfg->beta_fast > cfg->beta_slow) ||
          !std::isfinite(cfg->beta_fast)) {
        SetError("%s: SHAHD_ROPE_BY_PARTS needs original_positions >= 1 and 0 < beta_slow < beta_fast (got %d, %g, %g)", op,
                 cfg->original_positions, cfg->beta_slow, cfg->beta_fast);
        return SHAHD_EINVAL;
      }
      // the pair that makes `turns` turns in the original context: original / (2 pi turns) = base^(2 i / r)
      const auto pair = [&](double turns) {
        return r * std::log(cfg->original_positions / (turns * 2 * M_PI)) / (2 * std::log(cfg->base));
      };
      low = std::max(std::floor(pair(cfg->beta_fast)), 0.0);
      high = std::min(std::ceil(pair(cfg->beta_slow)), r - 1.0);
      break;
    }
    default:
      SetError("%s: unknown scaling %d", op, cfg->scaling);
      return SHAHD_EINVAL;
  }
  ShahdRope* p = new (std::nothrow) ShahdRope();
  if (!p) {
    SetError("%s: out of memory", op);
    return SHAHD_ENOMEM;
  }
  p->head_dim = cfg->head_dim;
  p->rotary = r;
  p->layout = cfg->layout;
  p->magnitude = (float)cfg->magnitude;
  const double base =
      cfg->scaling == SHAHD_ROPE_STRETCHED ? cfg->base * std::pow(cfg->factor, r / (r - 2.0)) : cfg->base;
  for (int i = 0; i < r / 2; i++) {
    double f = std::pow(base, -2.0 * i / r);
    if (cfg->scaling == SHAHD_ROPE_LINEAR) f /= cfg->factor;
    if (cfg->scaling == SHAHD_ROPE_BY_PARTS) {
      const double slow = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
      f = f * (1 - slow) + f / cfg->factor * slow;
    }
    p->turns[i] = f / (2 * M_PI);
  }
  *out = p;
  return SHAHD_OK;
}

int shahd_rope_destroy(ShahdRope* rope) {
  delete rope;
  return SHAHD_OK;
}

int shahd_rope_apply(const ShahdRope* rope, const ShahdRopeCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_rope_apply";
  ClearError();
  if (!rope || !c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  if (!CheckType(op, c->dtype, true)) return SHAHD_EINVAL;
  const bool q = c->num_heads > 0, k = c->kv_heads > 0, cache = c->cache.pool != nullptr;
  const int d = rope->head_dim;
  if (c->rows < 0 || c->num_heads < 0 || c->kv_heads < 0 || c->num_heads > (1 << 16) || c->kv_heads > (1 << 16) || !(q || k)) {
    SetError("%s: need rows >= 0 and num_heads or kv_heads (got rows=%d num_heads=%d kv_heads=%d)", op, c->rows, c->num_heads,
             c->kv_heads);
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
  if ((q && (!CheckRows(op, "q", c->q, c->rows, c->num_heads, d, 1) || !CheckRows(op, "q_out", c->q_out, c->rows, c->num_heads, d, 1))) ||
      (k && !CheckRows(op, "k", c->k, c->rows, c->kv_heads, d, 1)) ||
      (k && c->k_out.data && !CheckRows(op, "k_out", c->k_out, c->rows, c->kv_heads, d, 1)) ||
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
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  RopeArgs a = {};
  // 16-byte pieces of 8 values: every address and stride in use a multiple of 16 bytes, whole pieces on both sides of
  // the rotated part's end and of the pairs' halves
  bool vec = d % 8 == 0 && (rope->layout == SHAHD_ROPE_HALF ? rope->rotary % 16 == 0 : rope->rotary % 8 == 0);
  const auto operand = [&](const ShahdRows& in, const ShahdRows& out, int heads) {
    for (const ShahdRows* r : {&in, &out})
      if (r->data)
        vec = vec && reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->row_stride * size % 16 == 0 && r->head_stride * size % 16 == 0;
    return RopeOperand{in.data, out.data, in.row_stride, in.head_stride, out.row_stride, out.head_stride, heads};
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
  a.pieces = vec ? (a.interleaved ? d / 8 : (d - a.half) / 8) : d - a.half;
  a.shift = -1;
  for (int s = 0; s < 9; s++)
    if (a.pieces == 1 << s) a.shift = s;
  // as many rows as the block's table holds, fewer where that leaves multiprocessors without a block
  a.rows_per_block = std::max(1, std::min({kRopeMaxRows, kRopeTable / a.half, c->rows / (4 * info.sms)}));
  const int blocks = CeilDiv(c->rows, a.rows_per_block);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  TakeLaunchError(nullptr);
  if (c->dtype == SHAHD_F32) LaunchRope<float, bf16>(a, vec, blocks, st);
  else if (c->dtype == SHAHD_F16) LaunchRope<__half, __half>(a, vec, blocks, st);
  else LaunchRope<bf16, bf16>(a, vec, blocks, st);
  return LaunchStatus(op);
}

}  // extern "C"
