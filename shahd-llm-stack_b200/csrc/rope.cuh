// Rotary positions on packed rows (ApplyRope, Brain/Ops/RotaryEmbedding.ts:63-75, for prompts of different lengths
// and for the layouts and scalings that the session's fused RoPE does not have), with the append of the rotated keys
// and the values to a paged cache.
//
// The first r of a head's d values are r/2 pairs; pair i of a row at position p is turned by p * f_i:
//   (a, b) -> m (a cos - b sin, a sin + b cos),   f_i = base^(-2i/r), scaled as the plan says, m the plan's magnitude,
// with pairs (2i, 2i+1) or (i, i + r/2). Angles: the turn p * f_i / 2pi is formed in 64 bits and only its fraction is
// rounded to 32, so a position of 10^6 loses nothing (in 32 bits the angle alone would be off by 0.03).
//
// Bound by memory: each value is read once and written once. A warp takes a row at a time and waits for no other: its lanes
// form the row's (cos, sin), one sincospi per pair for all heads, in shared memory of the warp's own, and take their
// piece's into registers; a lane's piece of a head (8 values; in the half layout two pieces, as far apart as pairs are) is the same
// in all heads, so a lane goes over heads with up to eight 16-byte loads in flight. Where pairs do not
// fill whole pieces, a lane's eight values find their partners in shared memory, where the warp puts the heads it has loaded.
// Operands whose address or strides do not allow pieces go value by value. (Blocks of 256 threads over batches of rows, with a table per batch, lost a
// fifth of the time at the barriers: 59402 rows of 32 + 8 heads of 128 in f16, 1.22 GB, took 265 us where a warp per row took
// 209, now 206; 57344 rows, 1.17 GB, take 199 us, a plain copy of as much 180.)
#pragma once

#include "rope_call.cuh"

namespace shahd {

constexpr int kRopeWarps = 8;   // of a block, at most
// One pair per thread; pieces of either layout; pieces whose values find their partners in shared memory.
enum RopeMode { kRopeValues = 0, kRopeInterleaved = 1, kRopeHalf = 2, kRopeStaged = 3 };
// Blocks of a multiprocessor: in the half layout a lane holds two pieces and their eight (cos, sin), 16-bit ones twice, which spills
// at 80 registers (274 us instead of 199 for 57344 rows of 32 + 8 heads of 128), and so do staged pieces (268 us instead of 227,
// 126 of the 128 values turned). Interleaved 16-bit pieces spill a little (116 bytes) with three: 211 us, 205 with two.
template <class T, int MODE>
constexpr int kRopePerSm = (MODE == kRopeHalf && sizeof(T) == 2) || MODE == kRopeStaged ? 2 : 3;

// T: the operands' type, C: the cache's.
template <class T, class C, int MODE>
__global__ void __launch_bounds__(kRopeWarps * 32, kRopePerSm<T, MODE>) RopeKernel(const __grid_constant__ RopeArgs a) {
  __shared__ __align__(16) float2 tables[kRopeWarps][128];
  constexpr int kStage = sizeof(T) == 4 ? 2 : 4;  // staged: heads of a lane in flight
  __shared__ __align__(16) T stages[MODE == kRopeStaged ? kRopeWarps : 1][MODE == kRopeStaged ? kStage : 1][32 * 8];
  constexpr int kPer = MODE == kRopeHalf ? 8 : 4;  // pairs of a piece
  GridDepWait();
  GridDepLaunch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d = a.d, half = a.half, heads = a.q.heads + a.k.heads + a.v.heads;
  float2* turn = tables[warp];
  // pieces: this lane's place in a head, and its first head (of every `lanes`-th)
  const int piece = MODE == kRopeValues ? 0 : lane % a.pieces, lanes = MODE == kRopeValues ? 1 : 32 / a.pieces;
  const int n0 = MODE == kRopeValues ? 0 : lane / a.pieces;
  int j0 = piece * 8, apart = half;
  bool rotary = MODE == kRopeInterleaved ? j0 < 2 * half : j0 < half;
  if (MODE == kRopeHalf && !rotary) {  // behind the rotated part: this piece, and the one half of that part further on
    j0 += half;
    apart = d / 2 - half;
  }
  const int first = a.offsets ? a.offsets[0] : 0, end = a.offsets ? a.offsets[a.n] : a.rows;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  long long row = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  int next = row < a.rows ? a.positions[row] : -1;
  for (; row < a.rows; row += step) {
    const int p = next;
    next = row + step < a.rows ? a.positions[row + step] : -1;  // ahead of this row's values
    if (p < 0 || row < first || row >= end) continue;
    long long at = -1;  // the row's place in the cache (kv head 0, K)
    if (a.pool && (p >> 6) < a.max_blocks) {
      const int page = a.table[(long long)SequenceOf(a.offsets, a.n, (int)row) * a.max_blocks + (p >> 6)];
      if (page >= 0 && page < a.pages) at = page * a.page_stride + (long long)(p & 63) * d;
    }
    __syncwarp();  // the last row's table has been read
#pragma unroll 1
    for (int i = lane; i < half; i += 32) {
      // from the parameters by a generic load: as an indexed constant, 32 different frequencies take a warp 32 accesses
      double f;
      asm volatile("ld.f64 %0, [%1];" : "=d"(f) : "l"(a.turns + i));
      const double t = (double)p * f;
      float sn, cs;
      sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
      // two pairs of every piece side by side, so that the lanes' 16-byte reads lie next to each other
      const int place = MODE == kRopeValues || MODE == kRopeStaged ? i : (i % kPer / 2 * (half / kPer) + i / kPer) * 2 + i % 2;
      turn[place] = make_float2(cs * a.magnitude, sn * a.magnitude);
    }
    __syncwarp();
    if constexpr (MODE == kRopeValues) {
      for (int item = lane; item < heads * a.pieces; item += 32) {
        const int n = item / a.pieces, j = item - n * a.pieces;
        const int kv = n < a.q.heads ? -1 : n < a.q.heads + a.k.heads ? 0 : 1;  // 0 for a key, 1 for a value, -1 for a query
        const RopeOperand& o = kv < 0 ? a.q : kv == 0 ? a.k : a.v;
        const int h = kv < 0 ? n : kv == 0 ? n - a.q.heads : n - a.q.heads - a.k.heads;
        const bool two = j < half;  // a pair, or a value behind the rotated part
        const int v0 = !two ? j + half : a.interleaved ? 2 * j : j, v1 = a.interleaved ? v0 + 1 : v0 + half;
        const T* in = static_cast<const T*>(o.in) + row * o.in_row + h * o.in_head;
        float x = ToFloat(in[v0]), y = two ? ToFloat(in[v1]) : 0.f;
        if (two && kv != 1) {
          const float2 cs = turn[j];
          const float u = x * cs.x - y * cs.y;
          y = x * cs.y + y * cs.x;
          x = u;
        }
        if (o.out) {
          T* out = static_cast<T*>(o.out) + row * o.out_row + h * o.out_head;
          out[v0] = FromFloat<T>(x);
          if (two) out[v1] = FromFloat<T>(y);
        }
        if (kv >= 0 && at >= 0) {
          C* cache = reinterpret_cast<C*>(a.pool) + at + (long long)(2 * h + kv) * kOpsPage * d;
          cache[v0] = FromFloat<C>(x);
          if (two) cache[v1] = FromFloat<C>(y);
        }
      }
    } else if constexpr (MODE == kRopeStaged) {
      // of this lane's eight values: cos, sin with its sign, and how far away the partner lies (0: not turned)
      float cv[8], sv[8];
      int apart_v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int v = j0 + i, first_of = a.interleaved ? !(v & 1) : v < half;
        apart_v[i] = v >= 2 * half ? 0 : a.interleaved ? (first_of ? 1 : -1) : first_of ? half : -half;
        const float2 cs = turn[apart_v[i] == 0 ? 0 : a.interleaved ? v >> 1 : first_of ? v : v - half];
        cv[i] = cs.x;
        sv[i] = first_of ? -cs.y : cs.y;
      }
      const auto turn_heads = [&](const RopeOperand& o, int kv) {
        const T* in = static_cast<const T*>(o.in) + row * o.in_row + j0;
        T* out = o.out ? static_cast<T*>(o.out) + row * o.out_row + j0 : nullptr;
        C* cache = kv >= 0 && at >= 0 ? reinterpret_cast<C*>(a.pool) + at + (long long)kv * kOpsPage * d + j0 : nullptr;
#pragma unroll 1
        for (int h = 0; h < o.heads; h += kStage * lanes) {
          Raw8<T> raw[kStage];
#pragma unroll
          for (int k = 0; k < kStage; k++) {
            const int hk = h + n0 + k * lanes;
            if (n0 < lanes && hk < o.heads) raw[k].Load(in + hk * o.in_head);
          }
          if (kv != 1) {
            __syncwarp();  // the last heads have been read
#pragma unroll
            for (int k = 0; k < kStage; k++)
#pragma unroll
              for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4*>(&stages[warp][k][lane * 8])[i] = raw[k].u[i];
            __syncwarp();
          }
#pragma unroll
          for (int k = 0; k < kStage; k++) {
            const int hk = h + n0 + k * lanes;
            if (n0 >= lanes || hk >= o.heads) break;
            float x[8];
            raw[k].Get(x);
            if (kv != 1) {
              const T* own = &stages[warp][k][lane * 8];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float y = ToFloat(own[i + apart_v[i]]);
                if (apart_v[i] != 0) x[i] = x[i] * cv[i] + y * sv[i];
              }
            }
            if (out) Store8(out + hk * o.out_head, x);
            if (cache) Store8(cache + (long long)hk * 2 * kOpsPage * d, x);
          }
        }
      };
      turn_heads(a.q, -1);
      turn_heads(a.k, 0);
      turn_heads(a.v, 1);
    } else if (n0 < lanes) {
      float4 cs[kPer / 2];
      if (rotary) {
        const float4* from = reinterpret_cast<const float4*>(turn) + piece;
#pragma unroll
        for (int q = 0; q < kPer / 2; q++) cs[q] = from[q * (half / kPer)];
      }
      // one operand's heads; kv: 0 for keys, 1 for values, -1 for queries
      const auto turn_heads = [&](const RopeOperand& o, int kv, int h0) {
        constexpr int kDeep = (sizeof(T) == 4 ? 2 : 4) / (MODE == kRopeHalf ? 2 : 1);  // heads in flight
        const T* in = static_cast<const T*>(o.in) + row * o.in_row + j0;
        T* out = o.out ? static_cast<T*>(o.out) + row * o.out_row + j0 : nullptr;
        C* cache = kv >= 0 && at >= 0 ? reinterpret_cast<C*>(a.pool) + at + (long long)kv * kOpsPage * d + j0 : nullptr;
#pragma unroll 1
        for (int h = h0; h < o.heads; h += kDeep * lanes) {
          Raw8<T> ra[kDeep], rb[kDeep];
#pragma unroll
          for (int k = 0; k < kDeep; k++) {
            const int hk = h + k * lanes;
            if (hk < o.heads) {
              ra[k].Load(in + hk * o.in_head);
              if (MODE == kRopeHalf) rb[k].Load(in + hk * o.in_head + apart);
            }
          }
#pragma unroll
          for (int k = 0; k < kDeep; k++) {
            const int hk = h + k * lanes;
            if (hk >= o.heads) break;
            float x[8], y[8];
            ra[k].Get(x);
            if (MODE == kRopeHalf) rb[k].Get(y);
            if (rotary && kv != 1) {
#pragma unroll
              for (int q = 0; q < kPer / 2; q++) {
                if (MODE == kRopeInterleaved) {
                  const float u = x[4 * q], v = x[4 * q + 1], s = x[4 * q + 2], w = x[4 * q + 3];
                  x[4 * q] = u * cs[q].x - v * cs[q].y;
                  x[4 * q + 1] = u * cs[q].y + v * cs[q].x;
                  x[4 * q + 2] = s * cs[q].z - w * cs[q].w;
                  x[4 * q + 3] = s * cs[q].w + w * cs[q].z;
                } else {
                  const float u = x[2 * q], v = y[2 * q], s = x[2 * q + 1], w = y[2 * q + 1];
                  x[2 * q] = u * cs[q].x - v * cs[q].y;
                  y[2 * q] = u * cs[q].y + v * cs[q].x;
                  x[2 * q + 1] = s * cs[q].z - w * cs[q].w;
                  y[2 * q + 1] = s * cs[q].w + w * cs[q].z;
                }
              }
            }
            if (out) {
              Store8(out + hk * o.out_head, x);
              if (MODE == kRopeHalf) Store8(out + hk * o.out_head + apart, y);
            }
            if (cache) {
              C* to = cache + (long long)hk * 2 * kOpsPage * d;
              Store8(to, x);
              if (MODE == kRopeHalf) Store8(to + apart, y);
            }
          }
        }
      };
      turn_heads(a.q, -1, n0);
      turn_heads(a.k, 0, n0);
      turn_heads(a.v, 1, n0);
    }
  }
}

template <class T, class C, int MODE>
void LaunchRopeMode(const RopeArgs& a, int sms, cudaStream_t st) {
  // a warp per row while they last, spread over the multiprocessors; then as many blocks as run at once
  const int warps = std::max(1, std::min(kRopeWarps, a.rows / sms));
  const int blocks = std::min(CeilDiv(a.rows, warps), kRopePerSm<T, MODE> * sms);
  LaunchPdl(RopeKernel<T, C, MODE>, dim3(blocks), dim3(warps * 32), 0, st, a);
}

template <class T, class C>
void LaunchRope(const RopeArgs& a, int mode, int sms, cudaStream_t st) {
  if (mode == kRopeValues) LaunchRopeMode<T, C, kRopeValues>(a, sms, st);
  else if (mode == kRopeInterleaved) LaunchRopeMode<T, C, kRopeInterleaved>(a, sms, st);
  else if (mode == kRopeHalf) LaunchRopeMode<T, C, kRopeHalf>(a, sms, st);
  else LaunchRopeMode<T, C, kRopeStaged>(a, sms, st);
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
  const float magnitude = (float)cfg->magnitude;
  if (!(cfg->base > 1) || !std::isfinite(cfg->base) || !std::isfinite(magnitude) || magnitude == 0 ||
      (scaled && (!(cfg->factor >= 1) || !std::isfinite(cfg->factor)))) {
    SetError("%s: need a finite base > 1, a magnitude that is finite and not 0 in 32 bits and, for a scaling, a finite factor >= 1 (got "
             "base=%g magnitude=%g factor=%g)", op, cfg->base, cfg->magnitude, cfg->factor);
    return SHAHD_EINVAL;
  }
  double low = 0, high = 0, base = cfg->base;
  switch (cfg->scaling) {
    case SHAHD_ROPE_UNSCALED:
    case SHAHD_ROPE_LINEAR:
      break;
    case SHAHD_ROPE_STRETCHED:
      if (r < 4) {
        SetError("%s: SHAHD_ROPE_STRETCHED needs rotary_dim >= 4, got %d", op, r);
        return SHAHD_EINVAL;
      }
      base *= std::pow(cfg->factor, r / (r - 2.0));
      if (!std::isfinite(base)) {
        SetError("%s: the stretched base %g * %g^(r/(r-2)) is not finite", op, cfg->base, cfg->factor);
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
  p->magnitude = magnitude;
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
  RopeArgs a;
  RopePieces p;
  DeviceInfo info;
  int device = -1;
  const int rc = PrepareRope(op, rope, c, nullptr, 0, &a, &p, &info, &device);
  if (rc != SHAHD_OK || c->rows == 0) return rc;
  DeviceScope scope(device);
  if (!scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, device);
    return SHAHD_ENODEV;
  }
  const int mode = !p.vec ? kRopeValues : !p.whole ? kRopeStaged : a.interleaved ? kRopeInterleaved : kRopeHalf;
  a.pieces = mode == kRopeValues ? a.d - a.half : mode == kRopeHalf ? a.d / 16 : a.d / 8;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  TakeLaunchError(nullptr);
  if (c->dtype == SHAHD_F32) LaunchRope<float, bf16>(a, mode, info.sms, st);
  else if (c->dtype == SHAHD_F16) LaunchRope<__half, __half>(a, mode, info.sms, st);
  else LaunchRope<bf16, bf16>(a, mode, info.sms, st);
  return LaunchStatus(op);
}

}  // extern "C"
