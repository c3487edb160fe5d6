// Norms of the query and key heads with the rotary positions and the append to a paged cache, in one pass: what rope.cuh does to
// given heads, here to heads that are normalised first (NormRow, Brain/Sampling/CachedRowMath.ts:25-56, on each head's values).
//   y = (x - mu) / sqrt(var + eps) * w + b   over the d values of a head; mu = 0 and b = 0 for the root mean square,
//   then pair (a, b) of y -> m (a cos - b sin, a sin + b cos).
// Sums in 32 bits, the variance from the differences to the mean (a head's values are in registers, so a second pass over them
// reads nothing); one rounding, at the end.
//
// Bound by memory: each value is read once and written once. Lanes take pieces of heads as in rope.cuh; the lanes that hold one
// head's pieces lie side by side and add up their shares by shuffles, for all the heads in flight at once. Two blocks of threads on a
// multiprocessor, 128 registers a thread: the next heads' values come in while these are summed, which the third block's registers would
// be taken from.
//
// Measured, in one graph: 59402 rows of 32+8 f16 heads of 128 into the cache, 1.46 GB: 247 us, 5.9 TB/s; without the next heads' loads ahead
// 293, with three blocks, whose values spill, 394. 13872 rows of 16+4 f32 heads of 64, layer norm, 159 MB: 35 us, 4.5 TB/s: sums, shuffles and the
// sines of a row's positions take four of ten issue slots, and the rows are few for each warp. One token of 64 users: 6.4 us, latency.
#pragma once

#include "rope_call.cuh"

namespace shahd {

constexpr int kNormWarps = 8;  // of a block, at most
// Value by value; whole pieces of either layout; pieces whose values find their partners in shared memory.
enum NormMode { kNormValues = 0, kNormInterleaved = 1, kNormHalf = 2, kNormStaged = 3 };

struct NormRopeArgs {
  RopeArgs r;
  const void *weight[2], *bias[2];  // of queries and keys; null: 1 and 0
  int weight_type;
  float eps;
};

__device__ __forceinline__ float WeightAt(const void* w, int type, int i) {
  if (type == SHAHD_F32) return static_cast<const float*>(w)[i];
  if (type == SHAHD_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const bf16*>(w)[i]);
}

// T: the operands' type, C: the cache's.
template <class T, class C, int MODE, bool LAYER>
__global__ void __launch_bounds__(kNormWarps * 32, 2) NormRopeKernel(const __grid_constant__ NormRopeArgs A) {
  constexpr int kDeep = (sizeof(T) == 4 ? 2 : 4) / (MODE == kNormHalf ? 2 : 1);  // heads of a lane in flight
  constexpr bool kExchange = MODE == kNormValues || MODE == kNormStaged;
  __shared__ __align__(16) float2 tables[kNormWarps][128];
  __shared__ __align__(16) float weights[2][256], biases[2][256];
  // normalised values, for those that need a partner of another lane; value 8 l + i of a piece row at [i][l]: no bank twice
  __shared__ float stages[kExchange ? kNormWarps : 1][MODE == kNormStaged ? kDeep : 1][kExchange ? 256 : 1];
  const RopeArgs& a = A.r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d = a.d, half = a.half;
  GridDepWait();
  GridDepLaunch();
  for (int i = threadIdx.x; i < 2 * d; i += blockDim.x) {
    const int k = i >= d, j = i - k * d;
    weights[k][j] = A.weight[k] ? WeightAt(A.weight[k], A.weight_type, j) : 1.f;
    biases[k][j] = LAYER && A.bias[k] ? WeightAt(A.bias[k], A.weight_type, j) : 0.f;
  }
  __syncthreads();
  float2* turn = tables[warp];
  const float per = 1.f / (float)d;
  const int pieces = a.pieces, lanes = 32 / pieces;  // pieces: a power of two; a head's lanes lie side by side
  const int piece = lane % pieces, n0 = lane / pieces;
  int j0 = piece * 8, apart = half;
  bool rotary = MODE == kNormInterleaved ? j0 < 2 * half : j0 < half;
  if (MODE == kNormHalf && !rotary) {  // behind the rotated part: this piece, and the one half of that part further on
    j0 += half;
    apart = d / 2 - half;
  }
  // The next heads' values are on their way while these are worked on, from one operand to the next and from a row to the next.
  Raw8<T> na[kDeep], nb[kDeep];
  const auto load = [&](const RopeOperand& o, long long r, int h) {
    const T* in = static_cast<const T*>(o.in) + r * o.in_row + j0;
#pragma unroll
    for (int k = 0; k < kDeep; k++) {
      const int hk = h + n0 + k * lanes;
      if (hk < o.heads) {
        na[k].Load(in + hk * o.in_head);
        if (MODE == kNormHalf) nb[k].Load(in + hk * o.in_head + apart);
      }
    }
  };
  const RopeOperand& begin = a.q.heads > 0 ? a.q : a.k;  // the first operand
  long long loaded = -1;                                 // the row whose first heads have been asked for
  const int first = a.offsets ? a.offsets[0] : 0, end = a.offsets ? a.offsets[a.n] : a.rows;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  long long row = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  int next = row < a.rows ? a.positions[row] : -1;
  for (; row < a.rows; row += step) {
    const int p = next;
    next = row + step < a.rows ? a.positions[row + step] : -1;  // ahead of this row's values
    if (p < 0 || row < first || row >= end) continue;
    if (MODE != kNormValues && loaded != row) load(begin, row, 0);
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
      constexpr int kPer = MODE == kNormHalf ? 8 : 4;
      const int place = kExchange ? i : (i % kPer / 2 * (half / kPer) + i / kPer) * 2 + i % 2;
      turn[place] = make_float2(cs * a.magnitude, sn * a.magnitude);
    }
    __syncwarp();
    if constexpr (MODE == kNormValues) {
      // a head at a time, value lane + 32 i in lane `lane`
      float* own = stages[warp][0];
      const auto heads = [&](const RopeOperand& o, int kv) {
#pragma unroll 1
        for (int h = 0; h < o.heads; h++) {
          const T* in = static_cast<const T*>(o.in) + row * o.in_row + h * o.in_head;
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = lane + 32 * i < d ? ToFloat(in[lane + 32 * i]) : 0.f;
          if (kv != 1) {
            float sum = 0.f;
            if (LAYER) {
#pragma unroll
              for (int i = 0; i < 8; i++) sum += x[i];
              const float mu = WarpSum(sum) * per;
              sum = 0.f;
#pragma unroll
              for (int i = 0; i < 8; i++) x[i] = lane + 32 * i < d ? x[i] - mu : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) sum = fmaf(x[i], x[i], sum);
            const float scale = __frsqrt_rn(fmaf(WarpSum(sum), per, A.eps));
            const float *w = weights[kv < 0 ? 0 : 1], *b = biases[kv < 0 ? 0 : 1];
            __syncwarp();  // the last head has been read
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int v = lane + 32 * i;
              if (v >= d) break;
              x[i] = fmaf(x[i] * scale, w[v], b[v]);
              own[v] = x[i];
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int v = lane + 32 * i;
              if (v >= 2 * half) break;
              const bool one = a.interleaved ? !(v & 1) : v < half;  // the first of its pair
              const float2 cs = turn[a.interleaved ? v >> 1 : one ? v : v - half];
              const float y = own[a.interleaved ? v ^ 1 : one ? v + half : v - half];
              x[i] = one ? x[i] * cs.x - y * cs.y : x[i] * cs.x + y * cs.y;
            }
          }
          T* out = o.out ? static_cast<T*>(o.out) + row * o.out_row + h * o.out_head : nullptr;
          C* cache = kv >= 0 && at >= 0 ? reinterpret_cast<C*>(a.pool) + at + (long long)(2 * h + kv) * kOpsPage * d : nullptr;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int v = lane + 32 * i;
            if (v >= d) break;
            if (out) out[v] = FromFloat<T>(x[i]);
            if (cache) cache[v] = FromFloat<C>(x[i]);
          }
        }
      };
      heads(a.q, -1);
      heads(a.k, 0);
      heads(a.v, 1);
    } else {
      // pairs of a lane's own pieces
      float4 cs[MODE == kNormHalf ? 4 : 2];
      // staged: cos, sin with its sign, and the place of the partner (-1: not turned)
      float cv[8], sv[8];
      int partner[8];
      if constexpr (MODE == kNormStaged) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int v = j0 + i;
          const bool one = a.interleaved ? !(v & 1) : v < half;
          const int far = v >= 2 * half ? 0 : a.interleaved ? (one ? 1 : -1) : one ? half : -half;
          const float2 c2 = turn[far == 0 ? 0 : a.interleaved ? v >> 1 : one ? v : v - half];
          cv[i] = c2.x;
          sv[i] = one ? -c2.y : c2.y;
          const int y = lane * 8 + i + far;
          partner[i] = far == 0 ? -1 : (y & 7) * 32 + (y >> 3);
        }
      } else if (rotary) {
        constexpr int kPer = MODE == kNormHalf ? 8 : 4;
        const float4* from = reinterpret_cast<const float4*>(turn) + piece;
#pragma unroll
        for (int q = 0; q < kPer / 2; q++) cs[q] = from[q * (half / kPer)];
      }
      // one operand's heads; kv: 0 for keys, 1 for values, -1 for queries
      const auto heads = [&](const RopeOperand& o, int kv, const RopeOperand& then, long long then_row) {
        T* out = o.out ? static_cast<T*>(o.out) + row * o.out_row + j0 : nullptr;
        C* cache = kv >= 0 && at >= 0 ? reinterpret_cast<C*>(a.pool) + at + (long long)kv * kOpsPage * d + j0 : nullptr;
        const float *w = weights[kv < 0 ? 0 : 1] + j0, *b = biases[kv < 0 ? 0 : 1] + j0;
        // the whole warp goes through the same heads: its lanes meet in the sums
#pragma unroll 1
        for (int h = 0; h < o.heads; h += kDeep * lanes) {
          Raw8<T> ra[kDeep], rb[kDeep];
#pragma unroll
          for (int k = 0; k < kDeep; k++) {
            ra[k] = na[k];
            if (MODE == kNormHalf) rb[k] = nb[k];
          }
          if (h + kDeep * lanes < o.heads) load(o, row, h + kDeep * lanes);
          else load(then, then_row, 0);
          float mu[kDeep], scale[kDeep];
          if (kv != 1) {
            const auto all = [&](float (&s)[kDeep]) {  // sums over the lanes of a head
#pragma unroll 1
              for (int far = pieces >> 1; far > 0; far >>= 1)
#pragma unroll
                for (int k = 0; k < kDeep; k++) s[k] += __shfl_xor_sync(0xffffffffu, s[k], far);
            };
#pragma unroll
            for (int k = 0; k < kDeep; k++) mu[k] = 0.f;
            if (LAYER) {
#pragma unroll
              for (int k = 0; k < kDeep; k++) {
                if (h + n0 + k * lanes >= o.heads) continue;
                float x[8];
                ra[k].Get(x);
#pragma unroll
                for (int i = 0; i < 8; i++) mu[k] += x[i];
                if (MODE == kNormHalf) {
                  rb[k].Get(x);
#pragma unroll
                  for (int i = 0; i < 8; i++) mu[k] += x[i];
                }
              }
              all(mu);
#pragma unroll
              for (int k = 0; k < kDeep; k++) mu[k] *= per;
            }
#pragma unroll
            for (int k = 0; k < kDeep; k++) {
              scale[k] = 0.f;
              if (h + n0 + k * lanes >= o.heads) continue;
              float x[8];
              ra[k].Get(x);
#pragma unroll
              for (int i = 0; i < 8; i++) scale[k] = LAYER ? fmaf(x[i] - mu[k], x[i] - mu[k], scale[k]) : fmaf(x[i], x[i], scale[k]);
              if (MODE == kNormHalf) {
                rb[k].Get(x);
#pragma unroll
                for (int i = 0; i < 8; i++) scale[k] = LAYER ? fmaf(x[i] - mu[k], x[i] - mu[k], scale[k]) : fmaf(x[i], x[i], scale[k]);
              }
            }
            all(scale);
#pragma unroll
            for (int k = 0; k < kDeep; k++) scale[k] = __frsqrt_rn(fmaf(scale[k], per, A.eps));
          }
          const auto normal = [&](float (&x)[8], int k, int from) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 wv = *reinterpret_cast<const float4*>(w + from + i);
              const float4 bv = LAYER ? *reinterpret_cast<const float4*>(b + from + i) : make_float4(0, 0, 0, 0);
              x[i] = LAYER ? fmaf((x[i] - mu[k]) * scale[k], wv.x, bv.x) : x[i] * scale[k] * wv.x;
              x[i + 1] = LAYER ? fmaf((x[i + 1] - mu[k]) * scale[k], wv.y, bv.y) : x[i + 1] * scale[k] * wv.y;
              x[i + 2] = LAYER ? fmaf((x[i + 2] - mu[k]) * scale[k], wv.z, bv.z) : x[i + 2] * scale[k] * wv.z;
              x[i + 3] = LAYER ? fmaf((x[i + 3] - mu[k]) * scale[k], wv.w, bv.w) : x[i + 3] * scale[k] * wv.w;
            }
          };
          if constexpr (MODE == kNormStaged) {
            if (kv != 1) {
              __syncwarp();  // the last heads have been read
#pragma unroll
              for (int k = 0; k < kDeep; k++) {
                if (h + n0 + k * lanes >= o.heads) continue;
                float x[8];
                ra[k].Get(x);
                normal(x, k, 0);
#pragma unroll
                for (int i = 0; i < 8; i++) stages[warp][k][i * 32 + lane] = x[i];
              }
              __syncwarp();
            }
          }
#pragma unroll
          for (int k = 0; k < kDeep; k++) {
            const int hk = h + n0 + k * lanes;
            if (hk >= o.heads) continue;
            float x[8], y[8];
            if (MODE == kNormStaged && kv != 1) {
              const float* own = stages[warp][k];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                x[i] = own[i * 32 + lane];
                if (partner[i] >= 0) x[i] = x[i] * cv[i] + own[partner[i]] * sv[i];
              }
            } else {
              ra[k].Get(x);
              if (MODE == kNormHalf) rb[k].Get(y);
              if (kv != 1) {
                normal(x, k, 0);
                if (MODE == kNormHalf) normal(y, k, apart);
                if (rotary) {
#pragma unroll
                  for (int q = 0; q < (MODE == kNormHalf ? 4 : 2); q++) {
                    if (MODE == kNormInterleaved) {
                      const float u = x[4 * q], v = x[4 * q + 1], s = x[4 * q + 2], t = x[4 * q + 3];
                      x[4 * q] = u * cs[q].x - v * cs[q].y;
                      x[4 * q + 1] = u * cs[q].y + v * cs[q].x;
                      x[4 * q + 2] = s * cs[q].z - t * cs[q].w;
                      x[4 * q + 3] = s * cs[q].w + t * cs[q].z;
                    } else {
                      const float u = x[2 * q], v = y[2 * q], s = x[2 * q + 1], t = y[2 * q + 1];
                      x[2 * q] = u * cs[q].x - v * cs[q].y;
                      y[2 * q] = u * cs[q].y + v * cs[q].x;
                      x[2 * q + 1] = s * cs[q].z - t * cs[q].w;
                      y[2 * q + 1] = s * cs[q].w + t * cs[q].z;
                    }
                  }
                }
              }
            }
            if (out) {
              Store8(out + hk * o.out_head, x);
              if (MODE == kNormHalf) Store8(out + hk * o.out_head + apart, y);
            }
            if (cache) {
              C* to = cache + (long long)hk * 2 * kOpsPage * d;
              Store8(to, x);
              if (MODE == kNormHalf) Store8(to + apart, y);
            }
          }
        }
      };
      // (an operand that there is not has no heads: nothing is done and nothing loaded)
      const long long next_row = next >= 0 && row + step < end ? row + step : row;  // no other rows are read
      if (a.q.heads > 0) heads(a.q, -1, a.k.heads > 0 ? a.k : a.q, a.k.heads > 0 ? row : next_row);
      if (a.k.heads > 0) heads(a.k, 0, a.v.heads > 0 ? a.v : begin, a.v.heads > 0 ? row : next_row);
      if (a.v.heads > 0) heads(a.v, 1, begin, next_row);
      loaded = next_row;
    }
  }
}

template <class T, class C, int MODE, bool LAYER>
void LaunchNormRopeKind(const NormRopeArgs& a, int sms, cudaStream_t st) {
  // a warp per row while they last, spread over the multiprocessors; then as many blocks as run at once
  const int warps = std::max(1, std::min(kNormWarps, a.r.rows / sms));
  const int blocks = std::min(CeilDiv(a.r.rows, warps), 2 * sms);
  LaunchPdl(NormRopeKernel<T, C, MODE, LAYER>, dim3(blocks), dim3(warps * 32), 0, st, a);
}

template <class T, class C, int MODE>
void LaunchNormRopeMode(const NormRopeArgs& a, bool layer, int sms, cudaStream_t st) {
  if (layer) LaunchNormRopeKind<T, C, MODE, true>(a, sms, st);
  else LaunchNormRopeKind<T, C, MODE, false>(a, sms, st);
}

template <class T, class C>
void LaunchNormRope(const NormRopeArgs& a, int mode, bool layer, int sms, cudaStream_t st) {
  if (mode == kNormValues) LaunchNormRopeMode<T, C, kNormValues>(a, layer, sms, st);
  else if (mode == kNormInterleaved) LaunchNormRopeMode<T, C, kNormInterleaved>(a, layer, sms, st);
  else if (mode == kNormHalf) LaunchNormRopeMode<T, C, kNormHalf>(a, layer, sms, st);
  else LaunchNormRopeMode<T, C, kNormStaged>(a, layer, sms, st);
}

}  // namespace shahd

extern "C" {

int shahd_norm_rope_apply(const ShahdRope* rope, const ShahdRopeCall* c, const ShahdHeadNorm* norm, void* stream) {
  using namespace shahd;
  const char* op = "shahd_norm_rope_apply";
  ClearError();
  if (!rope || !c || !norm) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  if (norm->kind != SHAHD_NORM_RMS && norm->kind != SHAHD_NORM_LAYER) {
    SetError("%s: unknown norm %d", op, norm->kind);
    return SHAHD_EINVAL;
  }
  const bool layer = norm->kind == SHAHD_NORM_LAYER;
  const float eps = (float)norm->eps;
  if (!(eps > 0) || !std::isfinite(eps)) {
    SetError("%s: eps must be positive and finite in 32 bits (got %g)", op, norm->eps);
    return SHAHD_EINVAL;
  }
  if (norm->weight_dtype != SHAHD_F32 && norm->weight_dtype != SHAHD_BF16 && norm->weight_dtype != SHAHD_F16) {
    SetError("%s: weight_dtype must be SHAHD_BF16, SHAHD_F16 or SHAHD_F32, got %d", op, norm->weight_dtype);
    return SHAHD_EINVAL;
  }
  if (!layer && (norm->q_bias || norm->k_bias)) {
    SetError("%s: biases go with SHAHD_NORM_LAYER", op);
    return SHAHD_EINVAL;
  }
  NormRopeArgs a = {};
  MoreBuffer more[4];
  int count = 0;
  const size_t size = TypeBytes(norm->weight_dtype);
  const auto add = [&](const char* name, const void* p, bool used) -> const void* {
    if (!p || !used) return nullptr;
    more[count++] = {name, p, size};
    return p;
  };
  a.weight[0] = add("q_weight", norm->q_weight, c->num_heads > 0);
  a.weight[1] = add("k_weight", norm->k_weight, c->kv_heads > 0);
  a.bias[0] = add("q_bias", norm->q_bias, c->num_heads > 0);
  a.bias[1] = add("k_bias", norm->k_bias, c->kv_heads > 0);
  a.weight_type = norm->weight_dtype;
  a.eps = eps;
  RopePieces p;
  DeviceInfo info;
  int device = -1;
  const int rc = PrepareRope(op, rope, c, more, count, &a.r, &p, &info, &device);
  if (rc != SHAHD_OK || c->rows == 0) return rc;
  DeviceScope scope(device);
  if (!scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, device);
    return SHAHD_ENODEV;
  }
  // The lanes of a head add up by halves, so a head is a power of two of pieces; others go value by value.
  const int d = a.r.d;
  const bool even = d >= 8 && (d & (d - 1)) == 0;
  const int mode = !p.vec || !even ? kNormValues : !p.whole ? kNormStaged : a.r.interleaved ? kNormInterleaved : kNormHalf;
  a.r.pieces = mode == kNormValues ? 1 : mode == kNormHalf ? d / 16 : d / 8;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  TakeLaunchError(nullptr);
  if (c->dtype == SHAHD_F32) LaunchNormRope<float, bf16>(a, mode, layer, info.sms, st);
  else if (c->dtype == SHAHD_F16) LaunchNormRope<__half, __half>(a, mode, layer, info.sms, st);
  else LaunchNormRope<bf16, bf16>(a, mode, layer, info.sms, st);
  return LaunchStatus(op);
}

}  // extern "C"
