// Attention of 128-row query tiles on the tensor cores, for two operators:
//   packed prompts  out[i] = sum_{j <= i} softmax_j(scale q[i].k[j]) v[j] within each sequence (MultiHeadAttention.ts:46-74,
//                   CausalSoftmax.ts:17-33, for sequences of different lengths in one call), and
//   trees           the drafted nodes of a sequence against its cached positions and against each other by a bit mask.
//
// A tile's rows are (token, query head of one kv head) pairs, tokens outside: 128/G tokens times G heads, so the G heads
// that share keys sit in one tile, a decode step of few rows fills what it can, and a tile's last key block is cut close to
// the diagonal. A block of threads works on two tiles at a time: on two neighbours that read the same keys, or, when a
// sequence has only one tile of rows (decode steps, small trees), on that tile twice with the key blocks dealt out by turns
// and one merge at the end, so there is always one tile's softmax under the other's products.
//
//   S = Q K^T   tcgen05 M 128, N up to 128 keys, into TMEM (128 columns per tile);
//   softmax     one thread per row: the row's 128 scores in registers, running maximum and sum in 32 bits; the maximum
//               moves only when a row's new one is over 8 (in log2) above it, since a probability of up to 2^8 costs
//               nothing in floating point: then, rarely, the accumulator in TMEM is scaled;
//   O += P V    P rounded to 16 bits (as every attention on these units) overwrites S in TMEM and is the A operand there; V
//               is the MN-major B operand; O stays in TMEM until the end.
// Keys and values come by TMA (128-byte swizzle) through a ring of 128-key units; the cache's pages are boxes of 64 positions.
// A block that is cut short (a sequence's end, the diagonal) loads only the 64-row boxes and multiplies only the 16-key
// steps that hold keys; rows of V behind a sequence's end are zeroed in shared memory, since 0 * inf would not be 0.
//
// Warps 0-3 and 4-7: the softmax of tile 0 and 1; warp 8: MMA issue; warp 9: loads.
#pragma once

#include "ops_common.cuh"
#include "rope.cuh"

namespace shahd {

constexpr int kTaThreads = 320;
constexpr int kTaBox = 8192;   // 64 rows of 64 values
constexpr int kTaHalf = 16384;  // 128 rows of 64 values
constexpr float kTaLazy = 8.f;  // log2 of what a probability may grow to before the accumulator is scaled

template <int D>
struct TaCfg {
  static constexpr int kHalves = D == 128 ? 2 : 1;  // 64-value columns of a row (head_dim 32: half of one, the rest zero)
  static constexpr int kUnit = kTaHalf * kHalves;   // 128 rows: a Q tile, or a block's K or V
  static constexpr int kUnits = D == 128 ? 5 : 10;  // ring depth
  static constexpr int kSmem = 1024 + (2 + kUnits) * kUnit + 512;
};

struct TaShared {
  uint64_t full[10], empty[10], q_full, s_full[2], p_full[2], o_full[2], drained;
  uint32_t tmem;
  volatile int abort;
};
static_assert(sizeof(TaShared) <= 512, "TaShared");

struct TaArgs {
  CUtensorMap qmap, kmap, vmap;  // rows: (value, head, row), boxes 64 x G x 128/G for q, 64 x 1 x 64 for k and v
  CUtensorMap pool;              // cache: (value, row of the page, page), boxes 64 x 64 x 1
  uint16_t* out;
  long long out_row, out_head;
  const int* offsets;
  int n, rows, H, Hk, G, TB;  // TB: tokens of a tile
  float scale_log2;           // scale * log2(e)
  // trees
  const unsigned long long* masks;
  const int* lengths;
  const int* table;
  int max_blocks, pages, max_nodes, pairs, nsplit;
  float* part_o;    // [n, Hk, nsplit, max_nodes * G, D]
  float2* part_ml;  // [n, Hk, nsplit, max_nodes * G]: running maximum (of scaled log2 scores) and sum
};

__device__ __forceinline__ void TmaLoad3D(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          SmemAddr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(SmemAddr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// D[tmem] (+)= A[tmem] B[smem], kind::f16, issued by one thread.
__device__ __forceinline__ void UmmaTmemA(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 / 32 consecutive columns per thread to TMEM.
__device__ __forceinline__ void TmemStore16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void TmemStore32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void TmemWaitSt() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool F16>
__device__ __forceinline__ uint32_t Pack2(float a, float b) {  // a in the low half
  uint32_t r;
  if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// A wait that ends: false once it, or another warp's, has given up.
__device__ __forceinline__ bool TaWait(TaShared* sh, uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kOpsWaitLimit; i++) {
    if (MbarTryWait(bar, parity)) return true;
    if (sh->abort) return false;
  }
  atomicCAS(&g_ops_device_error, 0, kOpsErrTimeout);
  sh->abort = 1;
  return false;
}

// What a block of threads works on.
struct TaWork {
  int seq, start;       // sequence and its first row
  int head;             // kv head
  int q0;               // first token of tile 0 within the sequence
  int tokens[2];        // of the tiles
  int blocks[2];        // key blocks of the tiles
  bool turns;           // one tile of rows, its key blocks dealt out by turns
  int first;            // trees: first key block
  int cached;           // trees: cached positions
  int cache_blocks;     // trees: 128-key blocks of the cache
  int nodes;            // trees: rows of the sequence; prompts: tokens of the sequence
};

// The prompt tile `tile` of all: sequence s owns tiles offsets[s] / (2 TB) + s .. offsets[s+1] / (2 TB) + s, at least as many
// as it needs, so the mapping is a search in the offsets and needs no table. Each warp finds the same.
__device__ __forceinline__ bool PromptWork(const TaArgs& A, int tile, TaWork& w) {
  const int lane = threadIdx.x & 31, span = 2 * A.TB;
  const auto off = [&](int s) { return min(max(A.offsets[s], 0), A.rows); };
  int lo = 0, cnt = A.n;
  while (cnt > 1) {
    const int step = (cnt + 31) / 32;
    const bool le = lane * step < cnt && off(lo + lane * step) / span + lo + lane * step <= tile;
    const unsigned hit = __ballot_sync(0xffffffffu, le);
    if (!hit) return false;
    const int k = 31 - __clz(hit);
    lo += k * step;
    cnt = min(step, cnt - k * step);
  }
  w.seq = lo;
  w.start = off(lo);
  const int len = max(off(lo + 1) - w.start, 0), local = tile - (w.start / span + lo);
  w.nodes = len;
  w.q0 = local * span;
  if (local < 0 || w.q0 >= len) return false;
  for (int i = 0; i < 2; i++) {
    w.tokens[i] = min(max(len - w.q0 - i * A.TB, 0), A.TB);
    w.blocks[i] = w.tokens[i] > 0 ? (w.q0 + i * A.TB + w.tokens[i] + 127) / 128 : 0;
  }
  w.turns = false;
  w.first = w.cached = w.cache_blocks = 0;
  return true;
}

__device__ __forceinline__ bool TreeWork(const TaArgs& A, int x, TaWork& w) {
  const int split = x % A.nsplit;
  x /= A.nsplit;
  const int pair = x % A.pairs;
  x /= A.pairs;
  w.head = x % A.Hk;
  w.seq = x / A.Hk;
  w.start = min(max(A.offsets[w.seq], 0), A.rows);
  const int end = min(max(A.offsets[w.seq + 1], w.start), A.rows);
  w.nodes = min(end - w.start, A.max_nodes);
  w.q0 = pair * 2 * A.TB;
  for (int i = 0; i < 2; i++) w.tokens[i] = min(max(w.nodes - w.q0 - i * A.TB, 0), A.TB);
  if (w.tokens[0] == 0) return false;
  w.cached = (int)min((long long)max(A.lengths[w.seq], 0), (long long)A.max_blocks * kOpsPage);
  w.cache_blocks = (w.cached + 127) / 128;
  const int all = w.cache_blocks + 1;
  w.first = (int)((long long)all * split / A.nsplit);
  const int count = (int)((long long)all * (split + 1) / A.nsplit) - w.first;
  w.turns = w.tokens[1] == 0;
  if (w.turns) {
    w.tokens[1] = w.tokens[0];
    w.blocks[0] = (count + 1) / 2;
    w.blocks[1] = count / 2;
  } else {
    w.blocks[0] = w.blocks[1] = count;
  }
  return true;
}

template <bool TREE>
struct TaBlocks {
  const TaArgs& A;
  const TaWork& w;
  // The key block of step t of tile i.
  __device__ __forceinline__ int Index(int i, int t) const { return TREE ? (w.turns ? w.first + 2 * t + i : w.first + t) : t; }
  // Keys of a block that belong to the sequence (1 .. 128).
  __device__ __forceinline__ int Keys(int b) const {
    if constexpr (TREE) return b < w.cache_blocks ? min(128, w.cached - 128 * b) : w.nodes;
    else return min(128, w.nodes - 128 * b);
  }
  // Keys of a block that some row of tile i may see.
  __device__ __forceinline__ int Seen(int i, int b) const {
    if constexpr (TREE) return Keys(b);
    else return min(128, w.q0 + i * A.TB + w.tokens[i] - 128 * b);
  }
};

template <int D, bool F16, bool TREE>
__global__ void __launch_bounds__(kTaThreads, 1) TileAttentionKernel(const __grid_constant__ TaArgs A) {
  using Cfg = TaCfg<D>;
  constexpr int U = Cfg::kUnits;
  extern __shared__ uint8_t ta_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ta_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = base;
  uint8_t* ring = base + 2 * Cfg::kUnit;
  TaShared* sh = reinterpret_cast<TaShared*>(ring + U * Cfg::kUnit);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  GridDepWait();
  TaWork w;
  if constexpr (TREE) {
    if (!TreeWork(A, blockIdx.x, w)) return;
  } else {
    // the last tiles of a sequence are the longest: they start first
    const int x = gridDim.x - 1 - blockIdx.x;
    w.head = x % A.Hk;
    if (!PromptWork(A, x / A.Hk, w)) return;
  }
  const TaBlocks<TREE> blk{A, w};

  if (threadIdx.x == 0) {
    for (int s = 0; s < U; s++) {
      MbarInit(&sh->full[s], 1);
      MbarInit(&sh->empty[s], 1);
    }
    MbarInit(&sh->q_full, 1);
    for (int i = 0; i < 2; i++) {
      MbarInit(&sh->s_full[i], 1);
      MbarInit(&sh->p_full[i], 128);
      MbarInit(&sh->o_full[i], 1);
    }
    MbarInit(&sh->drained, 1);
    sh->abort = 0;
    FenceMbarInit();
  }
  if (warp == 8) {
    TmemAlloc(&sh->tmem, 512);
    TmemRelinquish();
  }
  TcgenFenceBefore();
  __syncthreads();
  TcgenFenceAfter();
  const uint32_t tmem = sh->tmem;
  GridDepLaunch();  // after this block holds its TMEM
  const int steps = max(w.blocks[0], w.blocks[1]);

  if (warp == 9) {
    if (lane == 0) {
      FenceProxyAsyncGlobal();
      const int tiles = !w.turns && w.tokens[1] > 0 ? 2 : 1;
      MbarArriveExpectTx(&sh->q_full, tiles * Cfg::kHalves * A.G * A.TB * 128);
      for (int i = 0; i < tiles; i++)
        for (int h = 0; h < Cfg::kHalves; h++)
          TmaLoad3D(sQ + i * Cfg::kUnit + h * kTaHalf, &A.qmap, &sh->q_full, 64 * h, w.head * A.G, w.start + w.q0 + i * A.TB);
      int u = 0;
      // one block's K or V into the next unit of the ring
      const auto load = [&](int b, int keys, bool value) -> bool {
        const int st = u % U;
        if (u >= U && !TaWait(sh, &sh->empty[st], (uint32_t)((u / U - 1) & 1))) return false;
        uint8_t* dst = ring + st * Cfg::kUnit;
        const int boxes = keys > 64 ? 2 : 1;
        MbarArriveExpectTx(&sh->full[st], boxes * Cfg::kHalves * kTaBox);
        for (int x = 0; x < boxes; x++) {
          if (TREE && b < w.cache_blocks) {
            const int p = 2 * b + x;
            int page = p < A.max_blocks ? A.table[(long long)w.seq * A.max_blocks + p] : -1;
            if (page < 0 || page >= A.pages) page = A.pages;  // behind the pool: TMA fills zeros, and the keys are masked
            for (int h = 0; h < Cfg::kHalves; h++)
              TmaLoad3D(dst + h * kTaHalf + x * kTaBox, &A.pool, &sh->full[st], 64 * h, (w.head * 2 + (value ? 1 : 0)) * kOpsPage, page);
          } else {
            const int row = w.start + (TREE ? 0 : 128 * b) + 64 * x;
            for (int h = 0; h < Cfg::kHalves; h++)
              TmaLoad3D(dst + h * kTaHalf + x * kTaBox, value ? &A.vmap : &A.kmap, &sh->full[st], 64 * h, w.head, row);
          }
        }
        u++;
        return true;
      };
      // the order in which the MMA warp comes to need them
      bool ok = true;
      if (w.turns) {
        for (int i = 0; i < 2 && ok; i++)
          if (w.blocks[i] > 0) ok = load(blk.Index(i, 0), blk.Keys(blk.Index(i, 0)), false);
        for (int t = 0; t < steps && ok; t++)
          for (int i = 0; i < 2 && ok; i++) {
            if (t < w.blocks[i]) ok = load(blk.Index(i, t), blk.Keys(blk.Index(i, t)), true);
            if (ok && t + 1 < w.blocks[i]) ok = load(blk.Index(i, t + 1), blk.Keys(blk.Index(i, t + 1)), false);
          }
      } else {
        const int last = w.tokens[1] > 0 ? 1 : 0;  // of the two tiles it sees most
        const auto keys = [&](int t) { return blk.Seen(last, blk.Index(last, t)); };
        if (steps > 0) ok = load(blk.Index(0, 0), keys(0), false);
        for (int t = 0; t < steps && ok; t++) {
          ok = load(blk.Index(0, t), keys(t), true);
          if (ok && t + 1 < steps) ok = load(blk.Index(0, t + 1), keys(t + 1), false);
        }
      }
      // every copy lands before the block may leave
      MbarWaitBounded(&sh->q_full, 0, kOpsWaitLimit);
      for (int v = max(0, u - U); v < u; v++) MbarWaitBounded(&sh->full[v % U], (uint32_t)((v / U) & 1), kOpsWaitLimit);
    }
  } else if (warp == 8) {
    // The whole warp follows the same path, lane 0 issues.
    constexpr uint32_t kTypes = F16 ? 0u : (1u << 7) | (1u << 10);
    const uint32_t idesc0 = (1u << 4) | kTypes | ((128u >> 4) << 24);
    const uint32_t idesc_pv = idesc0 | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // V is MN-major
    int u = 0;
    bool ok = true;
    const auto acquire = [&]() -> int {
      const int st = u % U;
      ok = ok && TaWait(sh, &sh->full[st], (uint32_t)((u / U) & 1));
      u++;
      return st;
    };
    const auto scores = [&](int i, int t, int st) {
      const int kc = (blk.Seen(i, blk.Index(i, t)) + 15) & ~15;
      if (lane == 0) {
        TcgenFenceAfter();
        const uint32_t idesc = idesc0 | ((uint32_t)(kc >> 3) << 17);
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {
          const uint64_t a = SmemDescSw128(SmemAddr(sQ + (w.turns ? 0 : i) * Cfg::kUnit + (kk / 4) * kTaHalf)) + (uint64_t)(2 * (kk % 4));
          const uint64_t b = SmemDescSw128(SmemAddr(ring + st * Cfg::kUnit + (kk / 4) * kTaHalf)) + (uint64_t)(2 * (kk % 4));
          UmmaBf16(tmem + 128u * i, a, b, idesc, kk > 0 ? 1u : 0u);
        }
        UmmaCommit(&sh->s_full[i]);
      }
    };
    const auto values = [&](int i, int t, int st) {
      const int steps16 = (blk.Seen(i, blk.Index(i, t)) + 15) / 16;
      if (lane == 0) {
        TcgenFenceAfter();
        // MN-major, 128-byte swizzle: 64-value columns kTaHalf apart, groups of 8 keys 1024 bytes apart
        uint64_t b = (uint64_t)((SmemAddr(ring + st * Cfg::kUnit) & 0x3FFFF) >> 4) | (uint64_t)(kTaHalf >> 4) << 16 |
                     (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
        for (int kk = 0; kk < steps16; kk++)
          UmmaTmemA(tmem + 256u + 128u * i, tmem + 128u * i + 8u * kk, b + (uint64_t)(kk * (2048 >> 4)), idesc_pv, t > 0 || kk > 0 ? 1u : 0u);
        if (t + 1 == w.blocks[i]) UmmaCommit(&sh->o_full[i]);
      }
    };
    const auto release = [&](int st) {
      if (lane == 0) UmmaCommit(&sh->empty[st]);
    };
    // rows of V behind the sequence's end, as far as the last 16-key step reaches, become 0
    const auto trim = [&](int b, int st) {
      const int keys = blk.Keys(b), upto = (keys + 15) & ~15;
      if (keys == upto || !ok) return;
      const int pieces = (upto - keys) * 8;
      for (int h = 0; h < Cfg::kHalves; h++)
        for (int c = lane; c < pieces; c += 32)
          *reinterpret_cast<uint4*>(ring + st * Cfg::kUnit + h * kTaHalf + (keys + (c >> 3)) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
      FenceProxyAsyncShared();
      __syncwarp();
    };
    ok = TaWait(sh, &sh->q_full, 0);
    if (w.turns) {
      for (int i = 0; i < 2 && ok; i++)
        if (w.blocks[i] > 0) {
          const int st = acquire();
          if (!ok) break;
          scores(i, 0, st);
          release(st);
        }
      for (int t = 0; t < steps && ok; t++)
        for (int i = 0; i < 2 && ok; i++) {
          if (t < w.blocks[i]) {
            const int st = acquire();
            trim(blk.Index(i, t), st);
            ok = ok && TaWait(sh, &sh->p_full[i], (uint32_t)(t & 1));
            if (!ok) break;
            values(i, t, st);
            release(st);
          }
          if (t + 1 < w.blocks[i]) {
            const int st = acquire();
            if (!ok) break;
            scores(i, t + 1, st);
            release(st);
          }
        }
    } else if (steps > 0) {
      // blocks[0] <= blocks[1], or there is no tile 1: the last tile of a step releases its units
      const int last0 = w.blocks[1] > 0 ? 1 : 0;
      int st = acquire();
      for (int i = 0; i <= last0 && ok; i++) scores(i, 0, st);
      if (ok) release(st);
      for (int t = 0; t < steps && ok; t++) {
        const int vst = acquire();
        trim(blk.Index(0, t), vst);
        int kst = -1;
        for (int i = 0; i < 2 && ok; i++) {
          if (t >= w.blocks[i]) continue;
          ok = TaWait(sh, &sh->p_full[i], (uint32_t)(t & 1));
          if (!ok) break;
          values(i, t, vst);
          if (i == last0) release(vst);
          if (t + 1 < w.blocks[i]) {
            if (kst < 0) kst = acquire();
            if (!ok) break;
            scores(i, t + 1, kst);
            if (i == last0) release(kst);
          }
        }
      }
    }
    if (lane == 0) UmmaCommit(&sh->drained);
    __syncwarp();
    MbarWaitBounded(&sh->drained, 0, kOpsWaitLimit);  // no product reads shared memory or TMEM after this
  } else {
    // ---- softmax: thread = row of its tile = TMEM lane ----
    const int i = warp >> 2, r = threadIdx.x & 127;
    const int token = r / A.G, g = r - token * A.G;
    const int tok0 = w.q0 + (w.turns ? 0 : i * A.TB);  // the tile's first token
    const bool mine = token < w.tokens[i];
    const bool busy = (r & ~31) < w.tokens[i] * A.G;  // some row of this warp is in use
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t scol = lanes + 128u * i, ocol = lanes + 256u + 128u * i;
    const float sc = A.scale_log2;
    constexpr float kBias = F16 ? 7.f : 0.f;  // probabilities up to 2^15 in fp16: 7 more bits above its smallest numbers
    unsigned long long bits = 0;
    if constexpr (TREE) {
      if (mine) bits = A.masks[w.start + tok0 + token];
      if (w.nodes < 64) bits &= (1ull << w.nodes) - 1;
    }
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int t = 0; t < w.blocks[i]; t++) {
      const int b = blk.Index(i, t), seen = blk.Seen(i, b);
      // columns this row sees: 0 .. lim-1, or the bits of the mask
      unsigned long long m0, m1;
      bool cut;
      if (TREE) {
        if (b < w.cache_blocks) {
          m0 = seen >= 64 ? ~0ull : (1ull << seen) - 1;
          m1 = seen >= 128 ? ~0ull : seen > 64 ? (1ull << (seen - 64)) - 1 : 0;
          const int* tb = A.table + (long long)w.seq * A.max_blocks + 2 * b;
          const int p0 = tb[0], p1 = 2 * b + 1 < A.max_blocks ? tb[1] : -1;
          if (p0 < 0 || p0 >= A.pages) m0 = 0;
          if (p1 < 0 || p1 >= A.pages) m1 = 0;
          cut = (m0 & m1) != ~0ull;
        } else {
          m0 = bits;
          m1 = 0;
          cut = true;
        }
      } else {
        const int lim = min(seen, tok0 + token - 128 * b + 1);
        m0 = lim >= 64 ? ~0ull : lim > 0 ? (1ull << lim) - 1 : 0;
        m1 = lim >= 128 ? ~0ull : lim > 64 ? (1ull << (lim - 64)) - 1 : 0;
        cut = tok0 < 128 * b + 127 || seen < 128;
      }
      ok = TaWait(sh, &sh->s_full[i], (uint32_t)(t & 1));
      if (!ok) break;
      TcgenFenceAfter();
      if (busy) {
        uint32_t s[128];
        if (!cut) {
#pragma unroll
          for (int c = 0; c < 4; c++) TmemLoad32(scol + 32u * c, s + 32 * c);
          TmemWaitLd();
        } else {
#pragma unroll
          for (int c = 0; c < 4; c++) {
            if (32 * c < seen) {
              TmemLoad32(scol + 32u * c, s + 32 * c);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k++) s[32 * c + k] = 0;
            }
          }
          TmemWaitLd();
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const uint32_t bm = (uint32_t)((c < 2 ? m0 : m1) >> (32 * (c & 1)));
#pragma unroll
            for (int k = 0; k < 32; k++)
              if (!(bm >> k & 1)) s[32 * c + k] = 0xff800000u;
          }
        }
        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; c++) x[c & 3] = fmaxf(x[c & 3], __uint_as_float(s[c]));
        const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (t == 0) {
          m = mx;
        } else if (__any_sync(0xffffffffu, (mx - m) * sc > kTaLazy)) {
          // block t-1's products are complete: S of block t was issued behind them
          const float mn = fmaxf(m, mx);
          const float alpha = mn == -INFINITY ? 1.f : Exp2((m - mn) * sc);
          m = mn;
          l *= alpha;
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            uint32_t o[32];
            TmemLoad32(ocol + 32u * c, o);
            TmemWaitLd();
#pragma unroll
            for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            TmemStore32(ocol + 32u * c, o);
          }
        }
        const float neg = m == -INFINITY ? 0.f : kBias - m * sc;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; c++) {
          if (c == 0 || 32 * c < seen) {
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; k++) {
              const float p0 = Exp2(fmaf(__uint_as_float(s[32 * c + 2 * k]), sc, neg));
              const float p1 = Exp2(fmaf(__uint_as_float(s[32 * c + 2 * k + 1]), sc, neg));
              sum[(2 * k) & 3] += p0;
              sum[(2 * k + 1) & 3] += p1;
              p[k] = Pack2<F16>(p0, p1);
            }
            TmemStore16(scol + 16u * c, p);
          }
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        TmemWaitSt();
      }
      TcgenFenceBefore();
      MbarArrive(&sh->p_full[i]);
    }
    // ---- the rows' results ----
    const bool merge = TREE && w.turns && w.blocks[1] > 0;
    bool have = w.blocks[i] > 0;
    if (have) have = TaWait(sh, &sh->o_full[i], 0);
    float* shared_o = reinterpret_cast<float*>(ring);  // tile 1's accumulator: [value][row], then its maximum and sum
    if (merge) {
      if (i == 1) {
        have = TaWait(sh, &sh->o_full[0], 0) && have;  // all loads and products are done: the ring is free
        TcgenFenceAfter();
        if (busy) {
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            uint32_t o[32];
            TmemLoad32(ocol + 32u * c, o);
            TmemWaitLd();
            if (have) {
#pragma unroll
              for (int k = 0; k < 32; k++) shared_o[(32 * c + k) * 128 + r] = __uint_as_float(o[k]);
            }
          }
          if (have) {
            shared_o[D * 128 + r] = m;
            shared_o[D * 128 + 128 + r] = l;
          }
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    if (busy && !(w.turns && i == 1)) {
      TcgenFenceAfter();
      float a0 = 1.f, a1 = 0.f;
      if (merge) {
        const float m2 = shared_o[D * 128 + r], l2 = shared_o[D * 128 + 128 + r];
        const float mn = fmaxf(m, m2);
        if (mn != -INFINITY) {
          a0 = Exp2((m - mn) * sc);
          a1 = Exp2((m2 - mn) * sc);
        }
        m = mn;
        l = l * a0 + l2 * a1;
      }
      const bool parts = TREE && A.nsplit > 1;
      if (!parts) {
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // nothing seen: 0; NaN stays
        a0 *= inv;
        a1 *= inv;
      }
      const int node = tok0 + token;
      uint16_t* out = A.out + (long long)(w.start + node) * A.out_row + (long long)(w.head * A.G + g) * A.out_head;
      const long long slot =
          parts ? ((long long)(w.seq * A.Hk + w.head) * A.nsplit + blockIdx.x % A.nsplit) * (A.max_nodes * A.G) + node * A.G + g : 0;
#pragma unroll
      for (int c = 0; c < D / 32; c++) {
        uint32_t o[32];
        if (have) {
          TmemLoad32(ocol + 32u * c, o);
          TmemWaitLd();
        } else {
#pragma unroll
          for (int k = 0; k < 32; k++) o[k] = 0;
        }
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = __uint_as_float(o[k]) * a0;
        if (merge) {
#pragma unroll
          for (int k = 0; k < 32; k++) v[k] = fmaf(shared_o[(32 * c + k) * 128 + r], a1, v[k]);
        }
        if (!parts && l == 0.f) {
#pragma unroll
          for (int k = 0; k < 32; k++) v[k] = 0.f;
        }
        if (mine && ok) {
          if (parts) {
            float4* dst = reinterpret_cast<float4*>(A.part_o + slot * D + 32 * c);
#pragma unroll
            for (int k = 0; k < 8; k++) dst[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          } else {
            uint4* dst = reinterpret_cast<uint4*>(out + 32 * c);
#pragma unroll
            for (int k = 0; k < 4; k++)
              dst[k] = make_uint4(Pack2<F16>(v[8 * k], v[8 * k + 1]), Pack2<F16>(v[8 * k + 2], v[8 * k + 3]),
                                  Pack2<F16>(v[8 * k + 4], v[8 * k + 5]), Pack2<F16>(v[8 * k + 6], v[8 * k + 7]));
          }
        }
      }
      if (parts && mine && ok) A.part_ml[slot] = make_float2(m * sc, l);
    }
  }
  TcgenFenceBefore();
  __syncthreads();
  TcgenFenceAfter();
  if (warp == 8) TmemDealloc(tmem, 512);
}

// Joins the parts of a tree call's rows: one warp per (row, query head), D / 32 values per lane.
template <int D, bool F16>
__global__ void __launch_bounds__(256) TreeJoinKernel(const __grid_constant__ TaArgs A) {
  GridDepWait();
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)A.rows * A.H) return;
  const int row = (int)(item / A.H), h = (int)(item - (long long)row * A.H);
  if (row < A.offsets[0] || row >= A.offsets[A.n]) return;
  const int s = SequenceOf(A.offsets, A.n, row), node = row - A.offsets[s];
  if (node >= A.max_nodes) return;
  const int kv = h / A.G, stride = A.max_nodes * A.G;
  const long long slot = ((long long)s * A.Hk + kv) * A.nsplit * stride + node * A.G + (h - kv * A.G);
  float m = -INFINITY;
  for (int k = 0; k < A.nsplit; k++) m = fmaxf(m, A.part_ml[slot + (long long)k * stride].x);
  float l = 0.f, v[D / 32] = {};
  for (int k = 0; k < A.nsplit; k++) {
    const float2 ml = A.part_ml[slot + (long long)k * stride];
    const float a = m == -INFINITY ? 0.f : Exp2(ml.x - m);
    l = fmaf(ml.y, a, l);
    const float* o = A.part_o + (slot + (long long)k * stride) * D + lane * (D / 32);
#pragma unroll
    for (int j = 0; j < D / 32; j++) v[j] = fmaf(o[j], a, v[j]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = A.out + (long long)row * A.out_row + (long long)h * A.out_head + lane * (D / 32);
#pragma unroll
  for (int j = 0; j < D / 32; j++) {
    const float x = l == 0.f ? 0.f : v[j] * inv;
    out[j] = (uint16_t)Pack2<F16>(x, 0.f);
  }
}

}  // namespace shahd
