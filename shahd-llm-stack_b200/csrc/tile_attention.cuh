// Attention of 128-row query tiles on the tensor cores, for two operators:
//   packed prompts  out[i] = sum_{j <= i} softmax_j(scale q[i].k[j]) v[j] within each sequence (MultiHeadAttention.ts:46-74,
//                   CausalSoftmax.ts:17-33, for sequences of different lengths in one call), and
//   trees           the drafted nodes of a sequence against its cached positions and against each other by a bit mask.
//
// A tile's rows are (token, query head of one kv head) pairs, tokens outside: 128/G tokens times G heads, so the G heads
// that share keys sit in one tile, a decode step of few rows fills what it can, and a tile's last key block is cut close to
// the diagonal. A block of threads works on two tiles at a time: on two neighbours that read the same keys, or, when a
// sequence has only one tile of rows (decode steps, small trees), on those of two kv heads or on one tile twice, with the key
// blocks dealt out by turns and one merge at the end: so there is always one tile's softmax under the other's products.
//
//   S = Q K^T   tcgen05 M 128, N up to a block of 128 (head_dim 128) or 64 keys, into TMEM;
//   softmax     one thread per row: the row's scores of a block in registers, running maximum and sum in 32 bits; the maximum
//               moves only when a row's new one is over 8 (in log2) above it, since a probability of up to 2^8 costs
//               nothing in floating point: then, rarely, the accumulator in TMEM is scaled;
//   O += P V    P rounded to 16 bits (as every attention on these units) overwrites S in TMEM and is the A operand there; V
//               is the MN-major B operand; O stays in TMEM until the end.
// Keys and values come by TMA (128-byte swizzle) through a ring of one block's K or V; the cache's pages are boxes of 64
// positions.
// A block that is cut short (a sequence's end, the diagonal) loads only the 64-row boxes and multiplies only the 16-key
// steps that hold keys; rows of V behind a sequence's end are zeroed in shared memory, since 0 * inf would not be 0.
//
// Warps 0-3 and 4-7: the softmax of tile 0 and 1; warp 8: MMA issue; warp 9: loads; at head_dim 128, warps 10 and 11 only complete
// the third warpgroup, which gives registers to the other two.
#pragma once


#include "ops_common.cuh"
#include "rope.cuh"

namespace shahd {

constexpr int kTaBox = 8192;    // 64 rows of 64 values
constexpr int kTaQHalf = 16384;  // 128 rows of 64 values
constexpr float kTaLazy = 8.f;   // log2 of what a probability may grow to before the accumulator is scaled

// head_dim 128: blocks of 128 keys, and one block of threads per multiprocessor, whose TMEM it fills: S 2 x 128 columns (P over
// S), O 2 x 128. Its products and its exponentials take about the same 2048 clocks per step of two tiles.
// head_dim 64 and 32: products take half of that or less, so the steps are a chain of latencies around the exponentials.
// Blocks of 64 keys (S 2 x 64 columns, O 2 x 64) let two blocks of threads share a multiprocessor, four softmax warps to a
// scheduler instead of two (8192 tokens, 16 heads of 64: 218 us -> 196 us; 2048 tokens, 64 heads: 74 -> 60).
template <int D>
struct TaCfg {
  static constexpr bool kWide = D == 128;
  static constexpr int kKeys = kWide ? 128 : 64;
  static constexpr int kPerSm = kWide ? 1 : 2;
  static constexpr int kThreads = kWide ? 384 : 320;
  static constexpr int kHalves = kWide ? 2 : 1;        // 64-value columns of a row (head_dim 32: half of one, the rest zero)
  static constexpr int kQTile = kTaQHalf * kHalves;
  static constexpr int kHalf = kKeys * 128;            // a block's K or V: kHalves of these
  static constexpr int kUnit = kHalf * kHalves;
  static constexpr int kUnits = kWide ? 5 : 8;         // ring depth
  static constexpr int kSmem = 1024 + 2 * kQTile + kUnits * kUnit + 768 + 1024;
  static constexpr uint32_t kCols = kWide ? 512 : 256, kO = 2 * kKeys, kOStep = kWide ? 128 : 64;
  // of 16 pairs of probabilities, those that Exp2Poly takes
  static constexpr int kPoly = kWide ? 3 : 2;
};
// Registers at head_dim 128: launched with 168 per thread (384 x 168 = 64512). The two softmax warpgroups take 216 each, the third
// one, whose warps issue copies and products, keeps 72: 2 x 128 x 216 + 128 x 72 = 64512.
constexpr int kTaRegsSoftmax = 216, kTaRegsIssue = 72;

struct TaShared {
  uint64_t full[8], empty[8], q_full, q_empty, s_full[2], p_half[2], p_full[2], o_full[2], ml_full, ml_free, drained;
  uint64_t work_full[4], work_read[4];
  int4 work[4][4];  // trees: what the block works on, by turns; the loading warp writes it
  uint32_t tmem;
  volatile int abort;
  int found_seq, found_at, sums[12];  // trees: where the block's range begins
};
static_assert(sizeof(TaShared) <= 768, "TaShared");

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
  int max_blocks, pages, max_nodes, pairs, two_heads;  // two_heads: the pair's tiles are those of two kv heads
  // All key blocks of all tile pairs in one line, dealt out to the blocks of threads in ranges of equal length, at least
  // `least`: 0 where every pair has a block of threads of its own instead. A pair that a range cuts leaves parts: block of threads c
  // has room for two, [2 c] for a pair that it does not begin and [2 c + 1] for one that it does not end.
  int least, part_rows;
  float* part_o;    // [2 grid, part_rows, D]
  float2* part_ml;  // [2 grid, part_rows]: -Offset() of the running maximum, and the sum
  int* plan;        // the ranges' length, then for every sequence the blocks of all before it, and their total
};

__device__ __forceinline__ void TmaLoad3D(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          SmemAddr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(SmemAddr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Products and commits that a whole warp runs through and one elected lane issues. The warp's control flow and operands are
// kept uniform (Uniform(), votes on waits), so that descriptors stay in uniform registers: from ordinary ones each
// product took 67 cycles to issue in a loop, and 100 to 200 between the softmax warps' instructions.
// D[tmem] (+)= A[smem] B[smem], kind::f16.
__device__ __forceinline__ void UmmaIssueSS(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem], kind::f16.
__device__ __forceinline__ void UmmaIssueTS(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void UmmaIssueCommit(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(SmemAddr(bar))
      : "memory");
}
__device__ __forceinline__ int Uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// 16 consecutive columns per thread to TMEM.
__device__ __forceinline__ void TmemStore16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void TmemWaitSt() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void RegsUp() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void RegsDown() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Two floats in a register pair: one instruction for both.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 Two(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void Split(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 Fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 Add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest of three, NaN if one of them is.
__device__ __forceinline__ float Max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x of two values on the FMA units, for a part of the probabilities: the unit that Exp2 runs on gives 16 results a clock, and
// a 128 x 128 block of scores wants 16384 of them next to products of 1024 (head_dim 128) or 512 clocks. x = n + f with n the
// nearest integer (adding 1.5 * 2^23 leaves n in the low bits), 2^f by the degree-4 polynomial of least greatest relative
// error on [-1/2, 1/2] (Remez exchange; 2.7e-6 in 32 bits, a thousandth of a bf16 rounding), n added to the exponent.
// x is cut at -126: what is smaller becomes 2^-126, nothing next to a sum that holds at least one 2^-8. NaN and infinite x give
// numbers that mean nothing: Spoil() sees to the rows that have them.
__device__ __forceinline__ f32x2 Exp2Poly(float a, float b) {
  const f32x2 magic = Two(12582912.f, 12582912.f), x = Two(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const f32x2 r = Add2(x, magic);
  const f32x2 f = Add2(x, Fma2(r, Two(-1.f, -1.f), magic));
  f32x2 p = Fma2(Two(0.009570102207362652f, 0.009570102207362652f), f, Two(0.05591785907745361f, 0.05591785907745361f));
  p = Fma2(p, f, Two(0.240247443318367f, 0.240247443318367f));
  p = Fma2(p, f, Two(0.6931217908859253f, 0.6931217908859253f));
  p = Fma2(p, f, Two(0.9999992847442627f, 0.9999992847442627f));
  float p0, p1, r0, r1;
  Split(p, p0, p1);
  Split(r, r0, r1);
  return Two(__uint_as_float(__float_as_uint(p0) + (__float_as_uint(r0) << 23)), __uint_as_float(__float_as_uint(p1) + (__float_as_uint(r1) << 23)));
}

// A probability is 2^(s * scale + Offset(m)), one fused step per score. The offset is rounded, by up to 2^-24 of m * scale: a factor
// of all the row's probabilities, which leaves with the division by their sum as long as every place that changes from one
// maximum to another takes the difference of the rounded offsets.
__device__ __forceinline__ float Offset(float m, float scale, float bias) { return fmaf(-m, scale, bias); }
// What a row's maximum adds to its sum at the end: 0, or NaN where the row's weights mean nothing or that factor could leave the
// range that P has: scores that are not finite, or so large that it reaches 2^64 (bf16, at 2^30) or a quarter (fp16, whose P may
// grow to 2^15, at 2^23). Carried by the maximum, which a NaN or +inf never leaves again, such scores cost nothing per step, and the row
// comes out NaN whichever way its exponentials are formed. What a maximum below that range leaves behind when it moves up is
// multiplied by 2^-inf: gone, or NaN where it was infinite. -inf stands for no key yet, or only ones of weight 0, told apart at the end.
template <bool F16>
__device__ __forceinline__ float Spoil(float m, float scale) {
  constexpr float kMost = F16 ? 8388608.f : 1073741824.f;
  return fabsf(m * scale) < kMost ? 0.f : NAN;
}

// 32 bytes at once: a whole sector, where 16-byte stores of lanes that lie a row apart write halves.
__device__ __forceinline__ void Store32B(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

template <bool F16>
__device__ __forceinline__ uint32_t Pack2(float a, float b) {  // a in the low half
  uint32_t r;
  if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// A wait that ends: false once it, or another warp's, has given up. (Not unrolled: copies of the loop at every wait made the
// kernel larger than the instruction cache, and the warp that issues the products as slow as its fetches.)
__device__ __forceinline__ bool TaWait(TaShared* sh, uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < kOpsWaitLimit; i++) {
    if (MbarTryWait(bar, parity)) return true;
    if (sh->abort) return false;
  }
  atomicCAS(&g_ops_device_error, 0, kOpsErrTimeout);
  sh->abort = 1;
  return false;
}
// At the end of a block, whatever has given up before: what is in flight into the block's memory is waited for, within the limit.
__device__ __forceinline__ void TaDrain(uint64_t* bar, uint32_t parity) {
  if (!MbarWaitBounded(bar, parity, kOpsWaitLimit)) atomicCAS(&g_ops_device_error, 0, kOpsErrTimeout);
}
// The same for a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool TaWaitWarp(TaShared* sh, uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < kOpsWaitLimit; i++) {
    if (__all_sync(0xffffffffu, MbarTryWait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, sh->abort)) return false;
  }
  atomicCAS(&g_ops_device_error, 0, kOpsErrTimeout);
  sh->abort = 1;
  return false;
}

// Two barriers under one vote.
__device__ __forceinline__ bool TaWaitWarp2(TaShared* sh, uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
  const bool ra = MbarTryWait(a, pa), rb = MbarTryWait(b, pb);
  if (__all_sync(0xffffffffu, ra && rb)) return true;
  return TaWaitWarp(sh, a, pa) && TaWaitWarp(sh, b, pb);
}

// What the two tiles are: neighbours of one kv head that read the same key blocks; one tile of rows, its key blocks dealt out by
// turns and the results merged; or the one tile of rows of two kv heads, `head` and the next.
enum TaMode { kShared = 0, kTurns = 1, kHeads = 2 };

// What a block of threads works on at a time: key blocks of two tiles of rows.
struct TaWork {
  int seq, start;       // sequence and its first row
  int head;             // kv head
  int q0;               // first token of tile 0 within the sequence
  int tokens0, tokens1;  // of the tiles
  int blocks0, blocks1;  // key blocks of the tiles
  int turns;            // kShared, kTurns or kHeads
  int first;            // trees: first key block
  int cached;           // trees: cached positions
  int cache_blocks;     // trees: key blocks of the cache
  int nodes;            // trees: rows of the sequence; prompts: tokens of the sequence
  int part;             // trees: the place of the results among the block's parts, or -1: these are all key blocks
  int more;             // trees: there is another pair behind this one
  __device__ __forceinline__ int Tokens(int i) const { return i ? tokens1 : tokens0; }
  __device__ __forceinline__ int Blocks(int i) const { return i ? blocks1 : blocks0; }
};

// The pair of tiles that a block of threads takes: number `rank` of `all` places, of which some are empty. Each warp finds the same.
// The later a pair lies in its sequence, the more keys it has, and the longest should start first. 2 to 128 sequences, whose
// lengths fit a warp's registers: pairs go by their place in the sequence, last places first, over all sequences together, by a
// search for the place that number `rank` falls on (16 prompts of 300 to 2048 tokens, 16/4 heads of 64: 112 us, by sequences
// 118; 2 prompts of 7000 to 8192, 16/2 heads of 128, whose blocks all take long: 530 and 525). One sequence, where the
// order is the same without the search (64/16 heads of 64 over 2048 tokens: 60 us, with it 62), and more than 128 go by
// sequences: s owns places offsets[s] / span + s .. offsets[s+1] / span + s, at least as many as it needs, which a search in
// the offsets finds.
template <int KEYS>
__device__ __forceinline__ bool PromptWork(const TaArgs& A, int rank, int all, TaWork& w) {
  const int lane = threadIdx.x & 31, span = 2 * A.TB;
  const auto off = [&](int s) { return min(max(A.offsets[s], 0), A.rows); };
  int seq, local;
  if (A.n > 1 && A.n <= 128) {
    int count[4], most = 0, total = 0;
#pragma unroll
    for (int m = 0; m < 4; m++) {
      const int s = lane + 32 * m;
      count[m] = s < A.n ? (max(off(s + 1) - off(s), 0) + span - 1) / span : 0;
      most = max(most, count[m]);
      total += count[m];
    }
    most = __reduce_max_sync(0xffffffffu, most);
    total = __reduce_add_sync(0xffffffffu, total);
    if (rank >= total) return false;
    const auto from = [&](int j) {  // pairs at place j or behind it
      int v = 0;
#pragma unroll
      for (int m = 0; m < 4; m++)
        if (32 * m < A.n) v += max(count[m] - j, 0);
      return (int)__reduce_add_sync(0xffffffffu, v);
    };
    int lo = 0, hi = most, behind = 0;  // from(lo) > rank >= from(hi) = behind
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, f = from(mid);
      if (f > rank) lo = mid;
      else {
        hi = mid;
        behind = f;
      }
    }
    local = lo;
    seq = 0;
    int nth = rank - behind;  // the sequence: the nth of those with a pair at that place
#pragma unroll
    for (int m = 0; m < 4; m++) {
      if (32 * m >= A.n) break;
      const bool mine = count[m] > local;
      const unsigned have = __ballot_sync(0xffffffffu, mine);
      const unsigned hit = __ballot_sync(0xffffffffu, mine && __popc(have & ((1u << lane) - 1)) == nth);
      if (hit) seq = 32 * m + __ffs(hit) - 1;
      nth -= __popc(have);
    }
  } else {
    const int tile = all - 1 - rank;
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
    seq = lo;
    local = tile - (off(lo) / span + lo);
  }
  w.seq = seq;
  w.start = off(seq);
  const int len = max(off(seq + 1) - w.start, 0);
  w.nodes = len;
  w.q0 = local * span;
  if (local < 0 || w.q0 >= len) return false;
  w.tokens0 = min(len - w.q0, A.TB);
  w.tokens1 = min(max(len - w.q0 - A.TB, 0), A.TB);
  w.blocks0 = (w.q0 + w.tokens0 + KEYS - 1) / KEYS;
  w.blocks1 = w.tokens1 > 0 ? (w.q0 + A.TB + w.tokens1 + KEYS - 1) / KEYS : 0;
  w.turns = 0;
  w.first = w.cached = w.cache_blocks = 0;
  w.part = -1;
  return true;
}

// A sequence of a tree call: its rows, cached positions, tile pairs and key blocks (its own rows are the last block).
template <int KEYS>
struct TreeSeq {
  int start, nodes, cached, pairs, blocks;
  __device__ __forceinline__ TreeSeq(const TaArgs& A, int s) {
    start = min(max(A.offsets[s], 0), A.rows);
    nodes = min(min(max(A.offsets[s + 1], start), A.rows) - start, A.max_nodes);
    cached = (int)min((long long)max(A.lengths[s], 0), (long long)A.max_blocks * kOpsPage);
    pairs = (nodes + 2 * A.TB - 1) / (2 * A.TB);
    blocks = (cached + KEYS - 1) / KEYS + 1;
  }
};

// The key blocks of a tree call that this block of threads takes, pair by pair.
template <int KEYS>
struct TreeWalk {
  const TaArgs& A;
  TreeSeq<KEYS> q;         // of `seq`
  int seq, item, at, pos, end;  // the pair's sequence, number in it and first block; the range that is left
  // From block `at_` of sequence seq_'s on, pos_ in the line, to end_.
  __device__ __forceinline__ TreeWalk(const TaArgs& a, int seq_, int at_, int pos_, int end_)
      : A(a), q(a, seq_), seq(seq_), item(at_ / q.blocks), at(at_ - item * q.blocks), pos(pos_), end(end_) {}
  // Tile pairs of a sequence.
  static __device__ __forceinline__ int Items(const TaArgs& A, const TreeSeq<KEYS>& q) {
    return A.two_heads ? (q.pairs > 0 ? A.Hk / 2 : 0) : A.Hk * q.pairs;
  }
  // The next pair's work; there is one (pos < end).
  __device__ __forceinline__ TaWork Take() {
    TaWork w;
    const int count = min(q.blocks - at, end - pos);
    w.seq = seq;
    w.start = q.start;
    w.nodes = q.nodes;
    w.cached = q.cached;
    w.cache_blocks = q.blocks - 1;
    w.head = A.two_heads ? 2 * item : item / q.pairs;
    w.q0 = A.two_heads ? 0 : (item - w.head * q.pairs) * 2 * A.TB;
    w.tokens0 = min(w.nodes - w.q0, A.TB);
    w.tokens1 = min(max(w.nodes - w.q0 - A.TB, 0), A.TB);
    w.first = at;
    w.part = count == q.blocks ? -1 : 2 * (int)blockIdx.x + (at > 0 ? 0 : 1);
    w.turns = A.two_heads ? kHeads : w.tokens1 == 0 ? kTurns : kShared;
    if (w.turns != kShared) w.tokens1 = w.tokens0;
    if (w.turns == kTurns) {
      w.blocks0 = (count + 1) / 2;
      w.blocks1 = count / 2;
    } else {
      w.blocks0 = w.blocks1 = count;
    }
    pos += count;
    w.more = pos < end;
    if (w.more) {
      item++;
      at = 0;
      while (item >= Items(A, q) && seq + 1 < A.n) {  // also past sequences without rows
        item = 0;
        q = TreeSeq<KEYS>(A, ++seq);
      }
    }
    return w;
  }
};

struct NoWalk {  // where there are no ranges
  __device__ __forceinline__ NoWalk(const TaArgs&, int, int, int, int) {}
};

// Where this block of threads begins: the sequence, its key block in the line of the sequence's pairs, the range. All of its
// threads take part; false: there is nothing for it.
template <int KEYS, bool RANGES>
__device__ __forceinline__ bool TreeBegin(const TaArgs& A, TaShared* sh, int& seq, int& at, int& pos, int& end) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto work = [&](int s) {
    if (s >= A.n) return 0;
    const TreeSeq<KEYS> q(A, s);
    return TreeWalk<KEYS>::Items(A, q) * q.blocks;
  };
  if constexpr (!RANGES) {
    const int items = A.two_heads ? A.Hk / 2 : A.Hk * A.pairs;
    seq = blockIdx.x / items;
    const int item = blockIdx.x - seq * items;
    const TreeSeq<KEYS> q(A, seq);
    at = item * q.blocks;
    pos = 0;
    end = q.blocks;
    return item < TreeWalk<KEYS>::Items(A, q);
  } else {
    const int first = work(threadIdx.x);
    int sum = first;
    for (int s = threadIdx.x + blockDim.x; s < A.n; s += blockDim.x) sum += work(s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh->sums[warp] = sum;
    __syncthreads();
    int total = 0;
    for (int k = 0; k < warps; k++) total += sh->sums[k];
    const int per = max(A.least, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    pos = (int)min((long long)blockIdx.x * per, (long long)total);
    end = min(pos + per, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) A.plan[0] = per;
    if (pos >= end && blockIdx.x != 0) return false;
    int before = 0;
    for (int s0 = 0; s0 < A.n; s0 += blockDim.x) {
      const int s = s0 + threadIdx.x, mine = s0 == 0 ? first : work(s);
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      __syncthreads();
      if (lane == 31) sh->sums[warp] = incl;
      __syncthreads();
      int ahead = before;
      for (int k = 0; k < warps; k++) {
        if (k < warp) ahead += sh->sums[k];
        before += sh->sums[k];
      }
      ahead += incl - mine;
      if (blockIdx.x == 0 && s < A.n) A.plan[1 + s] = ahead;
      if (pos < end && ahead <= pos && pos < ahead + mine) {
        sh->found_seq = s;
        sh->found_at = pos - ahead;
      }
    }
    __syncthreads();
    if (pos >= end) return false;
    seq = sh->found_seq;
    at = sh->found_at;
    return true;
  }
}

__device__ __forceinline__ void PutWork(TaShared* sh, int slot, const TaWork& w) {
  sh->work[slot][0] = make_int4(w.seq, w.start, w.head, w.q0);
  sh->work[slot][1] = make_int4(w.tokens0, w.tokens1, w.blocks0, w.blocks1);
  sh->work[slot][2] = make_int4(w.turns, w.first, w.cached, w.cache_blocks);
  sh->work[slot][3] = make_int4(w.nodes, w.part, w.more, 0);
}
__device__ __forceinline__ void GetWork(const TaShared* sh, int slot, TaWork& w) {
  const int4 a = sh->work[slot][0], b = sh->work[slot][1], c = sh->work[slot][2], d = sh->work[slot][3];
  w.seq = Uniform(a.x);
  w.start = Uniform(a.y);
  w.head = Uniform(a.z);
  w.q0 = Uniform(a.w);
  w.tokens0 = Uniform(b.x);
  w.tokens1 = Uniform(b.y);
  w.blocks0 = Uniform(b.z);
  w.blocks1 = Uniform(b.w);
  w.turns = Uniform(c.x);
  w.first = Uniform(c.y);
  w.cached = Uniform(c.z);
  w.cache_blocks = Uniform(c.w);
  w.nodes = Uniform(d.x);
  w.part = Uniform(d.y);
  w.more = Uniform(d.z);
}

template <int KEYS, bool TREE>
struct TaBlocks {
  const TaArgs& A;
  const TaWork& w;
  // The key block of step t of tile i.
  __device__ __forceinline__ int Index(int i, int t) const { return TREE ? (w.turns == kTurns ? w.first + 2 * t + i : w.first + t) : t; }
  // Keys of a block that belong to the sequence (1 .. KEYS).
  __device__ __forceinline__ int Keys(int b) const {
    if constexpr (TREE) return b < w.cache_blocks ? min(KEYS, w.cached - KEYS * b) : w.nodes;
    else return min(KEYS, w.nodes - KEYS * b);
  }
  // Keys of a block that some row of tile i may see.
  __device__ __forceinline__ int Seen(int i, int b) const {
    if constexpr (TREE) return Keys(b);
    else return min(KEYS, w.q0 + i * A.TB + w.Tokens(i) - KEYS * b);
  }
};

// Prompts; trees with a block of threads for every tile pair; trees with a range of key blocks for every block of threads, pair after
// pair. (Pairs on their own are worth a kernel: what goes on from one pair to the next takes registers that head_dim 64
// does not have, and 256 single tokens over 512 positions took 27 us instead of 21.)
enum TaKind { kPrompt = 0, kTreePairs = 1, kTreeRanges = 2 };

template <int D, bool F16, int KIND>
__global__ void __launch_bounds__(TaCfg<D>::kThreads, TaCfg<D>::kPerSm) TileAttentionKernel(const __grid_constant__ TaArgs A) {
  constexpr bool TREE = KIND != kPrompt, RANGES = KIND == kTreeRanges;
  using Cfg = TaCfg<D>;
  constexpr int U = Cfg::kUnits, KEYS = Cfg::kKeys;
  extern __shared__ uint8_t ta_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ta_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = base;
  uint8_t* ring = base + 2 * Cfg::kQTile;
  TaShared* sh = reinterpret_cast<TaShared*>(ring + U * Cfg::kUnit);
  const int warp = Uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == 9 && lane < (TREE ? 4 : 3)) PrefetchTmaDesc(lane == 0 ? &A.qmap : lane == 1 ? &A.kmap : lane == 2 ? &A.vmap : &A.pool);
  GridDepWait();
  TaWork w;
  int begin_seq = 0, begin_at = 0, begin_pos = 0, begin_end = 0;
  if constexpr (TREE) {
    if (!TreeBegin<KEYS, RANGES>(A, sh, begin_seq, begin_at, begin_pos, begin_end)) return;
    if constexpr (!RANGES) {
      w = TreeWalk<KEYS>(A, begin_seq, begin_at, begin_pos, begin_end).Take();
      w.part = -1;
    }
  } else if (warp == 9) {  // one warp looks, the others prepare meanwhile
    w.head = blockIdx.x % A.Hk;
    if (!PromptWork<KEYS>(A, blockIdx.x / A.Hk, gridDim.x / A.Hk, w)) w.nodes = 0;
    if (lane == 0) PutWork(sh, 0, w);
  }
  if constexpr (KIND == kTreePairs) {
    w.seq = Uniform(w.seq);
    w.start = Uniform(w.start);
    w.head = Uniform(w.head);
    w.q0 = Uniform(w.q0);
    w.tokens0 = Uniform(w.tokens0);
    w.tokens1 = Uniform(w.tokens1);
    w.blocks0 = Uniform(w.blocks0);
    w.blocks1 = Uniform(w.blocks1);
    w.turns = Uniform(w.turns);
    w.first = Uniform(w.first);
    w.cached = Uniform(w.cached);
    w.cache_blocks = Uniform(w.cache_blocks);
    w.nodes = Uniform(w.nodes);
  }
  const TaBlocks<KEYS, TREE> blk{A, w};

  if (warp == 0) {
    if (lane < U) {
      MbarInit(&sh->full[lane], 1);
      MbarInit(&sh->empty[lane], 1);
    } else if (lane < U + 2) {
      const int i = lane - U;
      MbarInit(&sh->s_full[i], 1);
      MbarInit(&sh->p_half[i], 128);
      MbarInit(&sh->p_full[i], 128);
      MbarInit(&sh->o_full[i], 1);
    } else if (lane < U + 6) {
      MbarInit(&sh->work_full[lane - U - 2], 1);
      MbarInit(&sh->work_read[lane - U - 2], 9);  // by the MMA warp and the eight softmax warps
    } else if (lane == U + 6) {
      MbarInit(&sh->q_full, 1);
      MbarInit(&sh->q_empty, 1);
      MbarInit(&sh->ml_full, 128);
      MbarInit(&sh->ml_free, 128);
      MbarInit(&sh->drained, 1);
      sh->abort = 0;
    }
    FenceMbarInit();
  }
  if (warp == 8) {
    TmemAlloc(&sh->tmem, Cfg::kCols);
    TmemRelinquish();
  }
  TcgenFenceBefore();
  __syncthreads();
  TcgenFenceAfter();
  const uint32_t tmem = (uint32_t)Uniform((int)sh->tmem);
  if constexpr (KIND == kPrompt) {
    GetWork(sh, 0, w);
    w.turns = w.first = w.cached = w.cache_blocks = 0;
    w.part = -1;
    if (w.nodes == 0) {
      if (warp == 8) TmemDealloc(tmem, Cfg::kCols);
      return;
    }
  }
  // Ranges: work number `segment`, if there is any. The loading warp writes it down, in four places by turns; a warp that has no
  // rows for some time may be that far behind, so a place is written again only when all have read it (lane 0's values count).
  const auto next = [&](uint32_t segment, bool& ok) -> bool {
    if (!RANGES || !w.more) return false;
    const bool got = TaWaitWarp(sh, &sh->work_full[segment & 3], (segment >> 2) & 1);
    ok = ok && got;
    if (got) {
      GetWork(sh, segment & 3, w);
      if (lane == 0) MbarArrive(&sh->work_read[segment & 3]);
    }
    return got;
  };
  GridDepLaunch();  // after this block holds its TMEM
  float* const sml = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sh) + 768);  // tile 1's maxima and sums, for a merge

  if (warp >= 8) {
    if constexpr (Cfg::kWide) RegsDown<kTaRegsIssue>();
    if (warp == 9) {
      // The whole warp follows the same path, lane 0 issues. Lane l holds the l-th page of the 32 that come next.
      FenceProxyAsyncGlobal();
      constexpr int kPages = KEYS / 64;  // of a block
      int held = 0, ids = 0;             // the first of the 32 pages whose numbers the lanes hold
      const auto hold = [&](int from) {
        held = from;
        const int p = from + lane;
        ids = TREE && p < A.max_blocks ? A.table[(long long)w.seq * A.max_blocks + p] : -1;
        if (ids < 0 || ids >= A.pages) ids = A.pages;  // behind the pool: TMA fills zeros, and the keys are masked
      };
      int st = 0, issued = 0;
      uint32_t round = 0;  // times the ring has been gone through
      // one block's K or V into the next unit of the ring
      const auto load = [&](int b, int keys, bool value, int head) -> bool {
        if (round > 0 && !TaWaitWarp(sh, &sh->empty[st], (round - 1) & 1)) return false;
        uint8_t* dst = ring + st * Cfg::kUnit;
        const int boxes = keys > 64 ? 2 : 1;
        if (lane == 0) MbarArriveExpectTx(&sh->full[st], boxes * Cfg::kHalves * kTaBox);
        if (TREE && b < w.cache_blocks && b * kPages + boxes > held + 32) hold((b - 2) * kPages);  // by turns, a block before the last one can follow it
#pragma unroll 1
        for (int x = 0; x < boxes; x++) {
          if (TREE && b < w.cache_blocks) {
            const int page = __shfl_sync(0xffffffffu, ids, b * kPages + x - held);
            if (lane == 0)
              for (int h = 0; h < Cfg::kHalves; h++)
                TmaLoad3D(dst + h * Cfg::kHalf + x * kTaBox, &A.pool, &sh->full[st], 64 * h, (head * 2 + (value ? 1 : 0)) * kOpsPage, page);
          } else if (lane == 0) {
            const int row = w.start + (TREE ? 0 : KEYS * b) + 64 * x;
            for (int h = 0; h < Cfg::kHalves; h++)
              TmaLoad3D(dst + h * Cfg::kHalf + x * kTaBox, value ? &A.vmap : &A.kmap, &sh->full[st], 64 * h, head, row);
          }
        }
        issued++;
        if (++st == U) {
          st = 0;
          round++;
        }
        return true;
      };
      // the order in which the MMA warp takes them: K of the first blocks, then by steps V of this and K of the next one, for
      // both tiles at once or, by turns, for each
      bool ok = true;
      uint32_t segment = 0;
      typename std::conditional<RANGES, TreeWalk<KEYS>, NoWalk>::type walk(A, begin_seq, begin_at, begin_pos, begin_end);
      do {
        if (segment > 0) ok = TaWaitWarp(sh, &sh->q_empty, (segment - 1) & 1);
        if (!ok) break;
        if constexpr (RANGES) {
          w = walk.Take();
          if (segment >= 4) ok = TaWaitWarp(sh, &sh->work_read[segment & 3], ((segment >> 2) - 1) & 1);
          if (!ok) break;
          if (lane == 0) {
            PutWork(sh, segment & 3, w);
            MbarArrive(&sh->work_full[segment & 3]);
          }
          __syncwarp();
          GetWork(sh, segment & 3, w);
        }
        const int steps = max(w.blocks0, w.blocks1), last = w.tokens1 > 0 ? 1 : 0, units = w.turns ? 2 : 1;  // last: it sees most
        const int tiles = w.turns != kTurns && w.tokens1 > 0 ? 2 : 1;
        if (lane == 0) {
          MbarArriveExpectTx(&sh->q_full, tiles * Cfg::kHalves * A.G * A.TB * 128);
          for (int i = 0; i < tiles; i++)
            for (int h = 0; h < Cfg::kHalves; h++)
              TmaLoad3D(sQ + i * Cfg::kQTile + h * kTaQHalf, &A.qmap, &sh->q_full, 64 * h,
                        (w.head + (w.turns == kHeads ? i : 0)) * A.G, w.start + w.q0 + (w.turns == kShared ? i * A.TB : 0));
        }
        segment++;
        if (TREE) hold(w.first * kPages);
        const auto one = [&](int i, int t, bool value) {
          if (!ok || t >= (w.turns ? w.Blocks(i) : steps)) return;
          const int b = blk.Index(i, t);
          ok = load(b, w.turns ? blk.Keys(b) : blk.Seen(last, b), value, w.head + (w.turns == kHeads ? i : 0));
        };
        for (int i = 0; i < units; i++) one(i, 0, false);
#pragma unroll 1
        for (int t = 0; t < steps && ok; t++)
#pragma unroll 1
          for (int i = 0; i < units; i++) {
            one(i, t, true);
            one(i, t + 1, false);
          }
      } while (RANGES && ok && w.more);
      // every copy lands before the block may leave: the last phase of each unit's barrier
      if (segment > 0) TaDrain(&sh->q_full, (segment - 1) & 1);
      for (int v = max(0, issued - U); v < issued; v++) TaDrain(&sh->full[v % U], (uint32_t)((v / U) & 1));
    } else if (warp == 8) {
      // The whole warp follows the same path, one lane of it issues.
      constexpr uint32_t kTypes = F16 ? 0u : (1u << 7) | (1u << 10);
      constexpr uint32_t idesc0 = (1u << 4) | kTypes | ((128u >> 4) << 24);
      constexpr uint32_t idesc_pv = idesc0 | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // V is MN-major
      constexpr int kFull16 = KEYS / 16;
      int st = 0;
      uint32_t phase = 0;
      bool ok = true;
      const auto acquire = [&]() -> int {
        const int at = st;
        ok = ok && TaWaitWarp(sh, &sh->full[at], phase);
        if (++st == U) {
          st = 0;
          phase ^= 1;
        }
        return at;
      };
      int done0 = 0, done1 = 0;  // steps of the tiles in the segments before this one: barriers count on
      const auto wait = [&](uint64_t* bar, int i, int t) { ok = ok && TaWaitWarp(sh, bar, (uint32_t)((t + (i ? done1 : done0)) & 1)); };
      const uint64_t qdesc = SmemDescSw128(SmemAddr(sQ)), kdesc = SmemDescSw128(SmemAddr(ring));
      // MN-major, 128-byte swizzle: 64-value columns kHalf apart, groups of 8 keys 1024 bytes apart
      const uint64_t vdesc = (uint64_t)((SmemAddr(ring) & 0x3FFFF) >> 4) | (uint64_t)(Cfg::kHalf >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
                             (uint64_t)1 << 46 | (uint64_t)2 << 61;
      const auto scores = [&](int i, int t, int unit) {
        const int kc = (blk.Seen(i, blk.Index(i, t)) + 15) & ~15;
        const uint64_t a = qdesc + (uint64_t)((w.turns == kTurns ? 0 : i) * (Cfg::kQTile >> 4)), b = kdesc + (uint64_t)(unit * (Cfg::kUnit >> 4));
        const uint32_t idesc = idesc0 | ((uint32_t)(kc >> 3) << 17);
        TcgenFenceAfter();
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++)
          UmmaIssueSS(tmem + (uint32_t)(KEYS * i), a + (uint64_t)((kk / 4) * (kTaQHalf >> 4) + 2 * (kk % 4)),
                      b + (uint64_t)((kk / 4) * (Cfg::kHalf >> 4) + 2 * (kk % 4)), idesc, kk > 0 ? 1u : 0u);
        UmmaIssueCommit(&sh->s_full[i]);
      };
      // O += P V; at 128 keys the first 64 as soon as their probabilities are there
      const auto values = [&](int i, int t, int unit) {
        const int steps16 = (blk.Seen(i, blk.Index(i, t)) + 15) / 16;
        const uint64_t b = vdesc + (uint64_t)(unit * (Cfg::kUnit >> 4));
        const uint32_t d = tmem + Cfg::kO + Cfg::kOStep * i, a = tmem + (uint32_t)(KEYS * i);
        const uint32_t more = t > 0 ? 1u : 0u;
        const auto some = [&](int from, int to) {
#pragma unroll
          for (int kk = from; kk < to; kk++) UmmaIssueTS(d, a + 8u * kk, b + (uint64_t)(kk * (2048 >> 4)), idesc_pv, kk > 0 ? 1u : more);
        };
        if (Cfg::kWide && steps16 == kFull16) {
          wait(&sh->p_half[i], i, t);
          if (!ok) return;
          TcgenFenceAfter();
          some(0, 4);
        }
        wait(&sh->p_full[i], i, t);
        if (!ok) return;
        TcgenFenceAfter();
        if (steps16 == kFull16) {
          some(Cfg::kWide ? 4 : 0, kFull16);
        } else {
#pragma unroll 1
          for (int kk = 0; kk < steps16; kk++) UmmaIssueTS(d, a + 8u * kk, b + (uint64_t)(kk * (2048 >> 4)), idesc_pv, kk > 0 ? 1u : more);
        }
        if (t + 1 == w.Blocks(i)) UmmaIssueCommit(&sh->o_full[i]);
      };
      const auto release = [&](int unit) { UmmaIssueCommit(&sh->empty[unit]); };
      // rows of V behind the sequence's end, as far as the last 16-key step reaches, become 0
      const auto trim = [&](int b, int unit) {
        const int keys = blk.Keys(b), upto = (keys + 15) & ~15;
        if (keys == upto || !ok) return;
        const int pieces = (upto - keys) * 8;
        for (int h = 0; h < Cfg::kHalves; h++)
#pragma unroll 1
          for (int c = lane; c < pieces; c += 32)
            *reinterpret_cast<uint4*>(ring + unit * Cfg::kUnit + h * Cfg::kHalf + (keys + (c >> 3)) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        FenceProxyAsyncShared();
        __syncwarp();
      };
      uint32_t segment = 0;
      if constexpr (RANGES) w.more = 1;
      while ((segment == 0 && !RANGES) || next(segment, ok)) {
        const int steps = max(w.blocks0, w.blocks1);
        // A unit serves one tile, or both that share their keys: then the last tile of a step (tile 1, if there is one: blocks0 <= blocks1)
        // releases it.
        const int last = w.blocks1 > 0 ? 1 : 0;
        ok = TaWaitWarp(sh, &sh->q_full, segment & 1);
        segment++;
        int kunit = 0, vunit = 0;
        const auto next_scores = [&](int i, int t) {
          if (!ok || t >= w.Blocks(i)) return;
          if (w.turns) kunit = acquire();
          if (!ok) return;
          scores(i, t, kunit);
          if (w.turns || i == last) release(kunit);
        };
        const auto next_values = [&](int i, int t) {
          if (!ok || t >= w.Blocks(i)) return;
          if (w.turns) {
            vunit = acquire();
            trim(blk.Index(i, t), vunit);
          }
          values(i, t, vunit);
          if (ok && (w.turns || i == last)) release(vunit);
        };
        // prompts: V of step t and K of step t + 1, under one wait
        int vnext = 0, knext = 0;
        const auto acquire_step = [&](int t) {
          if (t >= steps) return;
          if (t + 1 == steps) {
            vnext = acquire();
            return;
          }
          const int v = st;
          const uint32_t pv = phase;
          if (++st == U) {
            st = 0;
            phase ^= 1;
          }
          const int k = st;
          const uint32_t pk = phase;
          if (++st == U) {
            st = 0;
            phase ^= 1;
          }
          ok = ok && TaWaitWarp2(sh, &sh->full[v], pv, &sh->full[k], pk);
          vnext = v;
          knext = k;
        };
        if (!w.turns) kunit = acquire();
        next_scores(0, 0);
        next_scores(1, 0);
        if (steps == 1 && ok) UmmaIssueCommit(&sh->q_empty);
        if (!TREE) acquire_step(0);
#pragma unroll 1
        for (int t = 0; t < steps && ok; t++) {
          if (!TREE) {
            vunit = vnext;
            kunit = knext;
            trim(blk.Index(0, t), vunit);
          } else if (!w.turns) {  // (trees, as above, lose a tenth: their units come from memory, not from the cache)
            vunit = acquire();
            trim(blk.Index(0, t), vunit);
            if (t + 1 < steps) kunit = acquire();
          }
          next_values(0, t);
          next_scores(0, t + 1);
          if (!TREE) acquire_step(t + 1);  // under the products just issued
          next_values(1, t);
          next_scores(1, t + 1);
          if (t + 2 == steps && ok) UmmaIssueCommit(&sh->q_empty);  // the last scores: Q may be replaced behind them
        }
        done0 += w.blocks0;
        done1 += w.blocks1;
      }
      UmmaIssueCommit(&sh->drained);
      __syncwarp();
      TaDrain(&sh->drained, 0);  // no product reads shared memory or TMEM after this
    }
  } else {
    if constexpr (Cfg::kWide) RegsUp<kTaRegsSoftmax>();
    // ---- softmax: thread = row of its tile = TMEM lane ----
    const int i = warp >> 2, r = threadIdx.x & 127;
    const int token = r / A.G, g = r - token * A.G;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t scol = lanes + (uint32_t)(KEYS * i), ocol = lanes + Cfg::kO + Cfg::kOStep * i;
    const float sc = A.scale_log2;
    constexpr float kBias = F16 ? 7.f : 0.f;  // probabilities up to 2^15 in fp16: 7 more bits above its smallest numbers
    bool ok = true;
    uint32_t done = 0, outs0 = 0, outs1 = 0, merges = 0;  // of the segments so far: this tile's steps, the tiles' results, merges
    uint32_t segment = 0;
    if constexpr (RANGES) w.more = 1;
    while ((segment == 0 && !RANGES) || next(segment, ok)) {
      segment++;
      const int tok0 = w.q0 + (w.turns ? 0 : i * A.TB);  // the tile's first token
      const bool mine = token < w.Tokens(i);
      const bool busy = ((warp & 3) << 5) < w.Tokens(i) * A.G;  // some row of this warp is in use
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int t = 0; t < w.Blocks(i); t++) {
        const int b = blk.Index(i, t), seen = blk.Seen(i, b);
        bool cut;  // some row does not see all keys of a whole block
        bool gone0 = false, gone1 = false;  // trees: cache pages of the block that are not there
        int page0 = 0, page1 = 0;           // read ahead of the wait, looked at behind it
        if constexpr (TREE) {
          if (b < w.cache_blocks) {
            const int* tb = A.table + (long long)w.seq * A.max_blocks + b * (KEYS / 64);
            page0 = tb[0];
            if (KEYS == 128 && seen > 64) page1 = tb[1];
          }
        }
        // A wait that gave up stops no lane here, since loads from TMEM take the whole warp: the steps run out (no wait holds any
        // more) and nothing is stored.
        ok = TaWait(sh, &sh->s_full[i], (done + t) & 1) && ok;
        TcgenFenceAfter();
        if constexpr (TREE) {
          gone0 = (unsigned)page0 >= (unsigned)A.pages;
          gone1 = (unsigned)page1 >= (unsigned)A.pages;
          cut = seen < KEYS || b >= w.cache_blocks || __any_sync(0xffffffffu, gone0 || gone1);
        } else {
          cut = tok0 < KEYS * b + KEYS - 1 || seen < KEYS;
        }
        if (!busy) {
          if (Cfg::kWide) MbarArrive(&sh->p_half[i]);
        } else {
          uint32_t s[KEYS];
          float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          const auto most = [&](int from, int to) {
#pragma unroll
            for (int c = from; c < to; c += 2)
              x[(c >> 1) & 3] = Max3(x[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
          };
          if (!cut) {
            // the maximum of one half runs under the load of the other
#pragma unroll
            for (int c = 0; c < KEYS / 64; c++) TmemLoad32(scol + 32u * c, s + 32 * c);
            TmemWaitLd();
#pragma unroll
            for (int c = KEYS / 64; c < KEYS / 32; c++) TmemLoad32(scol + 32u * c, s + 32 * c);
            most(0, KEYS / 2);
            TmemWaitLd();
            most(KEYS / 2, KEYS);
          } else {
#pragma unroll
            for (int c = 0; c < KEYS / 32; c++) {
              if (32 * c < seen) {
                TmemLoad32(scol + 32u * c, s + 32 * c);
              } else {
#pragma unroll
                for (int k = 0; k < 32; k++) s[32 * c + k] = 0;
              }
            }
            TmemWaitLd();
            // columns this row sees: 0 .. lim-1, or the bits of its mask
            unsigned long long m0, m1 = 0;
            if (TREE && b >= w.cache_blocks) {
              m0 = mine ? A.masks[w.start + tok0 + token] : 0;
              if (w.nodes < 64) m0 &= (1ull << w.nodes) - 1;
            } else {
              const int lim = TREE ? seen : min(seen, tok0 + token - KEYS * b + 1);
              m0 = lim >= 64 ? ~0ull : lim > 0 ? (1ull << lim) - 1 : 0;
              if (KEYS == 128) m1 = lim >= 128 ? ~0ull : lim > 64 ? (1ull << (lim - 64)) - 1 : 0;
              if (gone0) m0 = 0;
              if (gone1) m1 = 0;
            }
#pragma unroll
            for (int c = 0; c < KEYS / 32; c++) {
              const uint32_t bm = (uint32_t)((c < 2 ? m0 : m1) >> (32 * (c & 1)));
#pragma unroll
              for (int k = 0; k < 32; k++)
                if (!(bm >> k & 1)) s[32 * c + k] = 0xff800000u;
            }
            most(0, KEYS);
          }
          const float mx = Max3(Max3(x[0], x[1], x[2]), x[3], x[3]);
          if (t == 0) {
            m = mx;
          } else if (__any_sync(0xffffffffu, mine && !((mx - m) * sc <= kTaLazy))) {  // a NaN moves the maximum too
            // (lanes without a row hold other sequences' scores, or what shared memory held: they do not move the others' maxima,
            // or a result's last bits would hang on them)
            // step t-1's products are complete: S of step t was issued behind them
            const float mn = Max3(m, mx, mx);
            const float alpha = mn == -INFINITY ? 1.f : Exp2(Offset(mn, sc, kBias) - Offset(m, sc, kBias));
            m = mn;
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < D / 16; c++) {
              uint32_t o[16];
              TmemLoad16(ocol + 16u * c, o);
              TmemWaitLd();
#pragma unroll
              for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              TmemStore16(ocol + 16u * c, o);
            }
          }
          const float neg = m == -INFINITY ? 0.f : Offset(m, sc, kBias);
          const f32x2 sc2 = Two(sc, sc), neg2 = Two(neg, neg);
          f32x2 sum[2] = {0, 0};
          // 32 keys: the probabilities, their sum, and the 16-bit pairs into TMEM
          const auto exps = [&](int c, auto poly) {
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; k++) {
              float p0, p1;
              Split(Fma2(Two(__uint_as_float(s[32 * c + 2 * k]), __uint_as_float(s[32 * c + 2 * k + 1])), sc2, neg2), p0, p1);
              f32x2 e;
              // spread evenly: pair k where (k + 1) kPoly / 16 passes an integer
              if (decltype(poly)::value && (k + 1) * Cfg::kPoly / 16 != k * Cfg::kPoly / 16) e = Exp2Poly(p0, p1);
              else e = Two(Exp2(p0), Exp2(p1));
              sum[k & 1] = Add2(sum[k & 1], e);
              Split(e, p0, p1);
              p[k] = Pack2<F16>(p0, p1);
            }
            TmemStore16(scol + 16u * c, p);
          };
          const auto probabilities = [&](auto whole) {
            constexpr bool kAll = decltype(whole)::value;  // nothing is cut: all keys
            exps(0, whole);
            if (kAll || seen > 32) exps(1, whole);
            if constexpr (Cfg::kWide) {
              TmemWaitSt();
              TcgenFenceBefore();
              MbarArrive(&sh->p_half[i]);
              if (kAll || seen > 64) exps(2, whole);
              if (kAll || seen > 96) exps(3, whole);
            }
          };
          if (cut) probabilities(std::false_type());
          else probabilities(std::true_type());
          float l0, l1;
          Split(Add2(sum[0], sum[1]), l0, l1);
          l += l0 + l1;
          TmemWaitSt();
        }
        TcgenFenceBefore();
        MbarArrive(&sh->p_full[i]);
      }
      // ---- the rows' results ----
      done += w.Blocks(i);
      const bool merge = TREE && w.turns == kTurns && w.blocks1 > 0;
      if (w.Blocks(i) > 0) ok = TaWait(sh, &sh->o_full[i], (i ? outs1 : outs0) & 1) && ok;
      // No score above -inf: the row saw no key, or (the sum is then 1, and the row NaN) none of a weight.
      if (m == -INFINITY) {
        bool saw = !TREE && mine;
        if constexpr (TREE) {
#pragma unroll 1
          for (int t = 0; t < w.Blocks(i) && mine && !saw; t++) {
            const int b = blk.Index(i, t);
            if (b < w.cache_blocks) {
              const int* tb = A.table + (long long)w.seq * A.max_blocks + b * (KEYS / 64);
              saw = (unsigned)tb[0] < (unsigned)A.pages || (KEYS == 128 && blk.Keys(b) > 64 && (unsigned)tb[1] < (unsigned)A.pages);
            } else {
              const unsigned long long bits = A.masks[w.start + tok0 + token];
              saw = (w.nodes < 64 ? bits & ((1ull << w.nodes) - 1) : bits) != 0;
            }
          }
        }
        l = saw ? 1.f : 0.f;
      } else {
        l += Spoil<F16>(m, sc);
      }
      if (merge && i == 1) {
        // the same rows' other key blocks: tile 0's threads read this accumulator, in the same lanes, too
        sml[r] = m;
        sml[128 + r] = l;
        MbarArrive(&sh->ml_full);
        ok = TaWait(sh, &sh->ml_free, merges & 1) && ok;  // before the next segment's products may write over it
      } else if (!(w.turns == kTurns && i == 1)) {
        float a0 = 1.f, a1 = 1.f;
        if (merge) {
          ok = TaWait(sh, &sh->ml_full, merges & 1) && ok;
          ok = TaWait(sh, &sh->o_full[1], outs1 & 1) && ok;
          const float m2 = sml[r], l2 = sml[128 + r], mn = fmaxf(m, m2);
          if (mn != -INFINITY) {
            const float to = Offset(mn, sc, kBias);
            a0 = Exp2(to - Offset(m, sc, kBias));
            a1 = Exp2(to - Offset(m2, sc, kBias));
          }
          m = mn;
          l = l * a0 + l2 * a1;
        }
        if (busy) {
          TcgenFenceAfter();
          const bool parts = RANGES && w.part >= 0;
          if (!parts) {
            const float inv = m != -INFINITY ? 1.f / l : l == 0.f ? 0.f : NAN;  // nothing seen: 0
            a0 *= inv;
            a1 *= inv;
          }
          const bool zero = !parts && m == -INFINITY && l == 0.f;
          const int node = tok0 + token;
          uint16_t* out = A.out + (long long)(w.start + node) * A.out_row + (long long)((w.head + (w.turns == kHeads ? i : 0)) * A.G + g) * A.out_head;
          const long long slot = parts ? (long long)w.part * A.part_rows + (node - w.q0) * A.G + g : 0;
          // 16 columns at a time, 8 where registers are few
          constexpr int kCols = Cfg::kWide || !TREE ? 16 : 8;
          const auto columns = [](uint32_t addr, uint32_t* v) {
            if constexpr (kCols == 16) TmemLoad16(addr, v);
            else TmemLoad8(addr, v);
          };
#pragma unroll 1
          for (int c = 0; c < D; c += kCols) {
            uint32_t o[kCols], o1[kCols];
            columns(ocol + (uint32_t)c, o);
            if (merge) columns(ocol + Cfg::kOStep + (uint32_t)c, o1);
            TmemWaitLd();
            float v[kCols];
#pragma unroll
            for (int k = 0; k < kCols; k++) {
              v[k] = __uint_as_float(o[k]) * a0;
              if (merge) v[k] = fmaf(__uint_as_float(o1[k]), a1, v[k]);
              if (zero) v[k] = 0.f;
            }
            if (mine && ok) {
#pragma unroll
              for (int k = 0; k < kCols; k += 8) {
                if (parts) Store32B(A.part_o + slot * D + c + k, v + k);
                else
                  *reinterpret_cast<uint4*>(out + c + k) = make_uint4(Pack2<F16>(v[k], v[k + 1]), Pack2<F16>(v[k + 2], v[k + 3]),
                                                                      Pack2<F16>(v[k + 4], v[k + 5]), Pack2<F16>(v[k + 6], v[k + 7]));
              }
            }
          }
          if (parts && mine && ok) A.part_ml[slot] = make_float2(-Offset(m, sc, kBias), l);
        }
        if (merge) {
          TcgenFenceBefore();
          MbarArrive(&sh->ml_free);
        }
      }
      outs0 += w.blocks0 > 0;
      outs1 += w.blocks1 > 0;
      merges += merge;
    }
  }
  TcgenFenceBefore();
  __syncthreads();
  TcgenFenceAfter();
  if (warp == 8) TmemDealloc(tmem, Cfg::kCols);
}

// Joins the parts of a tree call's rows: one warp per (row, query head), D / 32 values per lane. Rows whose tile pair was not
// cut have their results already.
template <int D, bool F16>
__global__ void __launch_bounds__(256) TreeJoinKernel(const __grid_constant__ TaArgs A) {
  GridDepWait();
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)A.rows * A.H) return;
  const int row = (int)(item / A.H), h = (int)(item - (long long)row * A.H);
  if (row < A.offsets[0] || row >= A.offsets[A.n]) return;
  const int s = SequenceOf(A.offsets, A.n, row);
  const TreeSeq<TaCfg<D>::kKeys> q(A, s);
  const int node = row - q.start;
  if (node >= q.nodes) return;
  const int pair = node / (2 * A.TB), kv = h / A.G, per = A.plan[0];
  const int from = A.plan[1 + s] + (kv * q.pairs + pair) * q.blocks, c0 = from / per, c1 = (from + q.blocks - 1) / per;
  if (c0 == c1) return;
  const int local = (node - pair * 2 * A.TB) * A.G + h - kv * A.G;
  // the block of threads that begins the pair holds its part in its second place, the others in their first
  const auto slot = [&](int c) { return (long long)(2 * c + (c == c0 ? 1 : 0)) * A.part_rows + local; };
  float m = -INFINITY;
  for (int c = c0; c <= c1; c++) m = fmaxf(m, A.part_ml[slot(c)].x);
  float l = 0.f, v[D / 32] = {};
#pragma unroll 2
  for (int c = c0; c <= c1; c++) {
    const float2 ml = A.part_ml[slot(c)];
    const float a = m == -INFINITY ? 1.f : Exp2(ml.x - m);
    l = fmaf(ml.y, a, l);
    const float* o = A.part_o + slot(c) * D + lane * (D / 32);
#pragma unroll
    for (int j = 0; j < D / 32; j++) v[j] = fmaf(o[j], a, v[j]);
  }
  // a part whose maximum is NaN has a sum of NaN, which this sum takes over
  const float inv = m != -INFINITY ? 1.f / l : NAN;
  const bool zero = m == -INFINITY && l == 0.f;
  uint16_t* out = A.out + (long long)row * A.out_row + (long long)h * A.out_head + lane * (D / 32);
#pragma unroll
  for (int j = 0; j < D / 32; j++) {
    const float x = zero ? 0.f : v[j] * inv;
    out[j] = (uint16_t)Pack2<F16>(x, 0.f);
  }
}

}  // namespace shahd
