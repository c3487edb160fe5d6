// Verification of drafted token trees against the target's probabilities, with given random numbers: the rule of
// SpeculativeSample (Brain/Reasoning/SpeculativeSampling.ts:82-112) for trees, many sequences at once, decided on the
// device from probabilities that lie there.
//
// A sequence's walk starts at its root (node 0) with p the target's and q the draft's row of the current node. The
// children of the current node, in index order, are candidates drawn from q:
//   candidate x is taken with probability min(1, p_k(x) / q(x)) where p_0 = p and, after the k-th refusal,
//   p_k = max(0, p_{k-1} - q) / its sum;
// a taken child becomes the current node, and when no candidate is left the next token is drawn from p_k.
// Unrolled, p_k = max(0, p - a_k q) / Z_k with a_0 = 0, Z_0 = 1, a_{k+1} = a_k + Z_k and Z_k = sum max(0, p - a_k q):
// a refusal costs one pass over the two rows and no row is written. The test u q(x) Z < max(0, p(x) - a q(x)) is formed in 64
// bits from the rows' own values. In a pass, max(0, p - a q) of one token is two fused 32-bit steps (a as the sum of two
// floats; each rounds relative to its own result: off by 2^-23 of itself, or, where the second step cancels what the first has left,
// by less than 2^-47 a q), a 16-byte piece's tokens are added in 32 bits and the pieces in 64, in a fixed order: a running mass is good to about 2^-23 over the root of the
// number of pieces, 10^-9 in a row of 32768, and a run repeats bit for bit. (Element by element in 64 bits the conversions
// alone, 16 a clock, took twice as long as the rows from memory, and the registers left one block per multiprocessor: 64
// trees over 32768 tokens 30 us, 128 over 50257 in bf16 61 us; now 15.5 and 26.)
//
// Bound by latency: a walk is a chain of decisions. What the decisions read, p and q at each node's token in its parent's
// rows, does not hang on the walk, so a block's threads fetch it for 256 nodes at once into shared memory, and the walk
// itself reads memory only for refusals. A row is cut over the blocks of a cluster, which exchange 8 bytes per warp through
// distributed shared memory: one cluster barrier per refusal.
#pragma once

#include "ops_common.cuh"

namespace shahd {

constexpr int kVerThreads = 256;
constexpr int kVerPerSm = 4;  // blocks that fit a multiprocessor
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerMaxCluster = 8;

struct VerifyArgs {
  const void *target, *draft;
  long long target_row, draft_row;  // elements
  const int *tokens, *parents, *offsets;
  const float* uniforms;
  const int* lengths;
  int *path, *count, *next, *commit, *new_lengths;
  int n, rows, vocab, cluster;
};

template <class T>
__device__ __forceinline__ double Prob(T x) {
  const float f = float(x);
  return f > 0.f ? (double)f : 0.0;  // NaN and negative values are no mass
}

// max(0, p - a q): what is left of token v after refusals of weight a.
__device__ __forceinline__ double Left(double p, double q, double a) { return fmax(0.0, fma(-a, q, p)); }

__device__ __forceinline__ void StoreCluster(double* p, uint32_t rank, double v) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(SmemAddr(p)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(ra), "d"(v) : "memory");
}

// The same in 32 bits with a = hi + lo.
__device__ __forceinline__ float Left32(float p, float q, float hi, float lo) {
  p = fmaxf(p, 0.f);  // NaN and negative values are no mass
  q = fmaxf(q, 0.f);
  return fmaxf(fmaf(-lo, q, fmaf(-hi, q, p)), 0.f);
}

template <class T>
struct VerifyRows {
  static constexpr int PER = 16 / sizeof(T);  // values of a 16-byte piece
  const T *p, *q;
  int V, mis;       // mis: values between the start of value 0's piece and value 0
  int first, last;  // this warp's pieces
  int whole0, whole1;  // pieces that lie inside both rows and can be read as such (none where the rows lie unlike to each other)
  __device__ __forceinline__ int Value(int piece, int i) const { return piece * PER + i - mis; }
  // max(0, p - (hi + lo) q) of a whole piece from its 16-byte words, and of any piece value by value (0 outside the row).
  __device__ __forceinline__ void Whole(const uint4& u, const uint4& w, float hi, float lo, float (&x)[PER]) const {
    const T* h = reinterpret_cast<const T*>(&u);
    const T* g = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = Left32(float(h[i]), float(g[i]), hi, lo);
  }
  __device__ __forceinline__ void Any(int piece, float hi, float lo, float (&x)[PER]) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int v = Value(piece, i);
      x[i] = v >= 0 && v < V ? Left32(float(p[v]), hi != 0.f ? float(q[v]) : 0.f, hi, lo) : 0.f;
    }
  }
  static __device__ __forceinline__ double Sum(const float (&x)[PER]) {
    float s[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] = x[i];
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; i++) s[i] += s[i + o];
    return (double)s[0];
  }
};

template <class T>
__global__ void __launch_bounds__(kVerThreads, kVerPerSm) VerifyTreeKernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double sums[2][kVerMaxCluster * kVerWarps];  // every warp's sum of the latest passes, by turns
  __shared__ double s_p[kVerThreads], s_q[kVerThreads];
  __shared__ float s_u[kVerThreads];
  __shared__ int s_parent[kVerThreads];
  GridDepWait();
  GridDepLaunch();
  const int C = a.cluster, rank = blockIdx.x % C, sq = blockIdx.x / C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = min(max(a.offsets[sq], 0), a.rows), e = min(max(a.offsets[sq + 1], b), a.rows), N = e - b;
  const int len = a.lengths ? a.lengths[sq] : 0;
  if (rank == 0) {
    for (int i = b + threadIdx.x; i < e; i += kVerThreads) {
      a.path[i] = -1;
      if (a.commit) a.commit[i] = -1;
    }
  }
  if (N == 0) {  // the whole cluster leaves together
    if (rank == 0 && threadIdx.x == 0) {
      a.count[sq] = 0;
      a.next[sq] = -1;
      if (a.new_lengths) a.new_lengths[sq] = len;
    }
    return;
  }
  if (C > 1) ClusterSync();  // every block of the cluster runs before any writes to another's shared memory
  const T* target = static_cast<const T*>(a.target);
  const T* draft = static_cast<const T*>(a.draft);

  VerifyRows<T> rows;
  rows.V = a.vocab;
  const auto enter = [&](int node) {  // the rows of a node, cut into pieces over the cluster's warps in index order
    rows.p = target + (long long)(b + node) * a.target_row;
    rows.q = draft + (long long)(b + node) * a.draft_row;
    const int mp = (int)(reinterpret_cast<uintptr_t>(rows.p) % 16 / sizeof(T)), mq = (int)(reinterpret_cast<uintptr_t>(rows.q) % 16 / sizeof(T));
    rows.mis = mp == mq ? mp : 0;
    const int pieces = (rows.V + rows.mis + rows.PER - 1) / rows.PER;
    const int share = CeilDiv(pieces, C * kVerWarps);
    rows.first = min(pieces, (rank * kVerWarps + warp) * share);
    rows.last = min(pieces, rows.first + share);
    rows.whole0 = min(max(rows.first, rows.mis > 0 ? 1 : 0), rows.last);
    rows.whole1 = mp == mq ? min(max(rows.whole0, (rows.V + rows.mis) / rows.PER), rows.last) : rows.whole0;
  };
  int buf = 0;
  // of the latest pass: the mass ahead of this warp's pieces, up to their end, in them, in the whole row
  double before = 0, after = 0, mine = 0, total = 0;
  const auto pass = [&](double w) {        // Z = sum of max(0, p - w q)
    double z = 0;
    const float hi = (float)w, lo = (float)(w - (double)hi);
    float x[VerifyRows<T>::PER];
    const uint4* vp = reinterpret_cast<const uint4*>(rows.p - rows.mis);
    const uint4* vq = reinterpret_cast<const uint4*>(rows.q - rows.mis);
    // Four pieces of each row in flight. By ordinary loads: the rows are the kernel's before this one to write, and with programmatic
    // launches this kernel may have begun by then, which loads through the read-only path do not allow for.
    for (int c = rows.whole0 + lane; c < rows.whole1; c += 128) {
      uint4 u[4], v[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const bool in = c + 32 * k < rows.whole1;
        u[k] = in ? vp[c + 32 * k] : make_uint4(0, 0, 0, 0);
        v[k] = in && w != 0 ? vq[c + 32 * k] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        rows.Whole(u[k], v[k], hi, lo, x);
        z += rows.Sum(x);
      }
    }
    for (int c = rows.first + lane; c < rows.last; c += 32) {
      if (c >= rows.whole0 && c < rows.whole1) continue;
      rows.Any(c, hi, lo, x);
      z += rows.Sum(x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (C == 1) {
      if (lane == 0) sums[buf][warp] = z;
      __syncthreads();
    } else {
      if (lane < C) StoreCluster(&sums[buf][rank * kVerWarps + warp], lane, z);
      ClusterSync();
    }
    // Every warp adds the same sums in the same order, block by block: `after` of a warp is `before` of the next to the
    // last bit, and equal to its own `before` where it holds no mass, so exactly one warp holds the draw's goal.
    double t = 0, in0 = 0, in1 = 0;
    if (lane < C) {
      for (int i = 0; i < kVerWarps; i++) {
        if (i == warp) in0 = t;
        t += sums[buf][lane * kVerWarps + i];
        if (i == warp) in1 = t;
      }
    }
    double base = 0;
    total = 0;
    for (int c = 0; c < C; c++) {
      if (c == rank) base = total;
      total += __shfl_sync(0xffffffffu, t, c);
    }
    before = base + __shfl_sync(0xffffffffu, in0, rank);
    after = base + __shfl_sync(0xffffffffu, in1, rank);
    mine = z;
    buf ^= 1;  // the other half was last read before the barrier above
  };

  int cur = 0, depth = 0, window = 0;
  double w = 0, z = 1;
  bool passed = false;  // the latest pass is of the current node and weight
  enter(0);
  if (rank == 0 && threadIdx.x == 0) a.path[b] = 0;  // thread 0 filled this place itself
  int at = 1;  // first node not asked yet
  for (int loaded = -1; at < N;) {
    if (window != loaded) {  // what the decisions on nodes window .. window + 255 read
      __syncthreads();
      const int j = window + threadIdx.x;
      int parent = -1;
      if (j < N) {
        parent = a.parents[b + j];
        const int tok = a.tokens[b + j];
        if (parent < 0 || parent >= j || tok < 0 || tok >= a.vocab) parent = -1;  // no node's child
        if (parent >= 0) {
          s_p[threadIdx.x] = Prob(target[(long long)(b + parent) * a.target_row + tok]);
          s_q[threadIdx.x] = Prob(draft[(long long)(b + parent) * a.draft_row + tok]);
          s_u[threadIdx.x] = a.uniforms[b + j];
        }
      }
      s_parent[threadIdx.x] = parent;
      loaded = window;
      __syncthreads();
    }
    // the next child of the current node in this window (all warps find the same)
    int child = -1;
    for (int k = (at - window) & ~31; k < kVerThreads && window + k < N; k += 32) {
      const unsigned hit = __ballot_sync(0xffffffffu, window + k + lane >= at && s_parent[k + lane] == cur);
      if (hit) {
        child = k + __ffs(hit) - 1;
        break;
      }
    }
    if (child < 0) {
      window += kVerThreads;
      at = window;
      continue;
    }
    at = window + child + 1;
    const double p = s_p[child], q = s_q[child];
    if ((double)s_u[child] * q * z < Left(p, q, w)) {
      cur = window + child;
      depth++;
      w = 0;
      z = 1;
      passed = false;
      enter(cur);
      if (rank == 0 && threadIdx.x == 0) {
        a.path[b + depth] = cur;
        if (a.commit) a.commit[b + cur] = len + depth;
      }
    } else if (z > 0) {
      w += z;
      pass(w);
      z = total;
      passed = true;
    }
  }
  if (!(z > 0)) {  // nothing is left: the target's own row
    w = 0;
    passed = false;
  }
  if (!passed) pass(w);
  // the first token whose running mass reaches u * total; the root's number is the draw's
  const float uf = a.uniforms[b];
  const double goal = (uf > 0.f ? fmin((double)uf, 1.0) : 0.0) * total;
  const bool mass = total > 0 && isfinite(total);
  if (mass && mine > 0 && after >= goal && (before < goal || before == 0)) {
    int id = -1, seen = -1;
    double run = before;
    const float hi = (float)w, lo = (float)(w - (double)hi);
    for (int c0 = rows.first; c0 < rows.last && id < 0; c0 += 32) {
      const int c = c0 + lane;
      float x[VerifyRows<T>::PER];
      double own = 0;
#pragma unroll
      for (int i = 0; i < VerifyRows<T>::PER; i++) x[i] = 0.f;
      if (c < rows.last) rows.Any(c, hi, lo, x);
#pragma unroll
      for (int i = 0; i < VerifyRows<T>::PER; i++) own += (double)x[i];
      double incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      int found = -1, last = -1;
      double s = run + incl - own;
#pragma unroll
      for (int i = 0; i < VerifyRows<T>::PER; i++) {
        s += (double)x[i];
        if (x[i] > 0.f) last = rows.Value(c, i);
        if (x[i] > 0.f && s >= goal && found < 0) found = rows.Value(c, i);
      }
      const unsigned hit = __ballot_sync(0xffffffffu, found >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
      if (any) seen = __shfl_sync(0xffffffffu, last, 31 - __clz(any));
      if (hit) id = __shfl_sync(0xffffffffu, found, __ffs(hit) - 1);
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) a.next[sq] = id >= 0 ? id : seen;  // the scan's own rounding can end just below the goal
  }
  if (rank == 0 && threadIdx.x == 0) {
    if (!mass) a.next[sq] = 0;  // a row without mass, as SampleFromDistribution answers, or with an endless one
    a.count[sq] = depth;
    if (a.commit) a.commit[b] = len;
    if (a.new_lengths) a.new_lengths[sq] = len + depth + 1;
  }
  if (C > 1) ClusterSync();  // no block leaves while another may still write its sums
}

}  // namespace shahd

extern "C" int shahd_verify_tree(const ShahdVerifyCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_verify_tree";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  if (!CheckType(op, c->dtype, true)) return SHAHD_EINVAL;
  if (c->n < 0 || c->rows < 0 || c->vocab < 1 || c->vocab > (1 << 30) || c->target_stride < c->vocab || c->draft_stride < c->vocab ||
      c->target_stride > (1LL << 36) || c->draft_stride > (1LL << 36)) {
    SetError("%s: need n, rows >= 0, 1 <= vocab <= 2^30 and row strides of at least vocab (got n=%d rows=%d vocab=%d "
             "target_stride=%lld draft_stride=%lld)",
             op, c->n, c->rows, c->vocab, (long long)c->target_stride, (long long)c->draft_stride);
    return SHAHD_EINVAL;
  }
  if (c->rows > kOpsMaxRows || c->n > kOpsMaxRows) {
    SetError("%s: too many rows or sequences: %d and %d, at most 2^30", op, c->rows, c->n);
    return SHAHD_EINVAL;
  }
  if (c->n == 0) return SHAHD_OK;
  if ((c->commit || c->new_lengths) && !c->lengths) {
    SetError("%s: commit and new_lengths need lengths", op);
    return SHAHD_EINVAL;
  }
  const size_t size = TypeBytes(c->dtype);
  BufferCheck b(op);
  b.Add("offsets", c->offsets, 4);
  if (c->rows > 0) {
    b.Add("target", c->target, size);
    b.Add("draft", c->draft, size);
    b.Add("tokens", c->tokens, 4);
    b.Add("parents", c->parents, 4);
    b.Add("uniforms", c->uniforms, 4);
    b.Add("path", c->path, 4);
    if (c->commit) b.Add("commit", c->commit, 4);
  }
  b.Add("count", c->count, 4);
  b.Add("next_ids", c->next_ids, 4);
  if (c->lengths) b.Add("lengths", c->lengths, 4);
  if (c->new_lengths) b.Add("new_lengths", c->new_lengths, 4);
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  VerifyArgs a = {};
  a.target = c->target;
  a.draft = c->draft;
  a.target_row = c->target_stride;
  a.draft_row = c->draft_stride;
  a.tokens = c->tokens;
  a.parents = c->parents;
  a.offsets = c->offsets;
  a.uniforms = c->uniforms;
  a.lengths = c->lengths;
  a.path = c->path;
  a.count = c->count;
  a.next = c->next_ids;
  a.commit = c->commit;
  a.new_lengths = c->new_lengths;
  a.n = c->n;
  a.rows = c->rows;
  a.vocab = c->vocab;
  // A row is cut over as many blocks as leave each thread a 16-byte piece of it, as long as all blocks run at once: a pass is
  // then a few rounds of loads.
  const long long pieces = ((long long)c->vocab * (long long)size + 15) / 16;
  a.cluster = 1;
  while (a.cluster < kVerMaxCluster && pieces >= 2LL * a.cluster * kVerThreads && 2LL * a.cluster * c->n <= (long long)kVerPerSm * info.sms) a.cluster *= 2;
  if ((long long)c->n * a.cluster > 0x7fffffffLL) a.cluster = 1;
  TakeLaunchError(nullptr);
  const dim3 grid((unsigned)(c->n * a.cluster)), block(kVerThreads), cluster((unsigned)a.cluster);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c->dtype == SHAHD_F32) LaunchPdlCluster(VerifyTreeKernel<float>, grid, block, 0, cluster, st, a);
  else if (c->dtype == SHAHD_F16) LaunchPdlCluster(VerifyTreeKernel<__half>, grid, block, 0, cluster, st, a);
  else LaunchPdlCluster(VerifyTreeKernel<bf16>, grid, block, 0, cluster, st, a);
  return LaunchStatus(op);
}
