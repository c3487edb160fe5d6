// Penalties for repeated tokens, biases and grammar masks on rows of logits, before sampling.
//   x = logit of token v; c = how often v was generated, known = v is in the prompt or was generated;
//   known: x > 0 ? x / repetition : x * repetition;  x -= c frequency + [c > 0] presence;  x += bias of v;  not allowed: -inf.
// Formed in 32 bits, a rounding for each step (a quotient or product; c frequency + presence in one; their difference; the sum with the
// bias), then rounded to the result's type.
//
// Bound by memory, next to it by instructions: a row is read once and written once. A block of threads takes a slice of the tokens of a
// few rows into shared memory (asynchronous copies). While it comes, each warp looks through a part of the history and counts the tokens that
// lie in the slice in a table: whole numbers, so the order of the atomics does not matter. Where rows are on their own it puts them on a
// list of its own first; in groups it lists, behind a barrier, what its part of the table holds. Then it takes its list's counts out of the
// table, which empties it, and does what is to be done for those that it found there: of all that meet a token one. Then the rows
// go out in 16-byte pieces as the masks leave them. Rows of one sequence (drafted rows) share counts and lists. The history is read by every
// slice's block, from the cache but for the first: 4 bytes a token, four a load where it is aligned.
//
// Measured, in one graph, data from memory: 512 rows of 50257 bf16, four to a sequence of 4000 to 8000 tokens: 42 us for 108 MB, without the
// history 27: 13 blocks look through each. 256 rows of 32768 f32 with histories of 1000 to 2000: 27.1 us for 69 MB, without the history
// 19. From the cache: 40.6 and 21.3. What else was timed on the first, from the cache, where it then took 39.8: a look into the table for every value that goes
// out 54 us, the few values put right in global memory behind the copy 78, all that it met on lists 44.4, tables of 2048 or 8192
// tokens and blocks of 512 threads slower than that, all of the history in flight no faster, a cluster's blocks that share the history
// and count in one another's tables 57. 64 rows of 4096 f32: 4.0 us, latency.
#pragma once

#include "rows.cuh"

namespace shahd {

constexpr int kLogGroup = 4;     // rows of a block of threads, at most
constexpr int kLogDeep = 3;      // loads of the history of a thread in flight
constexpr int kLogTable = 3968;  // tokens of a slice's table, at most: four blocks of threads on a multiprocessor, with four 16-bit rows each
constexpr int kLogLists = 3200;  // tokens of the lists of a block's warps

struct LogitsArgs {
  const void* in;
  void* out;
  long long in_row, out_row;  // elements
  int rows, vocab, n, table, slices, group;  // table: tokens of a slice's table; group: rows of a block of threads
  const int* seqs;  // null: row r is sequence r
  const int* history;
  long long history_stride;
  const int *held, *prompt;
  const float *repetition, *presence, *frequency;
  const int *bias_offsets, *bias_tokens;
  const float* bias_values;
  int bias_entries;
  const uint32_t* masks;
  long long mask_stride;  // words
  const int* mask_rows;
  int mask_count;
};

// A piece with -inf where a token's bit is not set. Of 16-bit values a word's two bits are brought to the beginnings of its halves, and each
// times 0xffff fills its half.
template <class T>
__device__ __forceinline__ uint4 Masked(const uint4& u, uint32_t bits) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t r[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = bits >> i & 1 ? w[i] : 0xff800000u;
  } else {
    constexpr uint32_t kLow = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    const uint32_t both = (bits & 0xffu) | bits << 15;  // the odd bits, 16 above the even ones that they go with
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t keep = (both >> 2 * i & 0x10001u) * 0xffffu;
      r[i] = (w[i] & keep) | (kLow & ~keep);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Cells of a table in shared memory: 32 bits, or 16, two of which share a word that atomics work on.
template <bool WIDE>
struct LogCells {
  typedef typename std::conditional<WIDE, uint32_t, uint16_t>::type Cell;
  Cell* at;
  __device__ __forceinline__ uint32_t* Word(uint32_t t) const { return reinterpret_cast<uint32_t*>(at) + (WIDE ? t : t >> 1); }
  static __device__ __forceinline__ int Shift(uint32_t t) { return WIDE ? 0 : (t & 1) * 16; }
  __device__ __forceinline__ void Or(uint32_t t, uint32_t v) const { atomicOr(Word(t), v << Shift(t)); }
  __device__ __forceinline__ void Add(uint32_t t, uint32_t v) const { atomicAdd(Word(t), v << Shift(t)); }
  __device__ __forceinline__ void Max(uint32_t t, uint32_t v) const {
    if constexpr (WIDE) {
      atomicMax(Word(t), v);
    } else {
      uint32_t was = *Word(t);
      while ((was >> Shift(t) & 0xffffu) < v) {  // ends: the cell only grows, by this thread's value or another's
        const uint32_t seen = atomicCAS(Word(t), was, (was & ~(0xffffu << Shift(t))) | v << Shift(t));
        if (seen == was) break;
        was = seen;
      }
    }
  }
  // What a cell holds, which is 0 after that.
  __device__ __forceinline__ uint32_t Take(uint32_t t) const {
    if constexpr (WIDE) return atomicExch(Word(t), 0u);
    else return atomicAnd(Word(t), ~(0xffffu << Shift(t))) >> Shift(t) & 0xffffu;
  }
};

// Values between a 16-byte boundary and a row's beginning.
template <class T>
__device__ __forceinline__ int LeadOf(const LogitsArgs& a, int row) {
  return (int)((reinterpret_cast<uintptr_t>(a.in) + (uintptr_t)(row * a.in_row) * sizeof(T)) % 16 / sizeof(T));
}

// Threads of a block.
template <bool GROUPS>
constexpr int kLogThreadsOf = GROUPS ? 256 : 128;

// A token's count: 4 x times generated + 2 where it has a bias + 1 where the prompt has it.
template <class T, bool WIDE, bool GROUPS>
__global__ void __launch_bounds__(kLogThreadsOf<GROUPS>, 1024 / kLogThreadsOf<GROUPS>) AdjustLogitsKernel(const __grid_constant__ LogitsArgs a) {
  constexpr int kLogThreads = kLogThreadsOf<GROUPS>, kLogWarps = kLogThreads / 32, kLogList = kLogLists / kLogWarps, kCells = WIDE ? 4 : 8;
  typedef typename LogCells<WIDE>::Cell Cell;
  constexpr int PER = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t log_raw[];
  __shared__ int overflow, seqs[kLogGroup], mask_rows[kLogGroup], lead[kLogGroup];  // lead: values between a 16-byte boundary and the row's beginning
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x / a.slices * a.group, sl = blockIdx.x % a.slices, rows = min(a.group, a.rows - first);
  // Pieces begin at 16-byte boundaries, rows where they like: slices are whole pieces, and a row reaches up to PER - 1 tokens into the
  // slice before. The table begins 8 tokens ahead; rows have 8 places more at either end, so that every token of it has a place.
  const int slice = a.table - 8, base = sl * slice - 8, pitch = a.table + 8, mask_words = a.table / 32 + 2;
  const bool counts = a.history != nullptr, biases = a.bias_tokens != nullptr;
  T* const held_rows = reinterpret_cast<T*>(log_raw);                                                         // [group][pitch]
  uint32_t* const held_masks = reinterpret_cast<uint32_t*>(log_raw + (size_t)a.group * pitch * sizeof(T));    // [group][mask_words]
  const LogCells<WIDE> table{reinterpret_cast<Cell*>(held_masks + (a.group * mask_words + 3) / 4 * 4)};
  const LogCells<WIDE> entry{table.at + a.table};  // place of a token's last entry + 1
  uint16_t* const list = reinterpret_cast<uint16_t*>(entry.at + (biases ? a.table : 0)) + warp * kLogList;
  if (counts || biases)
    for (uint4* p = reinterpret_cast<uint4*>(table.at) + threadIdx.x; p < reinterpret_cast<uint4*>(entry.at + (biases ? a.table : 0)); p += kLogThreads)
      *p = make_uint4(0, 0, 0, 0);
  GridDepWait();
  GridDepLaunch();
  if (threadIdx.x == 0) overflow = 0;
  if ((int)threadIdx.x < rows) {
    seqs[threadIdx.x] = a.seqs ? a.seqs[first + threadIdx.x] : first + (int)threadIdx.x;
    mask_rows[threadIdx.x] = a.mask_rows ? a.mask_rows[first + threadIdx.x] : first + (int)threadIdx.x;
    lead[threadIdx.x] = LeadOf<T>(a, first + (int)threadIdx.x);
  }
  // The warps are dealt out to the rows: this one's row, its tokens v0 .. v1-1 of this slice, their whole pieces p0 .. p1-1 (inside the
  // row) and the values before and behind them; the warp takes every `step`-th 32 of what there is.
  const int mine = warp & (a.group - 1), begin = (warp / a.group) * 32 + lane, step = kLogThreads / a.group;
  const int mis = LeadOf<T>(a, first + min(mine, rows - 1)), v0 = max(sl * slice - mis, 0), v1 = min((sl + 1) * slice - mis, a.vocab);
  const int p0 = (v0 + mis + PER - 1) / PER, p1 = max((v1 + mis) / PER, p0), head = min(p0 * PER - mis, v1), tail = max(p1 * PER - mis, head);
  T* const held = held_rows + mine * pitch + 8 + mis - sl * slice;  // held[v]: token v
  uint32_t* const bits = held_masks + mine * mask_words;            // from the word of v0 on
  if (mine < rows) {  // also where the row will turn out to be nobody's: its values do not wait for its sequence's number
    const T* in = static_cast<const T*>(a.in) + (first + mine) * a.in_row;
    for (int c = p0 + begin; c < p1; c += step)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(SmemAddr(held + c * PER - mis)), "l"(in + c * PER - mis) : "memory");
    for (int v = v0 + begin; v < head; v += step) held[v] = in[v];
    for (int v = tail + begin; v < v1; v += step) held[v] = in[v];
  }
  __syncthreads();
  const bool busy = mine < rows && (unsigned)seqs[min(mine, rows - 1)] < (unsigned)a.n;
  const bool masked = busy && a.masks && (unsigned)mask_rows[mine] < (unsigned)a.mask_count && v0 < v1;
  if (masked) {
    const uint32_t* mask = a.masks + mask_rows[mine] * a.mask_stride + (v0 >> 5);
    const int words = ((v1 - 1) >> 5) - (v0 >> 5) + 1;
    for (int i = begin; i < words; i += step)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(SmemAddr(bits + i)), "l"(mask + i) : "memory");
  }
  for (int r = 0; (counts || biases) && r < rows;) {
    const int seq = seqs[r], from = r;
    while (r < rows && seqs[r] == seq) r++;
    if ((unsigned)seq >= (unsigned)a.n) continue;
    // ---- the tokens that there are: the table is empty ----
    int listed = 0;  // on the warp's list
    const unsigned below = (1u << lane) - 1;
    // All lanes: N tokens each are put on the list, those with a place in the table; false where they have not all room there.
    const auto enlist = [&](auto n, const uint32_t* t, const uint32_t* flag) {
      constexpr int N = decltype(n)::value;
      unsigned who[N];
      int all = 0;
#pragma unroll
      for (int j = 0; j < N; j++) {
        who[j] = __ballot_sync(0xffffffffu, t[j] < (uint32_t)a.table);
        all += __popc(who[j]);
      }
      if (listed + all > kLogList) return false;
#pragma unroll
      for (int j = 0; j < N; j++) {
        if (t[j] < (uint32_t)a.table) list[listed + __popc(who[j] & below)] = (uint16_t)(t[j] | flag[j]);
        listed += __popc(who[j]);
      }
      return true;
    };
    int b0 = 0;
    if (biases) {
      b0 = min(max(a.bias_offsets[seq], 0), a.bias_entries);
      const int count = min(max(a.bias_offsets[seq + 1], b0), a.bias_entries) - b0;
      for (int i0 = warp * 32; i0 < count; i0 += kLogThreads) {
        const int i = i0 + lane;
        // in unsigned numbers, which wrap: any value may stand there
        const uint32_t t = i < count ? (uint32_t)a.bias_tokens[b0 + i] - (uint32_t)base : 0xffffffffu;
        if (t < (uint32_t)a.table) {
          entry.Max(t, (uint32_t)i + 1u);
          table.Or(t, 2);
        }
        const uint32_t none = 0;
        if (!GROUPS && !enlist(std::integral_constant<int, 1>(), &t, &none)) overflow = 1;
      }
    }
    const int biased = listed;
    float rep = 1.f, freq = 0.f, pres = 0.f;
    double inv = 1.0;
    if (counts) {
      const int* h = a.history + seq * a.history_stride;
      const int length = (int)min((long long)max(a.held[seq], 0), a.history_stride), prompt = a.prompt ? a.prompt[seq] : 0;
      rep = a.repetition ? a.repetition[seq] : 1.f;
      freq = a.frequency ? a.frequency[seq] : 0.f;
      pres = a.presence ? a.presence[seq] : 0.f;
      const auto count = [&](uint32_t t, bool of_prompt) {
        if (of_prompt) table.Or(t, 1);
        else table.Add(t, 4);
      };
      constexpr uint32_t kPrompt = 0x8000u;
      // four tokens a lane, from place i[j] of the history each (INT32_MIN is no token of any table)
      const auto meet = [&](const int (&token)[4], const int (&i)[4]) {
        if constexpr (GROUPS) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t at = (uint32_t)token[j] - (uint32_t)base;
            if (at < (uint32_t)a.table) count(at, i[j] < prompt);
          }
        } else {
          uint32_t t[4], flag[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            t[j] = (uint32_t)token[j] - (uint32_t)base;
            flag[j] = i[j] < prompt ? kPrompt : 0u;
          }
          if (enlist(std::integral_constant<int, 4>(), t, flag)) return;
          overflow = 1;
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (t[j] < (uint32_t)a.table) count(t[j], flag[j] != 0);
        }
      };
      const int fours = reinterpret_cast<uintptr_t>(h) % 16 == 0 ? length / 4 : 0;
#pragma unroll 1
      for (int i0 = warp * 32; i0 < fours; i0 += kLogDeep * kLogThreads) {
        int4 u[kLogDeep];
#pragma unroll
        for (int k = 0; k < kLogDeep; k++) {
          const int i = i0 + k * kLogThreads + lane;
          u[k] = i < fours ? reinterpret_cast<const int4*>(h)[i] : make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
        }
#pragma unroll
        for (int k = 0; k < kLogDeep; k++) {
          if (i0 + k * kLogThreads >= fours) break;
          const int i = 4 * (i0 + k * kLogThreads + lane);
          meet({u[k].x, u[k].y, u[k].z, u[k].w}, {i, i + 1, i + 2, i + 3});
        }
      }
#pragma unroll 1
      for (int i0 = 4 * fours + warp * 32; i0 < length; i0 += 4 * kLogThreads) {
        int u[4], i[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          i[k] = i0 + k * kLogThreads + lane;
          u[k] = i[k] < length ? h[i[k]] : INT32_MIN;
        }
        meet(u, i);
      }
      __syncwarp();
      for (int i = biased + lane; i < listed; i += 32)  // none in groups
        count(list[i] & ~kPrompt, list[i] & kPrompt);
      // The quotient by a product in 64 bits, off by 2^-52 of itself: as x / rep rounds it, since a quotient of 24-bit numbers is a border between two
      // 32-bit values, which only one below 2^-126 can be and which then goes to either side, or 2^-49 of itself away from one. (A product in 32 bits is rounded twice, and inf for a rep below 2^-128. The drafted rows, from the
      // cache: 40.4 us, with it 39.4, with a division for each token 42.4; the 64 rows of 4096: 3.9, 3.9 and 4.3.)
      inv = 1.0 / (double)rep;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const auto adjust = [&](int t, uint32_t w) {
      uint32_t e = 0;
      if (w & 2) {
        e = entry.at[t];
        entry.at[t] = 0;
      }
      const float bias = e != 0 ? a.bias_values[b0 + (int)e - 1] : 0.f, fine = w > 3 ? fmaf((float)(w >> 2), freq, pres) : 0.f;
      for (int k = from; k < r; k++) {
        T* at = held_rows + k * pitch + lead[k] + t;
        float x = ToFloat(*at);
        if (w & ~2u) x = x > 0.f ? (float)((double)x * inv) : x * rep;
        if (w > 3) x -= fine;
        if (e != 0) x += bias;
        *at = FromFloat<T>(x);
      }
    };
    const auto see_to = [&] {
      for (int i = lane; i < listed; i += 32) {
        const int t = list[i] & 0x7fff;
        const uint32_t w = table.Take(t);
        if (w != 0) adjust(t, w);
      }
    };
    if constexpr (GROUPS) {
      // each warp lists the tokens of its part of the table: one for a lane at a time
      for (int c0 = warp * 32; c0 < a.table / kCells; c0 += kLogThreads) {
        const int c = c0 + lane;
        const uint4 u = c < a.table / kCells ? reinterpret_cast<const uint4*>(table.at)[c] : make_uint4(0, 0, 0, 0);
        const uint32_t words[4] = {u.x, u.y, u.z, u.w};
        uint32_t there = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (WIDE) there |= (uint32_t)(words[i] != 0) << i;
          else there |= (uint32_t)((words[i] & 0xffffu) != 0) << 2 * i | (uint32_t)(words[i] > 0xffffu) << (2 * i + 1);
        }
        int upto = __popc(there);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const int all = __shfl_sync(0xffffffffu, upto, 31);
        if (listed + all > kLogList) {
          __syncwarp();
          see_to();
          __syncwarp();
          listed = 0;
        }
        for (uint16_t* p = list + listed + upto - __popc(there); there != 0; there &= there - 1) *p++ = (uint16_t)(c * kCells + __ffs(there) - 1);
        listed += all;
      }
      __syncwarp();
    }
    see_to();
    if (!GROUPS && overflow) {  // some token is on no list
      __syncthreads();
      for (int t = threadIdx.x; t < a.table; t += kLogThreads)
        if (table.at[t] != 0) adjust(t, table.at[t]);
      __syncthreads();
      for (int t = threadIdx.x; t < a.table; t += kLogThreads) table.at[t] = 0;
      if (threadIdx.x == 0) overflow = 0;
    }
    if (r < rows) __syncthreads();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (!busy) return;
  T* out = static_cast<T*>(a.out) + (first + mine) * a.out_row;
  const int word0 = v0 >> 5;
  const bool alike = (int)(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T)) == mis;
  const int last = alike ? p1 : p0;
  for (int c = p0 + begin; c < last; c += step) {
    const int v = c * PER - mis;
    uint4 u = *reinterpret_cast<const uint4*>(held + v);
    if (masked) {
      u = Masked<T>(u, __funnelshift_r(bits[(v >> 5) - word0], bits[((v + PER - 1) >> 5) - word0], v & 31));
    }
    *reinterpret_cast<uint4*>(out + v) = u;
  }
  const auto single = [&](int v) { out[v] = !masked || (bits[(v >> 5) - word0] >> (v & 31) & 1) ? held[v] : FromFloat<T>(-INFINITY); };
  for (int v = v0 + begin; v < (alike ? head : v1); v += step) single(v);
  if (alike)
    for (int v = tail + begin; v < v1; v += step) single(v);
}

// Rows on their own: blocks of 128 threads, twice as many at a time, so that the steps of one run under the copies of others, and each
// warp lists the history's tokens that it met, since a row meets few (256 rows of 32768 f32, all from the cache: 20.9 us; with 256 threads 24.3; looking for them
// in the table 25.5). Groups: 256 threads, since four rows take the shared memory (512 rows of 50257 bf16: with 128 60 us), and
// the tokens are looked for in the table, which costs a lane less than a list of all that it met (39.8 us, with such lists 44.4). All before the quotient by
// a product in 64 bits, which costs 0.4 to 1.0.
template <class T, bool WIDE, bool GROUPS>
void LaunchLogitsAs(const LogitsArgs& a, int smem, cudaStream_t st) {
  if (!EnsureKernelAttrs((const void*)AdjustLogitsKernel<T, WIDE, GROUPS>, smem)) return;
  LaunchPdl(AdjustLogitsKernel<T, WIDE, GROUPS>, dim3((unsigned)(CeilDiv(a.rows, a.group) * a.slices)), dim3(kLogThreadsOf<GROUPS>), (size_t)smem, st, a);
}

template <class T>
void LaunchLogits(const LogitsArgs& a, bool wide, int smem, cudaStream_t st) {
  if (a.group > 1) wide ? LaunchLogitsAs<T, true, true>(a, smem, st) : LaunchLogitsAs<T, false, true>(a, smem, st);
  else wide ? LaunchLogitsAs<T, true, false>(a, smem, st) : LaunchLogitsAs<T, false, false>(a, smem, st);
}

// Whether some row of `out` shares bytes with some row of `in` (rows of `width` bytes, `in_row` and `out_row` apart, no row across the next one's
// beginning). Rows that lie in the gaps of the others do not: two halves of one buffer.
inline bool RowsOverlap(const void* in, const void* out, long long rows, long long width, long long in_row, long long out_row) {
  const long long a = reinterpret_cast<long long>(in), b = reinterpret_cast<long long>(out);
  if (b >= a + (rows - 1) * in_row + width || a >= b + (rows - 1) * out_row + width) return false;
  // row i of `in` begins `ahead` bytes behind a row of `out`, and that many less than out_row before the next one
  const long long look = in_row == out_row ? 1 : rows;  // the same for all of them
  for (long long i = 0; i < look; i++) {
    const long long apart = a + i * in_row - b, row = apart >= 0 ? apart / out_row : -((-apart + out_row - 1) / out_row), ahead = apart - row * out_row;
    // with one stride, row i of `in` meets rows i + row and i + row + 1: some i has them as long as they are less than `rows` off
    const long long least = in_row == out_row ? 1 - rows : 0;
    if ((row >= least && row < rows && ahead < width) || (row + 1 >= least && row + 1 < rows && out_row - ahead < width)) return true;
  }
  return false;
}

}  // namespace shahd

extern "C" {

int shahd_adjust_logits(const ShahdLogitsCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_adjust_logits";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  if (!CheckType(op, c->dtype, true)) return SHAHD_EINVAL;
  if (c->rows < 0 || c->n < 0 || c->vocab < 1 || c->vocab > (1 << 24) || c->rows > (1 << 20) || c->n > (1 << 20)) {
    SetError("%s: need rows and n in 0 .. 2^20 and 1 <= vocab <= 2^24 (got rows=%d n=%d vocab=%d)", op, c->rows, c->n, c->vocab);
    return SHAHD_EINVAL;
  }
  if (!c->sequences && c->rows > c->n) {
    SetError("%s: without sequences there is a row for each of them (got rows=%d n=%d)", op, c->rows, c->n);
    return SHAHD_EINVAL;
  }
  if (c->logits_stride < c->vocab || c->out_stride < c->vocab || c->logits_stride > (1LL << 36) || c->out_stride > (1LL << 36)) {
    SetError("%s: need strides of at least vocab %d elements, below 2^36 (got %lld and %lld)", op, c->vocab, (long long)c->logits_stride, (long long)c->out_stride);
    return SHAHD_EINVAL;
  }
  if (c->logits == c->out && c->logits_stride != c->out_stride) {
    SetError("%s: logits adjusted in place have one stride (got %lld and %lld)", op, (long long)c->logits_stride, (long long)c->out_stride);
    return SHAHD_EINVAL;
  }
  if (c->history ? c->history_stride < 0 || c->history_stride >= (1 << 30) || !c->history_lengths
                 : c->history_lengths || c->prompt_lengths || c->repetition || c->presence || c->frequency) {
    SetError("%s: a history goes with history_lengths and a stride in 0 .. 2^30 - 1, and penalties with a history (got stride %lld)", op, (long long)c->history_stride);
    return SHAHD_EINVAL;
  }
  if (c->bias_tokens ? !c->bias_offsets || !c->bias_values || c->bias_entries < 0 : c->bias_offsets || c->bias_values || c->bias_entries != 0) {
    SetError("%s: bias_offsets, bias_tokens, bias_values and bias_entries >= 0 go together (got bias_entries=%d)", op, c->bias_entries);
    return SHAHD_EINVAL;
  }
  if (c->masks ? c->mask_count < 0 || c->mask_stride < (c->vocab + 31) / 32 || c->mask_stride > (1LL << 32) : c->mask_rows || c->mask_count != 0) {
    SetError("%s: masks need mask_count >= 0 and a stride of at least %d words (got %d and %lld)", op, (c->vocab + 31) / 32, c->mask_count, (long long)c->mask_stride);
    return SHAHD_EINVAL;
  }
  if (c->rows == 0 || c->n == 0) return SHAHD_OK;
  const size_t size = TypeBytes(c->dtype);
  if (c->logits != c->out && RowsOverlap(c->logits, c->out, c->rows, (long long)c->vocab * size, c->logits_stride * size, c->out_stride * size)) {
    SetError("%s: logits and out overlap; they may be one", op);
    return SHAHD_EINVAL;
  }
  BufferCheck b(op);
  b.Add("logits", c->logits, size);
  if (c->out != c->logits) b.Add("out", c->out, size);
  const struct {
    const char* name;
    const void* p;
  } more[] = {{"sequences", c->sequences}, {"history", c->history}, {"history_lengths", c->history_lengths}, {"prompt_lengths", c->prompt_lengths},
              {"repetition", c->repetition}, {"presence", c->presence}, {"frequency", c->frequency}, {"bias_offsets", c->bias_offsets},
              {"bias_tokens", c->bias_tokens}, {"bias_values", c->bias_values}, {"masks", c->masks}, {"mask_rows", c->mask_rows}};
  for (const auto& m : more)
    if (m.p) b.Add(m.name, m.p, 4);
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  LogitsArgs a = {};
  a.in = c->logits;
  a.out = c->out;
  a.in_row = c->logits_stride;
  a.out_row = c->out_stride;
  a.rows = c->rows;
  a.vocab = c->vocab;
  a.n = c->n;
  a.seqs = c->sequences;
  a.history = c->history;
  a.history_stride = c->history_stride;
  a.held = c->history_lengths;
  a.prompt = c->prompt_lengths;
  a.repetition = c->repetition;
  a.presence = c->presence;
  a.frequency = c->frequency;
  a.bias_offsets = c->bias_offsets;
  a.bias_tokens = c->bias_tokens;
  a.bias_values = c->bias_values;
  a.bias_entries = c->bias_entries;
  a.masks = c->masks;
  a.mask_stride = c->mask_stride;
  a.mask_rows = c->mask_rows;
  a.mask_count = c->mask_count;
  // Slices of whole pieces and of one size, as many as give every multiprocessor a few blocks of threads, a thousand tokens at least; rows in
  // groups where they share sequences and enough are left. (A row that does not begin at a boundary reaches up to 7 values further.)
  const int reach = c->vocab + 7, wanted = std::max(CeilDiv(reach, kLogTable - 8), std::min(CeilDiv(4 * info.sms, c->rows), CeilDiv(reach, 1016)));
  const int slice = RoundUp(CeilDiv(reach, wanted), 8);
  a.table = slice + 8;
  a.slices = CeilDiv(reach, slice);
  a.group = 1;
  while (c->rows / c->n >= 2 * a.group && a.group < kLogGroup && (long long)c->rows / (2 * a.group) * a.slices >= 4 * info.sms) a.group *= 2;
  if ((long long)a.rows * a.slices > 0x7fffffffLL) {
    SetError("%s: too many rows of this vocabulary: %d of %d", op, c->rows, c->vocab);
    return SHAHD_EINVAL;
  }
  const bool wide = (a.history && a.history_stride > 0x3fff) || a.bias_entries > 0xfffe;  // a cell of 16 bits holds 4 x 2^14 - 1, and 2^16 - 1
  // rows, masks, counts, entries, lists
  const int smem = a.group * (a.table + 8) * (int)size + RoundUp(a.group * (a.table / 32 + 2), 4) * 4 +
                   (a.history || a.bias_tokens ? a.table * (a.bias_tokens ? 2 : 1) * (wide ? 4 : 2) + kLogLists * 2 : 0);
  TakeLaunchError(nullptr);
  if (c->dtype == SHAHD_F32) LaunchLogits<float>(a, wide, smem, static_cast<cudaStream_t>(stream));
  else if (c->dtype == SHAHD_F16) LaunchLogits<__half>(a, wide, smem, static_cast<cudaStream_t>(stream));
  else LaunchLogits<bf16>(a, wide, smem, static_cast<cudaStream_t>(stream));
  return LaunchStatus(op);
}

}  // extern "C"
