// Penalties for repeated tokens, biases and grammar masks on rows of logits, before sampling.
//   x = logit of token v; c = how often v was generated, known = v is in the prompt or was generated;
//   known: x > 0 ? x / repetition : x * repetition;  x -= c frequency + [c > 0] presence;  x += bias of v;  not allowed: -inf.
// Formed in 32 bits, rounded once.
//
// Bound by memory: a row is read once and written once. A block of threads takes a slice of the tokens of a few rows into shared memory
// (asynchronous copies), and while it comes counts the history's tokens of the slice there: whole numbers, so the order of the atomics
// does not matter. Few tokens of a vocabulary are in a history or a list of biases: each warp looks through a part of the counts, makes a
// list of those that are, and does what is to be done for its list; then the rows go out in 16-byte pieces as the masks leave them.
// Rows of one sequence (drafted rows) share counts and lists. The history is read by every slice's block, from the cache but for the
// first: 4 bytes a token, four a load where it is aligned.
#pragma once

#include "rows.cuh"

namespace shahd {

constexpr int kLogThreads = 256;
constexpr int kLogWarps = kLogThreads / 32;
constexpr int kLogGroup = 4;     // rows of a block of threads, at most
constexpr int kLogDeep = 3;      // loads of the history of a thread in flight
constexpr int kLogTable = 4096;  // tokens of a slice's table, at most

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

// Two 16-bit or one 32-bit value, -inf where a token's bit is not set.
template <class T>
__device__ __forceinline__ uint32_t Masked(uint32_t u, uint32_t bits) {
  if constexpr (sizeof(T) == 4) {
    return bits & 1 ? u : 0xff800000u;
  } else {
    constexpr uint32_t kLow = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
    const uint32_t keep = (bits & 1 ? 0xffffu : 0u) | (bits & 2 ? 0xffff0000u : 0u);
    return (u & keep) | ((kLow << 16 | kLow) & ~keep);
  }
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
  // Which of the eight cells from t on are not 0.
  __device__ __forceinline__ uint32_t Eight(int t) const {
    uint32_t some = 0;
#pragma unroll
    for (int j = 0; j < (WIDE ? 2 : 1); j++) {
      const uint4 u = reinterpret_cast<const uint4*>(at + t)[j];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (WIDE) some |= (w[i] != 0 ? 1u : 0u) << (4 * j + i);
        else some |= ((w[i] & 0xffffu) != 0 ? 1u << 2 * i : 0u) | (w[i] >> 16 != 0 ? 2u << 2 * i : 0u);
      }
    }
    return some;
  }
};

// A token's count: 2 x times generated + whether the prompt has it.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kLogThreads, 4) AdjustLogitsKernel(const __grid_constant__ LogitsArgs a) {
  typedef typename LogCells<WIDE>::Cell Cell;
  constexpr int PER = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t log_raw[];
  __shared__ int seqs[kLogGroup], mask_rows[kLogGroup], lead[kLogGroup];  // lead: values between a 16-byte boundary and the row's beginning
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x / a.slices * a.group, sl = blockIdx.x % a.slices, rows = min(a.group, a.rows - first);
  // Pieces begin at 16-byte boundaries, rows where they like: slices are whole pieces, and a row reaches up to PER - 1 tokens into the
  // slice before. The table begins 8 tokens ahead; rows have 8 places more at either end, so that every token of it has a place.
  const int slice = a.table - 8, base = sl * slice - 8, pitch = a.table + 8, mask_words = a.table / 32 + 2;
  const bool counts = a.history != nullptr, biases = a.bias_tokens != nullptr;
  T* const held_rows = reinterpret_cast<T*>(log_raw);                                                         // [group][pitch]
  uint32_t* const held_masks = reinterpret_cast<uint32_t*>(log_raw + (size_t)a.group * pitch * sizeof(T));    // [group][mask_words]
  const LogCells<WIDE> table{reinterpret_cast<Cell*>(held_masks + (a.group * mask_words + 3) / 4 * 4)};
  const LogCells<WIDE> entry{table.at + (counts ? a.table : 0)};  // place of a token's last entry + 1
  uint16_t* const list = reinterpret_cast<uint16_t*>(entry.at + (biases ? a.table : 0)) + warp * 256;
  if (counts || biases)
    for (uint4* p = reinterpret_cast<uint4*>(table.at) + threadIdx.x; p < reinterpret_cast<uint4*>(entry.at + (biases ? a.table : 0)); p += kLogThreads)
      *p = make_uint4(0, 0, 0, 0);
  GridDepWait();
  GridDepLaunch();
  if ((int)threadIdx.x < rows) {
    seqs[threadIdx.x] = a.seqs ? a.seqs[first + threadIdx.x] : first + (int)threadIdx.x;
    mask_rows[threadIdx.x] = a.mask_rows ? a.mask_rows[first + threadIdx.x] : first + (int)threadIdx.x;
    lead[threadIdx.x] = (int)((reinterpret_cast<uintptr_t>(a.in) + (uintptr_t)((first + threadIdx.x) * a.in_row) * sizeof(T)) % 16 / sizeof(T));
  }
  __syncthreads();
  // The warps are dealt out to the rows: this one's row, its tokens v0 .. v1-1 of this slice, their whole pieces p0 .. p1-1 (inside the
  // row) and the values before and behind them; the warp takes every `step`-th 32 of what there is.
  const int mine = warp & (a.group - 1), begin = (warp / a.group) * 32 + lane, step = kLogThreads / a.group;
  const bool busy = mine < rows && (unsigned)seqs[min(mine, rows - 1)] < (unsigned)a.n;
  const int mis = lead[min(mine, rows - 1)], v0 = max(sl * slice - mis, 0), v1 = min((sl + 1) * slice - mis, a.vocab);
  const int p0 = (v0 + mis + PER - 1) / PER, p1 = max((v1 + mis) / PER, p0), head = min(p0 * PER - mis, v1), tail = max(p1 * PER - mis, head);
  T* const held = held_rows + mine * pitch + 8 + mis - sl * slice;  // held[v]: token v
  uint32_t* const bits = held_masks + mine * mask_words;            // from the word of v0 on
  const bool masked = busy && a.masks && (unsigned)mask_rows[mine] < (unsigned)a.mask_count && v0 < v1;
  if (busy) {
    const T* in = static_cast<const T*>(a.in) + (first + mine) * a.in_row;
    for (int c = p0 + begin; c < p1; c += step)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(SmemAddr(held + c * PER - mis)), "l"(in + c * PER - mis) : "memory");
    for (int v = v0 + begin; v < head; v += step) held[v] = in[v];
    for (int v = tail + begin; v < v1; v += step) held[v] = in[v];
    if (masked) {
      const uint32_t* mask = a.masks + mask_rows[mine] * a.mask_stride + (v0 >> 5);
      const int words = ((v1 - 1) >> 5) - (v0 >> 5) + 1;
      for (int i = begin; i < words; i += step)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(SmemAddr(bits + i)), "l"(mask + i) : "memory");
    }
  }
  for (int r = 0; (counts || biases) && r < rows;) {
    const int seq = seqs[r], from = r;
    while (r < rows && seqs[r] == seq) r++;
    if ((unsigned)seq >= (unsigned)a.n) continue;
    // ---- the tokens that there are: the table is empty ----
    int b0 = 0;
    if (biases) {
      b0 = min(max(a.bias_offsets[seq], 0), a.bias_entries);
      const int count = min(max(a.bias_offsets[seq + 1], b0), a.bias_entries) - b0;
      for (int i = threadIdx.x; i < count; i += kLogThreads) {
        // in unsigned numbers, which wrap: any value may stand there
        const uint32_t t = (uint32_t)a.bias_tokens[b0 + i] - (uint32_t)base;
        if (t < (uint32_t)a.table) entry.Max(t, (uint32_t)i + 1u);
      }
    }
    float rep = 1.f, inv = 1.f, freq = 0.f, pres = 0.f;
    if (counts) {
      const int* h = a.history + seq * a.history_stride;
      const int length = (int)min((long long)max(a.held[seq], 0), a.history_stride), prompt = a.prompt ? a.prompt[seq] : 0;
      rep = a.repetition ? a.repetition[seq] : 1.f;
      inv = 1.f / rep;  // a division for a row instead of one for a token: half a step more
      freq = a.frequency ? a.frequency[seq] : 0.f;
      pres = a.presence ? a.presence[seq] : 0.f;
      const auto meet = [&](int token, int i) {
        const uint32_t t = (uint32_t)token - (uint32_t)base;
        if (t < (uint32_t)a.table) {
          if (i < prompt) table.Or(t, 1);
          else table.Add(t, 2);
        }
      };
      const int fours = reinterpret_cast<uintptr_t>(h) % 16 == 0 ? length / 4 : 0;
#pragma unroll 1
      for (int i0 = threadIdx.x; i0 < fours; i0 += kLogDeep * kLogThreads) {
        int4 u[kLogDeep];
#pragma unroll
        for (int k = 0; k < kLogDeep; k++)
          if (i0 + k * kLogThreads < fours) u[k] = reinterpret_cast<const int4*>(h)[i0 + k * kLogThreads];
#pragma unroll
        for (int k = 0; k < kLogDeep; k++) {
          const int i = i0 + k * kLogThreads;
          if (i >= fours) break;
          meet(u[k].x, 4 * i);
          meet(u[k].y, 4 * i + 1);
          meet(u[k].z, 4 * i + 2);
          meet(u[k].w, 4 * i + 3);
        }
      }
#pragma unroll 1
      for (int i0 = 4 * fours + (int)threadIdx.x; i0 < length; i0 += 4 * kLogThreads) {
        int u[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (i0 + k * kLogThreads < length) u[k] = h[i0 + k * kLogThreads];
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (i0 + k * kLogThreads < length) meet(u[k], i0 + k * kLogThreads);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // ---- this warp's part of them: tokens 256 k + .. of every kLogWarps-th k ----
#pragma unroll 1
    for (int t0 = warp * 256; t0 < a.table; t0 += kLogWarps * 256) {
      const int t = t0 + 8 * lane;
      uint32_t some = 0;  // bit j: token t + j is there
      if (counts) some |= table.Eight(t);
      if (biases) some |= entry.Eight(t);
      int upto = __popc(some);  // of the lanes up to this one
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const int listed = __shfl_sync(0xffffffffu, upto, 31);
      int at = upto - __popc(some);
      __syncwarp();  // the last list has been read
      for (; some != 0; some &= some - 1) list[at++] = (uint16_t)(t + __ffs(some) - 1);
      __syncwarp();
#pragma unroll 1
      for (int i = lane; i < listed; i += 32) {
        const int t = list[i];
        const uint32_t w = counts ? table.at[t] : 0, e = biases ? entry.at[t] : 0, times = w >> 1;
        const float bias = e != 0 ? a.bias_values[b0 + (int)e - 1] : 0.f, fine = times != 0 ? fmaf((float)times, freq, pres) : 0.f;
        for (int k = from; k < r; k++) {
          T* at = held_rows + k * pitch + lead[k] + t;
          float x = ToFloat(*at);
          if (w != 0) x = x > 0.f ? x * inv : x * rep;
          if (times != 0) x -= fine;
          if (e != 0) x += bias;
          *at = FromFloat<T>(x);
        }
        if (r < rows) {  // empty again
          if (counts) table.at[t] = 0;
          if (biases) entry.at[t] = 0;
        }
      }
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
      constexpr int kTwo = PER / 4;  // tokens of a word
      const uint32_t allowed = __funnelshift_r(bits[(v >> 5) - word0], bits[((v + PER - 1) >> 5) - word0], v & 31);
      u = make_uint4(Masked<T>(u.x, allowed), Masked<T>(u.y, allowed >> kTwo), Masked<T>(u.z, allowed >> 2 * kTwo), Masked<T>(u.w, allowed >> 3 * kTwo));
    }
    *reinterpret_cast<uint4*>(out + v) = u;
  }
  const auto single = [&](int v) { out[v] = !masked || (bits[(v >> 5) - word0] >> (v & 31) & 1) ? held[v] : FromFloat<T>(-INFINITY); };
  for (int v = v0 + begin; v < (alike ? head : v1); v += step) single(v);
  if (alike)
    for (int v = tail + begin; v < v1; v += step) single(v);
}

template <class T>
void LaunchLogits(const LogitsArgs& a, bool wide, int smem, cudaStream_t st) {
  const auto kernel = wide ? AdjustLogitsKernel<T, true> : AdjustLogitsKernel<T, false>;
  if (!EnsureKernelAttrs((const void*)kernel, smem)) return;
  LaunchPdl(kernel, dim3((unsigned)(CeilDiv(a.rows, a.group) * a.slices)), dim3(kLogThreads), (size_t)smem, st, a);
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
  // Slices of whole pieces, as many as give every multiprocessor a few blocks of threads; rows in groups where they share sequences and enough are left.
  const auto lay = [&](int table) {
    a.table = table;
    a.slices = CeilDiv(c->vocab + 7, table - 8);  // a row that does not begin at a boundary reaches up to 7 values further
  };
  lay(kLogTable);
  while (a.table > 1024 && (long long)c->rows * a.slices < 4 * info.sms) lay(a.table / 2);
  a.group = 1;
  while (c->rows / c->n >= 2 * a.group && a.group < kLogGroup && (long long)c->rows / (2 * a.group) * a.slices >= 4 * info.sms) a.group *= 2;
  if ((long long)a.rows * a.slices > 0x7fffffffLL) {
    SetError("%s: too many rows of this vocabulary: %d of %d", op, c->rows, c->vocab);
    return SHAHD_EINVAL;
  }
  const bool wide = (a.history && a.history_stride > 0x7fff) || a.bias_entries > 0xfffe;  // a cell of 16 bits holds 2 x 2^15 - 1, and 2^16 - 1
  // rows, masks, counts, entries, lists
  const int smem = a.group * (a.table + 8) * (int)size + RoundUp(a.group * (a.table / 32 + 2), 4) * 4 +
                   (a.history || a.bias_tokens ? a.table * ((a.history ? 1 : 0) + (a.bias_tokens ? 1 : 0)) * (wide ? 4 : 2) + kLogWarps * 512 : 0);
  TakeLaunchError(nullptr);
  if (c->dtype == SHAHD_F32) LaunchLogits<float>(a, wide, smem, static_cast<cudaStream_t>(stream));
  else if (c->dtype == SHAHD_F16) LaunchLogits<__half>(a, wide, smem, static_cast<cudaStream_t>(stream));
  else LaunchLogits<bf16>(a, wide, smem, static_cast<cudaStream_t>(stream));
  return LaunchStatus(op);
}

}  // extern "C"
