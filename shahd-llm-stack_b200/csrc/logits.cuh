// Penalties for repeated tokens, biases and grammar masks on rows of logits, before sampling.
//   x = logit of token v; c = how often v was generated, known = v is in the prompt or was generated;
//   known: x > 0 ? x / repetition : x * repetition;  x -= c frequency + [c > 0] presence;  x += bias of v;  not allowed: -inf.
// Formed in 32 bits, rounded once.
//
// Bound by memory: a row is read once and written once. A block of threads takes a slice of a row's tokens: it counts the
// history's tokens of the slice in shared memory (whole numbers, so the order of the atomics does not matter), then runs over
// the slice in 16-byte pieces. The history is read by every slice's block, from the cache but for the first: 4 bytes a token.
#pragma once

#include "rows.cuh"

namespace shahd {

constexpr int kLogThreads = 256;
constexpr int kLogSlice = 8192;  // tokens of a slice, at most

struct LogitsArgs {
  const void* in;
  void* out;
  long long in_row, out_row;  // elements
  int rows, vocab, n, slice, slices;
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

template <class T>
__global__ void __launch_bounds__(kLogThreads) AdjustLogitsKernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ uint32_t table[];  // [slice] 2 x times generated + known; with biases then [slice] the place of the token's last entry + 1
  constexpr int PER = 16 / sizeof(T);
  GridDepWait();
  GridDepLaunch();
  const int row = blockIdx.x / a.slices, sl = blockIdx.x - row * a.slices;
  const int seq = a.seqs ? a.seqs[row] : row;
  if ((unsigned)seq >= (unsigned)a.n) return;
  const T* in = static_cast<const T*>(a.in) + row * a.in_row;
  T* out = static_cast<T*>(a.out) + row * a.out_row;
  // pieces begin at 16-byte boundaries; slices are whole pieces, so the first one may be short by what lies before the row
  const int mi = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T)), mo = (int)(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T));
  const int mis = mi == mo ? mi : 0;
  const int v0 = max(sl * a.slice - mis, 0), v1 = min((sl + 1) * a.slice - mis, a.vocab);
  if (v0 >= v1) return;
  const int size = v1 - v0;
  uint32_t* entry = table + a.slice;
  const bool counts = a.history != nullptr, biases = a.bias_tokens != nullptr;
  if (counts)
    for (int i = threadIdx.x; i < size; i += kLogThreads) table[i] = 0;
  if (biases)
    for (int i = threadIdx.x; i < size; i += kLogThreads) entry[i] = 0;
  __syncthreads();
  if (counts) {
    const int* h = a.history + seq * a.history_stride;
    const int held = (int)min((long long)max(a.held[seq], 0), a.history_stride), prompt = a.prompt ? a.prompt[seq] : 0;
    for (int i = threadIdx.x; i < held; i += kLogThreads) {
      const uint32_t t = (uint32_t)h[i] - (uint32_t)v0;  // in unsigned numbers, which wrap: any value may stand there
      if (t < (uint32_t)size) {
        if (i < prompt) atomicOr(&table[t], 1u);
        else atomicAdd(&table[t], 2u);
      }
    }
  }
  if (biases) {
    const int b = min(max(a.bias_offsets[seq], 0), a.bias_entries), e = min(max(a.bias_offsets[seq + 1], b), a.bias_entries);
    for (int i = b + (int)threadIdx.x; i < e; i += kLogThreads) {
      const uint32_t t = (uint32_t)a.bias_tokens[i] - (uint32_t)v0;
      if (t < (uint32_t)size) atomicMax(&entry[t], (uint32_t)i + 1u);
    }
  }
  const float rep = a.repetition ? a.repetition[seq] : 1.f, freq = a.frequency ? a.frequency[seq] : 0.f, pres = a.presence ? a.presence[seq] : 0.f;
  const uint32_t* mask = nullptr;
  if (a.masks) {
    const int m = a.mask_rows ? a.mask_rows[row] : row;
    if ((unsigned)m < (unsigned)a.mask_count) mask = a.masks + m * a.mask_stride;
  }
  __syncthreads();
  const auto adjusted = [&](float x, int v, bool allowed) {
    const uint32_t c = counts ? table[v - v0] : 0;
    if (c != 0) {
      x = x > 0.f ? x / rep : x * rep;
      if (c > 1) x -= fmaf((float)(c >> 1), freq, pres);
    }
    if (biases) {
      const uint32_t at = entry[v - v0];
      if (at != 0) x += a.bias_values[at - 1];
    }
    return allowed ? x : -INFINITY;
  };
  // whole pieces lie inside the row
  const int p0 = (v0 + mis + PER - 1) / PER, p1 = mi == mo ? max((v1 + mis) / PER, p0) : p0;
  for (int c = p0 + (int)threadIdx.x; c < p1; c += kLogThreads) {
    const int v = c * PER - mis;
    uint4 u = *reinterpret_cast<const uint4*>(in + v);
    uint32_t allowed = 0xffffffffu;
    if (mask) allowed = __funnelshift_r(mask[v >> 5], mask[(v + PER - 1) >> 5], v & 31);
    T* x = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = FromFloat<T>(adjusted(ToFloat(x[i]), v + i, allowed >> i & 1));
    *reinterpret_cast<uint4*>(out + v) = u;
  }
  const auto single = [&](int v) { out[v] = FromFloat<T>(adjusted(ToFloat(in[v]), v, mask ? mask[v >> 5] >> (v & 31) & 1 : true)); };
  const int head = p1 > p0 ? p0 * PER - mis : v1, tail = p1 > p0 ? p1 * PER - mis : v1;  // the values around the pieces
  for (int v = v0 + (int)threadIdx.x; v < head; v += kLogThreads) single(v);
  for (int v = tail + (int)threadIdx.x; v < v1; v += kLogThreads) single(v);
}

template <class T>
void LaunchLogits(const LogitsArgs& a, int smem, cudaStream_t st) {
  if (!EnsureKernelAttrs((const void*)AdjustLogitsKernel<T>, smem)) return;
  LaunchPdl(AdjustLogitsKernel<T>, dim3((unsigned)(a.rows * a.slices)), dim3(kLogThreads), (size_t)smem, st, a);
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
  if (c->history ? c->history_stride < 0 || c->history_stride > (1 << 30) || !c->history_lengths
                 : c->history_lengths || c->prompt_lengths || c->repetition || c->presence || c->frequency) {
    SetError("%s: a history goes with history_lengths and a stride in 0 .. 2^30, and penalties with a history (got stride %lld)", op, (long long)c->history_stride);
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
  // Slices: whole pieces, as many as give every multiprocessor a few blocks of threads, 1024 to kLogSlice tokens each.
  a.slice = kLogSlice;
  while (a.slice > 1024 && (long long)c->rows * CeilDiv(c->vocab, a.slice) < 2 * info.sms) a.slice /= 2;
  a.slices = CeilDiv(c->vocab + 7, a.slice);  // a row that does not begin at a boundary reaches up to 7 values further
  if ((long long)a.rows * a.slices > 0x7fffffffLL) {
    SetError("%s: too many rows of this vocabulary: %d of %d", op, c->rows, c->vocab);
    return SHAHD_EINVAL;
  }
  const int smem = a.slice * 4 * ((a.history ? 1 : 0) + (a.bias_tokens ? 2 : 0) > 1 ? 2 : 1);
  TakeLaunchError(nullptr);
  if (c->dtype == SHAHD_F32) LaunchLogits<float>(a, smem, static_cast<cudaStream_t>(stream));
  else if (c->dtype == SHAHD_F16) LaunchLogits<__half>(a, smem, static_cast<cudaStream_t>(stream));
  else LaunchLogits<bf16>(a, smem, static_cast<cudaStream_t>(stream));
  return LaunchStatus(op);
}

}  // extern "C"
