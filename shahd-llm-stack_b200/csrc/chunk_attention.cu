// The fourth translation unit of libshahd_b200.so: attention of chunks of new tokens over the paged cache (section 4 of shahd_b200.h),
// on the tile attention; a unit of its own, since its kernels take as long to compile as the others together.
#include "tile_host.cuh"

namespace shahd {

int ChunkDeviceError() { return TileDeviceError(); }

namespace {

template <int D, bool F16>
void LaunchChunks(const TaArgs& a, unsigned blocks, cudaStream_t st) {
  if (!EnsureKernelAttrs((const void*)TileAttentionKernel<D, F16, kChunkRanges>, TaCfg<D>::kSmem)) return;
  LaunchPdl(TileAttentionKernel<D, F16, kChunkRanges>, dim3(blocks), dim3(TaCfg<D>::kThreads), TaCfg<D>::kSmem, st, a);
  LaunchPdl(ChunkJoinKernel<D, F16>, dim3(blocks * CeilDiv(a.part_rows, 8)), dim3(256), 0, st, a);
}

// How a call's work is laid out: as many blocks of threads as run at once take ranges of equal length out of all key blocks of all tile
// pairs, 256 keys at least, and the pairs that a range cuts are joined by a second kernel.
struct ChunkLayout {
  int least, part_rows;
  long long grid;
  int64_t cut_bytes, bytes;
};

int LayChunks(const char* op, const ShahdChunkCall* c, ChunkLayout* out) {
  const int H = c->num_heads, Hk = c->cache.kv_heads, d = c->cache.head_dim;
  if (!CheckHeads(op, H, Hk, d) || !CheckCache(op, c->cache, Hk, d)) return SHAHD_EINVAL;
  if (c->n < 0 || c->rows < 0 || c->max_rows < 1) {
    SetError("%s: need n, rows >= 0 and max_rows >= 1 (got n=%d rows=%d max_rows=%d)", op, c->n, c->rows, c->max_rows);
    return SHAHD_EINVAL;
  }
  const int G = H / Hk, span = 2 * (128 / G), keys = d == 128 ? 128 : 64;
  const long long pairs = std::min((long long)c->rows / span + c->n, (long long)c->n * CeilDiv(std::min(c->max_rows, 1 << 30), span));
  const long long most = pairs * Hk * CeilDiv(c->cache.max_blocks, keys / 64);  // key blocks of all pairs, if all sequences were as long
  if (c->rows > kOpsMaxRows || pairs > (1 << 23) || most > 0x3fffffffLL) {
    SetError("%s: too many rows or key blocks: %d rows, %d sequences, %d pages each", op, c->rows, c->n, c->cache.max_blocks);
    return SHAHD_EINVAL;
  }
  ChunkLayout l = {};
  const long long slots = kTaSms * (d == 128 ? 1 : 2);
  l.least = 256 / keys;
  l.grid = std::max(1LL, std::min(slots, (most + l.least - 1) / l.least));
  l.part_rows = std::min(c->max_rows, span) * G;
  l.cut_bytes = (l.grid * (int64_t)sizeof(int4) + 255) / 256 * 256;
  l.bytes = l.cut_bytes + 2 * l.grid * l.part_rows * (d + 2) * (int64_t)sizeof(float);
  *out = l;
  return SHAHD_OK;
}

}  // namespace
}  // namespace shahd

extern "C" {

int64_t shahd_chunk_attention_workspace(const ShahdChunkCall* c) {
  using namespace shahd;
  const char* op = "shahd_chunk_attention_workspace";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  ChunkLayout l;
  const int rc = LayChunks(op, c, &l);
  return rc == SHAHD_OK ? l.bytes : rc;
}

int shahd_chunk_attention(const ShahdChunkCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_chunk_attention";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  TaArgs a = {};
  const int H = c->num_heads, Hk = c->cache.kv_heads, d = c->cache.head_dim;
  ChunkLayout lay;
  const int rc = LayChunks(op, c, &lay);
  if (rc != SHAHD_OK) return rc;
  if (!CheckType(op, c->dtype, false) || !ScaleOf(op, c->scale, d, &a.scale_log2)) return SHAHD_EINVAL;
  if (!CheckRows(op, "q", c->q, c->rows, H, d, 8) || !CheckRows(op, "out", c->out, c->rows, H, d, 8, true)) return SHAHD_EINVAL;
  if (c->n == 0 || c->rows == 0) return SHAHD_OK;
  if (c->workspace_bytes < lay.bytes) {
    SetError("%s: needs %lld bytes of workspace, got %lld", op, (long long)lay.bytes, (long long)c->workspace_bytes);
    return SHAHD_EINVAL;
  }
  BufferCheck b(op);
  b.Add("offsets", c->offsets, 4);
  b.Add("lengths", c->lengths, 4);
  b.Add("q", c->q.data, 16);
  b.Add("out", c->out.data, 16);
  b.Add("cache.pool", c->cache.pool, 16);
  b.Add("cache.block_table", c->cache.block_table, 4);
  b.Add("workspace", c->workspace, 32);
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  a.G = H / Hk;
  a.TB = 128 / a.G;
  if (!MakeMap(c->dtype, c->q.data, d, H, c->rows, c->q.head_stride, c->q.row_stride, a.G, a.TB, &a.qmap) ||
      !MakeMap(c->dtype, c->cache.pool, d, (uint64_t)Hk * 2 * kOpsPage, c->cache.pages, d, c->cache.page_stride, kOpsPage, 1, &a.pool)) {
    SetError("%s: a tensor map of q or the cache could not be made", op);
    return SHAHD_ECUDA;
  }
  a.out = static_cast<uint16_t*>(c->out.data);
  a.out_row = c->out.row_stride;
  a.out_head = c->out.head_stride;
  a.offsets = c->offsets;
  a.n = c->n;
  a.rows = c->rows;
  a.H = H;
  a.Hk = Hk;
  a.lengths = c->lengths;
  a.table = c->cache.block_table;
  a.max_blocks = c->cache.max_blocks;
  a.pages = c->cache.pages;
  a.max_nodes = c->max_rows;
  a.least = lay.least;
  a.part_rows = lay.part_rows;
  a.cuts = static_cast<int4*>(c->workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(c->workspace) + lay.cut_bytes);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + 2 * lay.grid * lay.part_rows * d);
  TakeLaunchError(nullptr);
  g_waiting_devices.Add(b.device);
  const unsigned blocks = (unsigned)lay.grid;
  const bool f16 = c->dtype == SHAHD_F16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d == 32) f16 ? LaunchChunks<32, true>(a, blocks, st) : LaunchChunks<32, false>(a, blocks, st);
  else if (d == 64) f16 ? LaunchChunks<64, true>(a, blocks, st) : LaunchChunks<64, false>(a, blocks, st);
  else f16 ? LaunchChunks<128, true>(a, blocks, st) : LaunchChunks<128, false>(a, blocks, st);
  return LaunchStatus(op);
}

}  // extern "C"
