// The fourth translation unit of libshahd_b200.so: attention of chunks of new tokens over the paged cache (section 4 of shahd_b200.h),
// on the tile attention; a unit of its own, since its kernels take as long to compile as the others together.
#include "tile_host.cuh"

namespace shahd {

int ChunkDeviceError() { return TileDeviceError(); }

namespace {

template <int D, bool F16>
void LaunchChunks(const TaArgs& a, unsigned blocks, cudaStream_t st) {
  if (a.split > 1) {
    if (!EnsureKernelAttrs((const void*)TileAttentionKernel<D, F16, kChunkSplit>, TaCfg<D>::kSmem)) return;
    LaunchPdlCluster(TileAttentionKernel<D, F16, kChunkSplit>, dim3(blocks), dim3(TaCfg<D>::kThreads), TaCfg<D>::kSmem, dim3((unsigned)a.split), st, a);
    return;
  }
  if (a.least == 0) {
    if (!EnsureKernelAttrs((const void*)TileAttentionKernel<D, F16, kChunkPairs>, TaCfg<D>::kSmem)) return;
    LaunchPdl(TileAttentionKernel<D, F16, kChunkPairs>, dim3(blocks), dim3(TaCfg<D>::kThreads), TaCfg<D>::kSmem, st, a);
    return;
  }
  if (!EnsureKernelAttrs((const void*)TileAttentionKernel<D, F16, kChunkRanges>, TaCfg<D>::kSmem)) return;
  LaunchPdl(TileAttentionKernel<D, F16, kChunkRanges>, dim3(blocks), dim3(TaCfg<D>::kThreads), TaCfg<D>::kSmem, st, a);
  LaunchPdl(ChunkJoinKernel<D, F16>, dim3(blocks * CeilDiv(a.part_rows, kJoinRows<D>)), dim3(256), 0, st, a);
}

// How a call's work is laid out; times are of one graph, 16/4 heads of 64 if nothing else is said.
//   Pairs: a block of threads for every pair of tiles, longest first, where there are many of them. 16 chunks of 300 to 2048 rows from position
//     0: 121 us, ranges 154, tiles 151.
//   Tiles: a block of threads for every tile, its key blocks by turns: half as many steps, at twice the loads. Where pairs are few enough that
//     the longest is what is waited for: 48 sequences, six of them with 200 to 512 rows, 0 to 1500 positions: 40 us, pairs 44, ranges 46; 8192
//     rows from position 0: 198, pairs 208, ranges 218. At head_dim 128 the loads tell: 2 chunks of 1024 over 12000, 32/8 heads: 500, pairs and
//     ranges 440 to 470 (454).
//   Split: a cluster of 2 to 8 blocks of threads for every tile, where that leaves multiprocessors for all and the steps are few: one
//     launch, no second kernel. 96 rows over 1700 positions: 11.2 us, pairs split in eight 13.4, ranges 20, pairs 36.
//   Ranges: as many blocks of threads as run at once take ranges of equal cost out of the line of all pairs, and what a range cuts is joined
//     by a second kernel. Long caches and few pairs: 4 chunks of 500 to 1024 rows over 3000 to 9000 positions: 143 to 166 us, tiles 202, pairs 220. The
//     second kernel and the parts cost about eight steps.
// Pairs go longest first over all kv heads; where the keys and values do not fit the L2 cache, head after head, so that the blocks of threads that
// run at a time read the same ones (4 chunks of 1500 to 2048 rows over 10 to 24 thousand positions, 32/8 heads of 128, 427 MB: 2820 us and
// 2511; but 2 of 7000 to 8192 from position 0, 16/2 heads of 128, 16 MB: 467 and 513).
// The lengths lie on the device, so the table's width stands for them, and a table much wider than its sequences are long may get the
// layout for longer ones.
struct ChunkLayout {
  int span, least, part_rows, two_heads, split, by_heads;
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
  const int G = H / Hk, TB = 128 / G, keys = d == 128 ? 128 : 64;
  // tiles of all sequences together, `span` tokens each, at most
  const auto tiles_of = [&](int span) { return std::min((long long)c->rows / span + c->n, (long long)c->n * CeilDiv(std::min(c->max_rows, 1 << 30), span)) * Hk; };
  const long long pairs = tiles_of(2 * TB), blocks = CeilDiv(c->cache.max_blocks, keys / 64);
  const long long most = pairs * (blocks + kPairCost);  // what all pairs cost, if all sequences were as long
  const long long places = (long long)c->rows / TB + c->n;
  if (c->rows > kOpsMaxRows || pairs / Hk > (1 << 23) || most > 0x3fffffffLL || places * Hk > 0x3fffffff) {
    SetError("%s: too many rows or key blocks: %d rows, %d sequences, %d pages each", op, c->rows, c->n, c->cache.max_blocks);
    return SHAHD_EINVAL;
  }
  ChunkLayout l = {};
  const long long slots = kTaSms * (d == 128 ? 1 : 2);
  l.split = 1;
  const long long tiles = tiles_of(TB);
  while (l.split < 8 && tiles * l.split * 2 <= slots) l.split *= 2;
  const bool many = pairs >= 4 * slots;
  const bool ranges = !many && (pairs >= slots ? blocks >= 64 && (d == 128 || tiles < 3 * slots)
                                               : (tiles * l.split + slots - 1) / slots * blocks / (2 * l.split) > pairs * blocks / slots + 8);
  l.span = many || ranges ? 2 * TB : TB;
  l.part_rows = std::min(c->max_rows, l.span) * G;
  if (ranges) {
    l.split = 1;
    l.least = 256 / keys + kPairCost;
    l.grid = std::max(1LL, std::min(slots, (most + l.least - 1) / l.least));
    l.cut_bytes = (l.grid * (int64_t)sizeof(int4) + 255) / 256 * 256;
    l.bytes = l.cut_bytes + 2 * l.grid * l.part_rows * (d + 2) * (int64_t)sizeof(float);
  } else if (l.split > 1) {
    l.grid = places * Hk * l.split;
    l.bytes = l.grid * l.part_rows * (d + 2) * (int64_t)sizeof(float);
  } else {  // one tile of rows: those of two kv heads together take half as many blocks of threads, and no merge
    l.two_heads = c->max_rows <= TB && Hk % 2 == 0;
    l.by_heads = (double)c->n * c->cache.max_blocks * kOpsPage * Hk * 2 * d * 2 > 126e6;
    l.grid = ((long long)c->rows / l.span + c->n) * Hk / (l.two_heads ? 2 : 1);
  }
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
  if (lay.bytes > 0) b.Add("workspace", c->workspace, 32);
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
  a.span = lay.span;
  a.two_heads = lay.two_heads;
  a.split = lay.split;
  a.by_heads = lay.by_heads;
  if (lay.bytes > 0) {
    a.part_rows = lay.part_rows;
    a.cuts = static_cast<int4*>(c->workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(c->workspace) + lay.cut_bytes);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (lay.split > 1 ? 1 : 2) * lay.grid * lay.part_rows * d);
  }
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
