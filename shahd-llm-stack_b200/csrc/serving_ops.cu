// The second translation unit of libshahd_b200.so: the operators on caller-owned device buffers (section 3 of
// shahd_b200.h). They share no device state with the session's kernels, so they compile beside them; their kernels record
// a wait that gave up in a flag of their own, which ShahdDeviceErrorFlag reads too.
#include <new>
#include <type_traits>

#include "device_flags.h"
#include "ops_common.cuh"
#include "rope.cuh"
#include "tile_attention.cuh"
#include "tree_verify.cuh"

namespace shahd {

// The operators run where their buffers are, so a wait that gave up may have been recorded on any device that a kernel with waits
// (the tile attention) has been launched on.
static DeviceSet g_waiting_devices;

int OpsDeviceError() {
  return FirstFlag(g_waiting_devices, [](int device, int* flag) {
    DeviceScope scope(device);
    if (scope.ok && cudaMemcpyFromSymbol(flag, g_ops_device_error, sizeof *flag) == cudaSuccess) return true;
    cudaGetLastError();
    return false;
  });
}

namespace {

typedef CUresult (*OpsEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

OpsEncodeFn OpsEncode() {
  static const OpsEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<OpsEncodeFn>(p);
  }();
  return fn;
}

// A map of 16-bit values (x, y, z) with 128-byte swizzle and boxes of 64 x by x bz. Made for every call: it is a
// computation of the call's own pointers and strides, a fraction of a microsecond.
bool MakeMap(int dtype, const void* p, uint64_t nx, uint64_t ny, uint64_t nz, int64_t sy, int64_t sz, int by, int bz, CUtensorMap* m) {
  const OpsEncodeFn enc = OpsEncode();
  if (!enc) return false;
  if (ny == 1) sy = (int64_t)nx;  // the stride of a single row or head is free: TMA wants one that it could use
  if (nz == 1) sz = (int64_t)nx;
  const cuuint64_t dims[3] = {nx, ny, nz}, strides[2] = {(cuuint64_t)sy * 2, (cuuint64_t)sz * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)by, (cuuint32_t)bz}, step[3] = {1, 1, 1};
  return enc(m, dtype == SHAHD_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims,
             strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool CheckHeads(const char* op, int H, int Hk, int d) {
  if (H >= 1 && Hk >= 1 && H % Hk == 0 && H / Hk <= 8 && H <= (1 << 16) && (d == 32 || d == 64 || d == 128)) return true;
  SetError("%s: need kv_heads dividing num_heads with at most 8 query heads per kv head and head_dim 32, 64 or 128 (got "
           "num_heads=%d kv_heads=%d head_dim=%d)", op, H, Hk, d);
  return false;
}

bool ScaleOf(const char* op, double scale, int d, float* log2) {
  if (scale == 0) scale = 1.0 / std::sqrt((double)d);
  *log2 = (float)(scale * M_LOG2E);
  if (!(*log2 > 0) || !std::isfinite(*log2)) {  // in 32 bits, too: masked scores are -inf times it
    SetError("%s: scale must be positive and finite in 32 bits, or 0 for 1/sqrt(head_dim) (got %g)", op, scale);
    return false;
  }
  return true;
}

template <int D, bool F16, int KIND>
void LaunchTiles(const TaArgs& a, unsigned blocks, cudaStream_t st) {
  if (!EnsureKernelAttrs((const void*)TileAttentionKernel<D, F16, KIND>, TaCfg<D>::kSmem)) return;
  LaunchPdl(TileAttentionKernel<D, F16, KIND>, dim3(blocks), dim3(TaCfg<D>::kThreads), TaCfg<D>::kSmem, st, a);
  if constexpr (KIND == kTreeRanges)
    LaunchPdl(TreeJoinKernel<D, F16>, dim3((unsigned)(((long long)a.rows * a.H + 7) / 8)), dim3(256), 0, st, a);
}

template <int KIND>
void LaunchTiles(int d, int dtype, const TaArgs& a, unsigned blocks, cudaStream_t st) {
  const bool f16 = dtype == SHAHD_F16;
  if (d == 32) f16 ? LaunchTiles<32, true, KIND>(a, blocks, st) : LaunchTiles<32, false, KIND>(a, blocks, st);
  else if (d == 64) f16 ? LaunchTiles<64, true, KIND>(a, blocks, st) : LaunchTiles<64, false, KIND>(a, blocks, st);
  else f16 ? LaunchTiles<128, true, KIND>(a, blocks, st) : LaunchTiles<128, false, KIND>(a, blocks, st);
}

bool MakeRowMaps(const char* op, int dtype, int d, int H, int Hk, int rows, const ShahdRows& q, const ShahdRows& k, const ShahdRows& v, TaArgs* a) {
  if (MakeMap(dtype, q.data, d, H, rows, q.head_stride, q.row_stride, a->G, a->TB, &a->qmap) &&
      MakeMap(dtype, k.data, d, Hk, rows, k.head_stride, k.row_stride, 1, kOpsPage, &a->kmap) &&
      MakeMap(dtype, v.data, d, Hk, rows, v.head_stride, v.row_stride, 1, kOpsPage, &a->vmap))
    return true;
  SetError("%s: a tensor map of q, k or v could not be made", op);
  return false;
}

// How a tree call's work is laid out. Where there are many tile pairs, or enough with short caches, each has a block of threads
// of its own. Elsewhere as many blocks of threads as run at once take ranges of equal length out of all key blocks of all pairs,
// 256 keys at least, and the pairs that a range cuts are joined by a second kernel: so long caches and short ones, one sequence and a
// few hundred, end together. A range costs the second kernel, about as long as eight steps, and both parts' rows written and
// read in 32 bits; so where there is a place for every pair and its steps are few, pairs it is (72 trees of 13 to 26 nodes,
// 12/4 heads of 64, up to 254 positions: ranges 29 us, pairs 10.9; 8 single tokens, 32/8 heads of 128, up to 2000 positions: 25.9
// and 21.6; one tree of 24 over 2047 positions, 16/4 heads of 64: 13.5 and 23.3). 16 trees over 20 to 32 thousand positions, 8
// kv heads of 128, kernel alone: a block of threads for each pair 490 us, parts of 2048 keys 513, ranges 427; but 512 pairs of
// 400 to 576 positions, 1.7 for each place: 33 us and 42, 31 as 256 pairs of heads. The lengths lie on the device, so the table's width
// stands for them: in one much wider than its sequences are long a call may take the slower layout (256 single tokens, 8/2 heads of
// 64, 400 to 576 positions: 19 us in a table of 9 pages, 45 in one of 64 or 512; 72 trees as above, one of them over 32000 positions: 311).
constexpr int kTaSms = 148;  // of a B200: the layout, and so the workspace, does not hang on a device being there
struct TreeLayout {
  int pairs, two_heads, least, part_rows;
  long long grid;
  int64_t plan_bytes, bytes;
};

int LayTree(const char* op, const ShahdTreeCall* c, TreeLayout* out) {
  const int H = c->num_heads, Hk = c->cache.kv_heads, d = c->cache.head_dim;
  if (!CheckHeads(op, H, Hk, d) || !CheckCache(op, c->cache, Hk, d)) return SHAHD_EINVAL;
  if (c->n < 0 || c->max_nodes < 1 || c->max_nodes > 64) {
    SetError("%s: need n >= 0 and max_nodes in 1 .. 64 (got n=%d max_nodes=%d)", op, c->n, c->max_nodes);
    return SHAHD_EINVAL;
  }
  const int G = H / Hk, TB = 128 / G, keys = d == 128 ? 128 : 64;
  TreeLayout l = {};
  l.pairs = CeilDiv(c->max_nodes, 2 * TB);
  const long long slots = kTaSms * (d == 128 ? 1 : 2), tiles = (long long)c->n * Hk * l.pairs;
  const long long most = tiles * (CeilDiv(c->cache.max_blocks, keys / 64) + 1);  // key blocks of all pairs, if all sequences were as long
  if (most > 0x3fffffffLL) {
    SetError("%s: too many key blocks: %lld tile pairs over %d pages each", op, tiles, c->cache.max_blocks);
    return SHAHD_EINVAL;
  }
  // steps of a pair's two tiles, the whole call's in ranges (by turns a step takes two blocks of keys, and costs a merge of about two)
  const bool turns = c->max_nodes <= TB;
  const long long blocks = CeilDiv(c->cache.max_blocks, keys / 64) + 1, alone = turns ? blocks / 2 + 2 : blocks;
  const long long dealt = std::max(most / slots, 256LL / keys) / (turns ? 2 : 1) + 8 + 4LL * std::min(c->max_nodes, 2 * TB) * G / keys;
  if (tiles >= 8 * slots || (tiles >= slots && c->cache.max_blocks < 64) || (tiles < slots && alone <= dealt)) {
    // one tile of rows: those of two kv heads together take half as many blocks of threads as one by turns, and no merge; where
    // there are places for all, by turns half the steps (72 trees of 13 to 26, 12/4 heads, up to 254 positions: 10.9 and 11.7 us)
    l.two_heads = turns && Hk % 2 == 0 && tiles >= slots;
    l.grid = l.two_heads ? tiles / 2 : tiles;
  } else {
    l.least = 256 / keys;
    l.grid = std::max(1LL, std::min(slots, (most + l.least - 1) / l.least));
    l.part_rows = std::min(c->max_nodes, 2 * TB) * G;
    l.plan_bytes = ((int64_t)c->n + 1) * 4;
    l.plan_bytes = (l.plan_bytes + 255) / 256 * 256;
    l.bytes = l.plan_bytes + 2 * l.grid * l.part_rows * (d + 2) * (int64_t)sizeof(float);
  }
  *out = l;
  return SHAHD_OK;
}

}  // namespace
}  // namespace shahd

extern "C" {

int shahd_prompt_attention(const ShahdPromptCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_prompt_attention";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  const int H = c->num_heads, Hk = c->kv_heads, d = c->head_dim;
  TaArgs a = {};
  if (!CheckType(op, c->dtype, false) || !CheckHeads(op, H, Hk, d) || !ScaleOf(op, c->scale, d, &a.scale_log2)) return SHAHD_EINVAL;
  if (c->n < 0 || c->rows < 0) {
    SetError("%s: need n, rows >= 0 (got n=%d rows=%d)", op, c->n, c->rows);
    return SHAHD_EINVAL;
  }
  if (!CheckRows(op, "q", c->q, c->rows, H, d, 8) || !CheckRows(op, "k", c->k, c->rows, Hk, d, 8) ||
      !CheckRows(op, "v", c->v, c->rows, Hk, d, 8) || !CheckRows(op, "out", c->out, c->rows, H, d, 8, true))
    return SHAHD_EINVAL;
  if (c->n == 0 || c->rows == 0) return SHAHD_OK;
  a.G = H / Hk;
  a.TB = 128 / a.G;
  const long long blocks = ((long long)c->rows / (2 * a.TB) + c->n) * Hk;
  if (blocks > kOpsMaxRows) {
    SetError("%s: too many rows and sequences (%d and %d)", op, c->rows, c->n);
    return SHAHD_EINVAL;
  }
  BufferCheck b(op);
  b.Add("offsets", c->offsets, 4);
  b.Add("q", c->q.data, 16);
  b.Add("k", c->k.data, 16);
  b.Add("v", c->v.data, 16);
  b.Add("out", c->out.data, 16);
  if (b.rc != SHAHD_OK) return b.rc;
  const DeviceInfo info = InfoOf(b.device);
  DeviceScope scope(b.device);
  if (!info.usable || !scope.ok) {
    SetError("%s: device %d is not a usable sm_100 device", op, b.device);
    return SHAHD_ENODEV;
  }
  if (!MakeRowMaps(op, c->dtype, d, H, Hk, c->rows, c->q, c->k, c->v, &a)) return SHAHD_ECUDA;
  a.out = static_cast<uint16_t*>(c->out.data);
  a.out_row = c->out.row_stride;
  a.out_head = c->out.head_stride;
  a.offsets = c->offsets;
  a.n = c->n;
  a.rows = c->rows;
  a.H = H;
  a.Hk = Hk;
  TakeLaunchError(nullptr);
  g_waiting_devices.Add(b.device);
  LaunchTiles<kPrompt>(d, c->dtype, a, (unsigned)blocks, static_cast<cudaStream_t>(stream));
  return LaunchStatus(op);
}

int64_t shahd_tree_attention_workspace(const ShahdTreeCall* c) {
  using namespace shahd;
  const char* op = "shahd_tree_attention_workspace";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  TreeLayout l;
  const int rc = LayTree(op, c, &l);
  return rc == SHAHD_OK ? l.bytes : rc;
}

int shahd_tree_attention(const ShahdTreeCall* c, void* stream) {
  using namespace shahd;
  const char* op = "shahd_tree_attention";
  ClearError();
  if (!c) {
    SetError("%s: null argument", op);
    return SHAHD_EINVAL;
  }
  TaArgs a = {};
  const int H = c->num_heads, Hk = c->cache.kv_heads, d = c->cache.head_dim;
  TreeLayout lay;
  const int rc = LayTree(op, c, &lay);
  if (rc != SHAHD_OK) return rc;
  if (!CheckType(op, c->dtype, false) || !ScaleOf(op, c->scale, d, &a.scale_log2)) return SHAHD_EINVAL;
  if (c->rows < 0) {
    SetError("%s: need rows >= 0 (got %d)", op, c->rows);
    return SHAHD_EINVAL;
  }
  if (!CheckRows(op, "q", c->q, c->rows, H, d, 8) || !CheckRows(op, "k", c->k, c->rows, Hk, d, 8) ||
      !CheckRows(op, "v", c->v, c->rows, Hk, d, 8) || !CheckRows(op, "out", c->out, c->rows, H, d, 8, true))
    return SHAHD_EINVAL;
  if (c->n == 0 || c->rows == 0) return SHAHD_OK;
  a.G = H / Hk;
  a.TB = 128 / a.G;
  if (((long long)c->rows * H + 7) / 8 > 0x7fffffffLL) {
    SetError("%s: too many rows and sequences (%d and %d)", op, c->rows, c->n);
    return SHAHD_EINVAL;
  }
  if (c->workspace_bytes < lay.bytes) {
    SetError("%s: needs %lld bytes of workspace, got %lld", op, (long long)lay.bytes, (long long)c->workspace_bytes);
    return SHAHD_EINVAL;
  }
  BufferCheck b(op);
  b.Add("offsets", c->offsets, 4);
  b.Add("lengths", c->lengths, 4);
  b.Add("masks", c->masks, 8);
  b.Add("q", c->q.data, 16);
  b.Add("k", c->k.data, 16);
  b.Add("v", c->v.data, 16);
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
  if (!MakeRowMaps(op, c->dtype, d, H, Hk, c->rows, c->q, c->k, c->v, &a)) return SHAHD_ECUDA;
  if (!MakeMap(c->dtype, c->cache.pool, d, (uint64_t)Hk * 2 * kOpsPage, c->cache.pages, d, c->cache.page_stride, kOpsPage, 1, &a.pool)) {
    SetError("%s: a tensor map of the cache could not be made", op);
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
  a.masks = reinterpret_cast<const unsigned long long*>(c->masks);
  a.lengths = c->lengths;
  a.table = c->cache.block_table;
  a.max_blocks = c->cache.max_blocks;
  a.pages = c->cache.pages;
  a.max_nodes = c->max_nodes;
  a.pairs = lay.pairs;
  a.least = lay.least;
  a.two_heads = lay.two_heads;
  if (lay.bytes > 0) {
    a.part_rows = lay.part_rows;
    a.plan = static_cast<int*>(c->workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(c->workspace) + lay.plan_bytes);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + 2 * lay.grid * lay.part_rows * d);
  }
  TakeLaunchError(nullptr);
  g_waiting_devices.Add(b.device);
  if (lay.least > 0) LaunchTiles<kTreeRanges>(d, c->dtype, a, (unsigned)lay.grid, static_cast<cudaStream_t>(stream));
  else LaunchTiles<kTreePairs>(d, c->dtype, a, (unsigned)lay.grid, static_cast<cudaStream_t>(stream));
  return LaunchStatus(op);
}

}  // extern "C"
