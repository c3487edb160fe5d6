// Host side of the tile attention: tensor maps and checks that its operators share.
#pragma once

#include "device_flags.h"
#include "tile_attention.cuh"

namespace shahd {

constexpr int kTaSms = 148;  // of a B200: the layout of a call's work, and so its workspace, does not hang on a device being there

// The operators run where their buffers are, so a wait that gave up may have been recorded on any device that a kernel with waits
// (the tile attention) has been launched on. Each translation unit has a flag and a set of its own.
static DeviceSet g_waiting_devices;

static int TileDeviceError() {
  return FirstFlag(g_waiting_devices, [](int device, int* flag) {
    DeviceScope scope(device);
    if (scope.ok && cudaMemcpyFromSymbol(flag, g_ops_device_error, sizeof *flag) == cudaSuccess) return true;
    cudaGetLastError();
    return false;
  });
}

typedef CUresult (*OpsEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline OpsEncodeFn OpsEncode() {
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
inline bool MakeMap(int dtype, const void* p, uint64_t nx, uint64_t ny, uint64_t nz, int64_t sy, int64_t sz, int by, int bz, CUtensorMap* m) {
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

inline bool CheckHeads(const char* op, int H, int Hk, int d) {
  if (H >= 1 && Hk >= 1 && H % Hk == 0 && H / Hk <= 8 && H <= (1 << 16) && (d == 32 || d == 64 || d == 128)) return true;
  SetError("%s: need kv_heads dividing num_heads with at most 8 query heads per kv head and head_dim 32, 64 or 128 (got "
           "num_heads=%d kv_heads=%d head_dim=%d)", op, H, Hk, d);
  return false;
}

inline bool ScaleOf(const char* op, double scale, int d, float* log2) {
  if (scale == 0) scale = 1.0 / std::sqrt((double)d);
  *log2 = (float)(scale * M_LOG2E);
  if (!(*log2 > 0) || !std::isfinite(*log2)) {  // in 32 bits, too: masked scores are -inf times it
    SetError("%s: scale must be positive and finite in 32 bits, or 0 for 1/sqrt(head_dim) (got %g)", op, scale);
    return false;
  }
  return true;
}

}  // namespace shahd
