// Host side of the operators on caller-owned device buffers (rotary positions, packed prompt attention, tree
// attention, tree verification): argument checks, the device of the buffers, tensor maps, launch errors. The
// operators keep no state between calls: every buffer, the workspace included, is the caller's, so calls on
// different streams, devices or threads do not meet.
#pragma once

#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "../../include/shahd_b200.h"
#include "common.cuh"

namespace shahd {

constexpr int kOpsPage = 64;                     // positions of a cache page
constexpr uint32_t kOpsWaitLimit = 1u << 22;     // barrier probes before a wait gives up
constexpr int kOpsErrTimeout = 6;                // a bounded wait of the tile attention gave up

static __device__ int g_ops_device_error;  // 0, or the first kOpsErr* recorded on this device

inline size_t TypeBytes(int dtype) { return dtype == SHAHD_F32 ? 4 : 2; }

// The device of an address in a device's own memory; false for any other address, and where the driver cannot be asked: then the
// runtime is, which tells more and takes longer (0.39 us an address, the driver 0.03; a call has up to fourteen).
inline bool DeviceOfAddress(const void* p, int* device) {
  typedef CUresult (*Fn)(unsigned int, CUpointer_attribute*, void**, CUdeviceptr);
  static const Fn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<Fn>(f);
  }();
  if (!fn) return false;
  unsigned int type = 0;
  int ordinal = -1;
  CUpointer_attribute what[2] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
  void* to[2] = {&type, &ordinal};
  if (fn(2, what, to, reinterpret_cast<CUdeviceptr>(p)) != CUDA_SUCCESS) return false;
  if (type != CU_MEMORYTYPE_DEVICE || ordinal < 0) return false;
  *device = ordinal;
  return true;
}

// The device that every buffer of a call lives on. Add() takes the call's pointers one by one; a host pointer, an
// address that no allocation holds or a buffer of another device makes the call fail before anything is launched.
struct BufferCheck {
  const char* op;
  int device = -1;
  int rc = SHAHD_OK;
  explicit BufferCheck(const char* op_) : op(op_) {}
  void Add(const char* name, const void* p, size_t align) {
    if (rc != SHAHD_OK) return;
    if (!p) {
      SetError("%s: %s is null", op, name);
      rc = SHAHD_EINVAL;
      return;
    }
    if (reinterpret_cast<uintptr_t>(p) % align != 0) {
      SetError("%s: %s must be aligned to %zu bytes", op, name, align);
      rc = SHAHD_EINVAL;
      return;
    }
    int where = -1;
    if (!DeviceOfAddress(p, &where)) {
      cudaPointerAttributes at = {};
      const cudaError_t e = cudaPointerGetAttributes(&at, p);
      if (e != cudaSuccess) {
        cudaGetLastError();
        if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) {
          SetError("%s: no usable sm_100 device", op);
          rc = SHAHD_ENODEV;
        } else {
          SetError("%s: %s is not a device address (%s)", op, name, cudaGetErrorString(e));
          rc = SHAHD_EINVAL;
        }
        return;
      }
      if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
        SetError("%s: %s is not a device address", op, name);
        rc = SHAHD_EINVAL;
        return;
      }
      where = at.device;
    }
    if (device < 0) device = where;
    if (where != device) {
      SetError("%s: %s is on device %d, other buffers are on device %d", op, name, where, device);
      rc = SHAHD_EINVAL;
    }
  }
};

struct DeviceInfo {
  int sms = 0;
  bool usable = false;
};

// Multiprocessors of a device, and whether it is an sm_100 one; read once per device.
inline DeviceInfo InfoOf(int device) {
  static std::mutex mu;
  static DeviceInfo known[64];
  static bool have[64];
  if (device < 0 || device >= 64) return {};
  std::lock_guard<std::mutex> g(mu);
  if (!have[device]) {
    DeviceInfo d;
    int major = 0, minor = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) == cudaSuccess &&
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device) == cudaSuccess &&
        cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device) == cudaSuccess)
      d.usable = major == 10 && minor == 0;
    known[device] = d;
    have[device] = true;
  }
  return known[device];
}

// The call's launches: SHAHD_OK, or the first of them that failed.
inline int LaunchStatus(const char* op) {
  std::string what;
  const cudaError_t e = TakeLaunchError(&what);
  if (e == cudaSuccess) return SHAHD_OK;
  cudaGetLastError();
  SetError("%s: %s failed: %s", op, what.c_str(), cudaGetErrorString(e));
  return SHAHD_ECUDA;
}

inline bool CheckType(const char* op, int dtype, bool f32) {
  if (dtype == SHAHD_BF16 || dtype == SHAHD_F16 || (f32 && dtype == SHAHD_F32)) return true;
  SetError("%s: dtype must be SHAHD_BF16%s SHAHD_F16%s, got %d", op, f32 ? "," : " or", f32 ? " or SHAHD_F32" : "", dtype);
  return false;
}

// Rows and heads of an operand may lie in any order and distance; both strides are at least the head's extent
// where there is more than one of them. Rows of a result share no memory: either all heads of a row lie between it and the
// next, or all rows of a head. Row counts up to 2^30 leave 32-bit sums of a row and a step in range.
constexpr int64_t kOpsMaxRows = 1LL << 30;
inline bool CheckRows(const char* op, const char* name, const ShahdRows& r, int64_t rows, int heads, int d, int multiple, bool result = false) {
  if (rows > kOpsMaxRows) {
    SetError("%s: too many rows: %lld, at most 2^30", op, (long long)rows);
    return false;
  }
  if ((rows > 1 && r.row_stride < d) || (heads > 1 && r.head_stride < d) || r.row_stride < 0 || r.head_stride < 0) {
    SetError("%s: %s needs row and head strides of at least head_dim %d elements (got %lld and %lld)", op, name, d,
             (long long)r.row_stride, (long long)r.head_stride);
    return false;
  }
  if (r.row_stride > (1LL << 36) || r.head_stride > (1LL << 36)) {
    SetError("%s: %s has a stride beyond 2^36 elements", op, name);
    return false;
  }
  if (result && rows > 1 && heads > 1 && (double)r.row_stride < (heads - 1) * (double)r.head_stride + d &&
      (double)r.head_stride < (rows - 1) * (double)r.row_stride + d) {
    SetError("%s: rows and heads of %s share memory (strides %lld and %lld)", op, name, (long long)r.row_stride, (long long)r.head_stride);
    return false;
  }
  if ((rows > 1 && r.row_stride % multiple != 0) || (heads > 1 && r.head_stride % multiple != 0)) {
    SetError("%s: %s needs strides that are multiples of %d elements (got %lld and %lld)", op, name, multiple,
             (long long)r.row_stride, (long long)r.head_stride);
    return false;
  }
  return true;
}

inline bool CheckCache(const char* op, const ShahdKvCache& c, int kv_heads, int d) {
  if (c.kv_heads != kv_heads || c.head_dim != d) {
    SetError("%s: the cache holds %d kv heads of head_dim %d, the call has %d of %d", op, c.kv_heads, c.head_dim, kv_heads, d);
    return false;
  }
  const int64_t page = (int64_t)kv_heads * 2 * kOpsPage * d;
  if (c.pages < 1 || c.max_blocks < 1 || c.max_blocks > (1 << 24) || c.page_stride < page || c.page_stride % 8 != 0 ||
      c.page_stride > (1LL << 36)) {
    SetError("%s: the cache needs pages and max_blocks >= 1 and a page_stride of at least %lld elements that is a multiple "
             "of 8 (got pages=%d max_blocks=%d page_stride=%lld)",
             op, (long long)page, c.pages, c.max_blocks, (long long)c.page_stride);
    return false;
  }
  return true;
}

}  // namespace shahd
