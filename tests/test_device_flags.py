"""Error flags of several devices (csrc/device_flags.h) on the host: the first that is set, whichever device is current; one that
cannot be read is reported. The operators' calls on another device than the current one leave that one current."""
import ctypes
import os
import shutil
import subprocess

import pytest

from tests.helpers import pkg

SOURCE = r"""
#include "device_flags.h"
static unsigned long long asked;  // bits of the devices whose flags were read
extern "C" int first(const int* devices, int n, const int* held) {
  shahd::DeviceSet set;
  for (int i = 0; i < n; i++) set.Add(devices[i]);
  asked = 0;
  return shahd::FirstFlag(set, [&](int device, int* flag) {
    asked |= 1ull << device;
    if (held[device] == -7) return false;
    *flag = held[device];
    return true;
  });
}
extern "C" unsigned long long asked_for() { return asked; }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("needs g++")
    at = tmp_path_factory.mktemp("flags")
    (at / "flags.cc").write_text(SOURCE)
    csrc = os.path.join(os.path.dirname(pkg.__file__), "csrc")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", csrc, "-o", str(at / "flags.so"), str(at / "flags.cc")], check=True)
    lib = ctypes.CDLL(str(at / "flags.so"))
    lib.asked_for.restype = ctypes.c_ulonglong
    return lib


@pytest.mark.parametrize("devices,held,want", [
    ([], {0: 6}, 0),
    ([0], {0: 0, 1: 6}, 0),
    ([1], {1: 6}, 6),          # on a device that is not the first
    ([0, 63], {63: 6}, 6),
    ([0, 1, 2], {1: -7, 2: 6}, -1),  # cannot be read
    ([2, 1, 1], {1: 5, 2: 6}, 5),
])
def test_first_flag(lib, devices, held, want):
    values = (ctypes.c_int * 64)(*[held.get(i, 0) for i in range(64)])
    assert lib.first((ctypes.c_int * max(1, len(devices)))(*devices), len(devices), values) == want
    assert lib.asked_for() & ~sum(1 << d for d in set(devices)) == 0  # no other device is touched


@pytest.mark.gpu
def test_flag_of_another_device_than_the_current_one():
    torch = pytest.importorskip("torch")
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    q = torch.randn(90, 4, 64, device="cuda:1").bfloat16()
    out, off = torch.empty_like(q), torch.tensor([0, 90], dtype=torch.int32, device="cuda:1")
    torch.cuda.synchronize(1)
    rows = lambda t: pkg.Rows(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    with torch.cuda.device(0):
        pkg.prompt_attention(pkg.BF16, rows(q), rows(q), rows(q), rows(out), off.data_ptr(), 1, 90, 4, 4, 64)
        torch.cuda.synchronize(1)
        assert pkg.load().ShahdDeviceErrorFlag() == 0 and torch.cuda.current_device() == 0
