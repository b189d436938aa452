"""The launches that a library's host code makes, without running them: the source compiled for the CPU with a launch
that only records its grid. For sizes whose memory or time no test can have."""

import ctypes
import os
import shutil
import subprocess

import pytest

import _emu

RECORDER = """
#include <hip/hip_runtime.h>
static unsigned long long recorded[64][4];
static int launches = 0;
static void record(dim3 grid, dim3 block) {
  unsigned long long* r = recorded[launches++ % 64];
  r[0] = grid.x, r[1] = grid.y, r[2] = grid.z, r[3] = (unsigned long long)block.x * block.y * block.z;
}
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(K, G, B, SH, ST, ...) record(dim3(G), dim3(B))
extern "C" __attribute__((visibility("default"))) int recorded_launches() { return launches; }
extern "C" __attribute__((visibility("default"))) unsigned long long recorded_launch(int n, int what) {
  return recorded[n % 64][what];
}
"""


def build(tmpdir, source):
    """csrc/<source> as a shared library whose launches are recorded; launches(lib) tells of them."""
    clang = _emu._clang()
    if clang is None:
        pytest.skip("clang++ (for the kernels' vector extensions on the host) is missing")
    kern = _emu.kernel_source(tmpdir, source)
    for name in ("matrix.hpp", "fp4.hpp"):
        shutil.copy(os.path.join(_emu.EMU, name), os.path.join(str(tmpdir), name))
    with open(kern) as f:
        text = f.read()
    with open(kern, "w") as f:
        f.write(RECORDER + text)
    out = os.path.join(str(tmpdir), "librecorded.so")
    proc = subprocess.run([clang, "-std=c++17", "-O1", "-fPIC", "-shared", "-U_FORTIFY_SOURCE", "-D_FORTIFY_SOURCE=0",
                           "-fno-strict-aliasing", "-w", "-pthread", "-I", _emu.EMU, "-I", str(tmpdir), kern, "-o",
                           out], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-4000:]
    lib = ctypes.CDLL(out)
    lib.recorded_launch.restype = ctypes.c_ulonglong
    return lib


def launches(lib, call):
    """call()'s return code and the (grid x, y, z, threads of a workgroup) of the launches that it made."""
    before = lib.recorded_launches()
    code = call()
    made = range(before, lib.recorded_launches())
    return code, [tuple(int(lib.recorded_launch(n, w)) for w in range(4)) for n in made]


def accepted(grid):
    """Whether the device takes this launch: fewer than 2^32 threads in x, at most 65535 workgroups in y and in z."""
    x, y, z, threads = grid
    return 1 <= x and x * threads < 1 << 32 and 1 <= y <= 65535 and 1 <= z <= 65535
