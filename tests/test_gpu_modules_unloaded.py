"""Kernel modules that come and go: what a process keeps about kernels and memory does not go with the module that was first to need it, and a module gets answers of its own
although its kernels lie where another's were."""
import subprocess
import sys
from pathlib import Path

import pytest

import mlir_fixtures as F

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import gc, shutil, sys
import numpy as np
sys.path.insert(0, {root!r})
import __graft_entry__ as entry
pkg = entry.load_package()
dev = pkg.hal.CudaSm100Device(0)
s = dev.create_stream()
x = np.arange(1, 2 * 512 + 1, dtype=np.float32).reshape(2, 512)
a = np.zeros((256, 256), np.uint16)
a[np.arange(256), np.arange(256)] = 0x3f80  # bf16 ones
b = np.full((256, 256), 0x4000, np.uint16)  # twos
xb, ab, bb = (dev.alloc_from_slice(t, s) for t in (x, a, b))
yb, cb = dev.alloc(x.size, np.float32), dev.alloc(256 * 256, np.uint16)
want = x / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
for turn in range(4):  # the module is the first to ask, and is unloaded; a copy then has its place
    path = {so!r}.replace(".so", f"_{{turn}}.so")
    shutil.copy({so!r}, path)
    launcher = dev.create_launcher()
    launcher.load(path, pkg.hal.KernelMode.Vector)
    launcher.launch("rms_tiles", pkg.hal.LaunchGrid.blocks_(1), [xb.as_raw_ptr(), yb.as_raw_mut_ptr()], s)
    assert np.abs(yb.copy_to_host(s).reshape(x.shape) / want - 1).max() < 1e-5
    launcher.launch("mm_tiles", pkg.hal.LaunchGrid.blocks_(1), [ab.as_raw_ptr(), bb.as_raw_ptr(), cb.as_raw_mut_ptr()], s)
    assert (cb.copy_to_host(s) == 0x4000).all()
    if turn:
        dev.rms_norm(pkg.capi.F32, 2, 512, 1e-6, xb.as_raw_ptr(), yb.as_raw_mut_ptr(), stream=s.raw)
        assert np.abs(yb.copy_to_host(s).reshape(x.shape) / want - 1).max() < 1e-5
    s.synchronize()
    del launcher
    gc.collect()
assert dev.status(s) == 0
print("done")
"""


def test_modules_come_and_go(pkg, tmp_path):
    parts = [F.rms_norm("rms_tiles", 2, 512, eps="1.0e-6"), F.matmul("mm_tiles", 256, 256, 256, dt="bf16")]
    mlir = parts[0].rsplit("}", 1)[0] + parts[1].split("module {", 1)[1].rsplit("}", 1)[0] + "}\n"
    out = pkg.codegen.CudaSm100Target().emit(mlir)
    so = pkg.build.build_module(out.source, tmp_path / "module.so")
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(root=str(ROOT), so=str(so))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stdout, r.stderr[-3000:])
