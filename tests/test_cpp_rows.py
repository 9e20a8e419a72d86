"""include/radar/rows.h compiles with g++ -std=c++20, throws without a GPU, and gives the ctypes path's bytes with one."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "rm_radar_amd", "_build")
EXE = os.path.join(LIBDIR, "api_rows")


def _build():
    if not os.path.exists(os.path.join(LIBDIR, "librmr.so")):
        import __graft_entry__ as g
        g.build()
    subprocess.check_call(["g++", "-std=c++20", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I/opt/rocm/include",
                           os.path.join(ROOT, "tests", "cpp", "api_rows.cpp"), "-L", LIBDIR, "-lrmr", "-L/opt/rocm/lib", "-lamdhip64",
                           f"-Wl,-rpath,{LIBDIR}", "-Wl,-rpath,/opt/rocm/lib", "-o", EXE])


def test_compiles_and_throws_without_gpu():
    _build()
    import rm_radar_amd as r
    if r.device_count() > 0:
        pytest.skip("a GPU is present: covered by the gpu test")
    res = subprocess.run([EXE], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "api_rows ok" in res.stdout, res.stdout + res.stderr


@pytest.mark.gpu
def test_equals_the_ctypes_path(tmp_path):
    import torch

    import rm_radar_amd as rmr
    _build()
    rng = np.random.default_rng(5)
    x, w1, b1, w2 = (rng.standard_normal(s).astype(np.float32) for s in ((70, 200), (96, 200), (96,), (40, 96)))
    with open(tmp_path / "in.bin", "wb") as f:
        for a in (x, w1, b1, w2):
            f.write(a.tobytes())
    res = subprocess.run([EXE, str(tmp_path / "in.bin"), str(tmp_path / "out.bin")], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "api_rows ran" in res.stdout, res.stdout + res.stderr
    got = np.fromfile(tmp_path / "out.bin", np.float32)
    slots = torch.tensor([(i * 37) % 101 for i in range(70)]).cuda()
    cache = rmr.FeatureCache(101, 200)
    cache.write(torch.from_numpy(x).cuda(), slots)
    mid = rmr.Linear(w1, b1, activation="silu", format="mx8").kept(cache, slots, out_dtype=torch.float32)
    out = rmr.Linear(w2, format="mx8")(mid)
    assert got.tobytes() == mid.cpu().numpy().tobytes() + out.cpu().numpy().tobytes()
