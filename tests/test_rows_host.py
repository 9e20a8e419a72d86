"""Host code of the feature cache and the linear layer on a stand-in HIP runtime of two devices (cpp/fake_hip.cpp): which device is
current or waited for, what is refused and what is not.  No GPU takes part, kernels do nothing."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PRELUDE = """
import ctypes as C, os, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)          # before librmr.so: its calls go here
fake.fake_hip_synced.restype = fake.fake_hip_launches.restype = fake.fake_hip_priority_streams.restype = C.c_long
sys.path[:0] = [sys.argv[2], os.path.join(sys.argv[2], "tests")]
import numpy as np
import rm_radar_amd as rmr
from rm_radar_amd import _lib
L, OK, BAD = _lib.lib(), _lib.OK, _lib.ERR_INVALID_ARGUMENT
assert rmr.device_count() == 2

def current():
    d = C.c_int()
    fake.hipGetDevice(C.byref(d))
    return d.value

def cache(slots, width, device=0):
    h = C.c_void_p()
    return L.rmr_feature_cache_create(device, slots, width, C.byref(h)), h

def layer(k, n, fmt=0, device=0):
    h, w = C.c_void_p(), np.zeros((n, k), np.float32)
    return L.rmr_linear_create(C.byref(_lib.LinearCfg(device, k, n, fmt, 0)), w.ctypes.data, 2, k, None, 0, None, C.byref(h)), h
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    import __graft_entry__ as g
    from rm_radar_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        g.build()
    so = str(tmp_path_factory.mktemp("fake") / "libfakehip.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                           os.path.join(ROOT, "tests", "cpp", "fake_hip.cpp"), "-o", so])
    return so


def run(fake, body, *args, **env):
    res = subprocess.run([sys.executable, "-c", PRELUDE + body, fake, ROOT, *args], capture_output=True, text=True, timeout=300,
                         env={**os.environ, **env})
    assert res.returncode == 0, res.stdout + res.stderr


def test_creation_leaves_the_callers_device(fake):
    run(fake, """
for mine, other in ((0, 1), (1, 0)):
    fake.hipSetDevice(mine)
    for device in (mine, other, other, 7):       # the first handle of a device, a further one, a device that is not there
        for make in (lambda: cache(9, 40, device), lambda: layer(40, 9, 0, device), lambda: layer(40, 9, 2, device)):
            status, h = make()
            assert status == (OK if device < 2 else BAD) and current() == mine, (mine, device, status, current())
    h = cache(9, 40, other)[1]
    L.rmr_feature_cache_destroy(h)
    assert current() == mine
""")


def test_keep_feature_waits_for_the_detectors_device(fake, tmp_path):
    run(fake, """
import netutil
from rm_radar_amd import weights as W
pack = W.make_synthetic_pack(sys.argv[3], "s", 1, seed=3)
det = rmr.Detector(pack, 1, (160, 160), 1, device=1, input_width=160, input_height=160)
det.infer([netutil.test_image(0, 160, 160)])
h, w, c = det.read_feature("model.21", 0).shape
store = rmr.FeatureCache(h * w, c, device=1)
fake.hipSetDevice(0)
before = [fake.fake_hip_synced(d) for d in range(2)]
det.keep_feature("model.21", store, 0)
assert [fake.fake_hip_synced(d) for d in range(2)] == [before[0], before[1] + 1]
assert current() == 0
""", str(tmp_path / "car.rmrw"), RMR_ARENA_REUSE="0")


def test_the_workspace_query_reads_no_workspace(fake):
    run(fake, """
h = layer(203, 96)[1]
x, y, r = (np.zeros((400, 203), np.float16), np.zeros((400, 96), np.float16), np.zeros((400, 96), np.float16))
need, again = C.c_size_t(), C.c_size_t()
call = _lib.LinearCall(x.ctypes.data, 0, 203, 400, r.ctypes.data, 96, y.ctypes.data, 0, 96, None, 0)
assert L.rmr_linear_workspace(h, C.byref(call), 0, C.byref(need)) == OK and need.value > 0
for stale in (x, y, r):                         # what an earlier call may have left there
    call.workspace, call.workspace_bytes = stale.ctypes.data, 1 << 40
    assert L.rmr_linear_workspace(h, C.byref(call), 0, C.byref(again)) == OK and again.value == need.value
    assert L.rmr_linear_run(h, C.byref(call), None) == BAD
    call.workspace_bytes = need.value
    assert L.rmr_linear_run(h, C.byref(call), None) == BAD
space = np.zeros(need.value // 16 + 1, np.complex128)
call.workspace = space.ctypes.data
assert L.rmr_linear_run(h, C.byref(call), None) == OK
""")


def test_rows_that_span_more_than_an_address_are_refused(fake):
    """(rows - 1) * pitch * element size past 2^63: the operands' ranges could not be compared."""
    run(fake, """
rows, far = (1 << 30) + 2, 1 << 31
h, store = layer(8, 16)[1], cache(4, 8)[1]
p, q = 1 << 44, 1 << 45                        # addresses that nobody follows
for at in ((8, 16, far, 0), (8, 16, 16, far)):
    ldx, ldy, wide = at[0], at[2], at[3]
    call = _lib.LinearCall(p, 0, ldx, rows, q if wide else None, wide, q, 2, ldy, None, 0)
    before = fake.fake_hip_launches()
    assert L.rmr_linear_run(h, C.byref(call), None) == BAD and fake.fake_hip_launches() == before
    assert b"elements apart" in L.rmr_last_error(), L.rmr_last_error()
call = _lib.LinearCall(p, 0, far, (1 << 31) - 1, None, 0, q, 2, 16, None, 0)
assert L.rmr_linear_run(h, C.byref(call), None) == BAD and b"elements apart" in L.rmr_last_error()
assert L.rmr_feature_cache_write(store, p, 2, far, q, rows, None) == BAD and b"elements apart" in L.rmr_last_error()
assert L.rmr_feature_cache_read(store, q, rows, p, 2, far, None) == BAD and b"elements apart" in L.rmr_last_error()
assert L.rmr_feature_cache_read(store, q, 2, p, 2, far, None) == OK
""")


def test_overlap_goes_by_the_rows_not_by_what_lies_between(fake):
    """y against x, the residual and the workspace, compared with the sets of bytes: columns of one buffer are apart.  Operands inside
    each other's span at different pitches may be refused, but none that overlaps may pass."""
    run(fake, """
import random
rng = random.Random(11)
layers = {(k, n): layer(k, n)[1] for k in (8, 24) for n in (5, 16)}
base = 1 << 44

def taken(p, rows, width, ld):
    return {p + 2 * (i * ld + j) for i in range(rows) for j in range(width)}

seen = {True: 0, False: 0, "unsure": 0}
for turn in range(6000):
    (k, n), h = rng.choice(list(layers.items()))
    rows = rng.choice((1, 2, 3, 7))
    ldy = n + rng.choice((0, 1, 24, 40))
    same = rng.random() < 0.7
    other = rng.choice(("x", "residual", "workspace"))
    y = base + 2 * rng.randrange(0, 120)
    far = base + (1 << 20)
    p = base + 2 * rng.randrange(0, 120)
    x, ldx, r, ldr, ws, ws_bytes, single = far, k, None, 0, None, 0, rows == 1
    if other == "x":
        ldx = ldy if same else rng.choice((0, 3, k, k + 9))
        x, them, single = p, taken(p, rows, k, ldx), single or ldx <= k
    elif other == "residual":
        ldr = ldy if same else rng.choice((0, 2, n, n + 7))
        r, them, single = p, taken(p, rows, n, ldr), single or ldr <= n
        if r == y and (rows == 1 or ldr == ldy):
            them = set()                       # the residual may be y
    else:
        p -= p % 16
        size = rng.choice((16, 64, 400))
        ws, ws_bytes, them, single = p, size, taken(p, 1, size // 2, 0), True
    meets = bool(them & taken(y, rows, n, ldy))
    call = _lib.LinearCall(x, 0, ldx, rows, r, ldr, y, 0, ldy, ws, ws_bytes)
    status = L.rmr_linear_run(h, C.byref(call), None)
    sure = single or ldy == n or (ldx if other == "x" else ldr) == ldy
    if meets or sure:
        assert status == (BAD if meets else OK), (turn, other, rows, k, n, ldx, ldr, ldy, p - base, y - base, meets, L.rmr_last_error())
        seen[meets] += 1
    else:
        assert status in (OK, BAD)
        seen["unsure"] += 1
assert min(seen.values()) > 20, seen
# slots between the rows of an output that is written: 16 bytes of every 64, four slots are 32 bytes
store = cache(9, 8)[1]
for at in range(0, 256, 8):
    want = BAD if {*range(at, at + 32)} & {i * 64 + j for i in range(4) for j in range(16)} else OK
    assert L.rmr_feature_cache_read(store, base + at, 4, base, 0, 32, None) == want, at
""")


def test_every_stream_has_the_default_priority(fake, tmp_path):
    """Streams of different priorities at work beside each other have hung."""
    run(fake, """
import scenes
from rm_radar_amd import weights as W
cars = W.make_synthetic_pack(sys.argv[3] + "/car.rmrw", "s", 1, seed=3)
armors = W.make_synthetic_pack(sys.argv[3] + "/armor.rmrw", "s", 12, seed=4)
kept = [rmr.RobotDetector(cars, armors, (160, 160), 12, max_cars=2, opt_cars=2),
        rmr.Locator(640, 640, scenes.K640, scenes.SAMPLE_L2C, np.eye(4, dtype=np.float32)), rmr.UploadRing(1, 4096), rmr.FeatureCache(4, 8)]
assert layer(8, 16)[0] == OK
assert fake.fake_hip_priority_streams() == 0
""", str(tmp_path))
