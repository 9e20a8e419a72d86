"""The feature cache and the linear layer without a GPU: what is refused before any device work, the plain forms of their tests."""
import ctypes as C
import os
import re

import pytest
import torch

import rows_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rmr():
    import rm_radar_amd
    from rm_radar_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return rm_radar_amd


def test_creation_refusals(rmr):
    from rm_radar_amd import _lib
    L, bad = _lib.lib(), rmr.InvalidArgument
    h = C.c_void_p()
    for slots, width in ((0, 8), (-1, 8), (2 ** 41, 8), (8, 0), (8, -3), (8, 65537)):
        with pytest.raises(bad):
            _lib.check(L.rmr_feature_cache_create(0, slots, width, C.byref(h)))
    w = torch.zeros(4, 6)
    for k, n, fmt, act in ((0, 4, 0, 0), (6, 0, 0, 0), (65537, 4, 0, 0), (6, 4, 3, 0), (6, 4, -1, 0), (6, 4, 0, 5), (6, 4, 0, -1)):
        with pytest.raises(bad):
            _lib.check(L.rmr_linear_create(C.byref(_lib.LinearCfg(0, k, n, fmt, act)), w.data_ptr(), 2, 6, None, 0, None, C.byref(h)))
    good = _lib.LinearCfg(0, 6, 4, 0, 0)
    for args in ((None, w.data_ptr(), 2, 6, None, 0), (good, None, 2, 6, None, 0), (good, w.data_ptr(), 3, 6, None, 0), (good, w.data_ptr(), 2, 5, None, 0),
                 (good, w.data_ptr() + 2, 2, 6, None, 0), (good, w.data_ptr(), 2, 6, w.data_ptr() + 2, 0), (good, w.data_ptr(), 2, 6, None, 2)):
        with pytest.raises(bad):
            _lib.check(L.rmr_linear_create(C.byref(args[0]) if args[0] is not None else None, *args[1:], None, C.byref(h)))
    assert not h.value


def test_null_handles(rmr):
    from rm_radar_amd import _lib
    L, bad = _lib.lib(), rmr.InvalidArgument
    n = C.c_size_t()
    call = _lib.LinearCall()
    for status in (lambda: L.rmr_feature_cache_write(None, None, 0, 0, None, 0, None), lambda: L.rmr_feature_cache_read(None, None, 0, None, 0, 0, None),
                   lambda: L.rmr_linear_run(None, C.byref(call), None), lambda: L.rmr_linear_run_kept(None, None, None, C.byref(call), None),
                   lambda: L.rmr_linear_workspace(None, C.byref(call), 0, C.byref(n)), lambda: L.rmr_linear_workspace(None, C.byref(call), 0, None),
                   lambda: L.rmr_detector_keep_feature(None, b"model.21", 0, None, 0)):
        with pytest.raises(bad):
            _lib.check(status())
    assert L.rmr_feature_cache_bytes(None) == 0
    L.rmr_feature_cache_destroy(None)
    L.rmr_linear_destroy(None)


def test_python_refusals_before_the_library(rmr):
    w = torch.zeros(4, 6)
    for bad in (dict(weight=w, format="f8"), dict(weight=w, activation="tanh"), dict(weight=w[0]), dict(weight=w, bias=torch.zeros(3))):
        with pytest.raises(rmr.InvalidArgument):
            rmr.Linear(**bad)
    layer = object.__new__(rmr.Linear)       # as a handle would be: the tensors are looked at first
    layer.in_features, layer.out_features, layer.device = 6, 4, 0
    cache = object.__new__(rmr.FeatureCache)
    cache.width, cache.slots, cache.device = 6, 9, 0
    for call in (lambda: layer(torch.zeros(2, 6)), lambda: layer(torch.zeros(2, 6, dtype=torch.int32)), lambda: layer.kept(cache, torch.zeros(2, dtype=torch.int64)),
                 lambda: layer.kept(cache, torch.zeros(2)), lambda: cache.write(torch.zeros(2, 6), torch.zeros(2, dtype=torch.int64)),
                 lambda: cache.read(torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(rmr.InvalidArgument):
            call()


def test_constants_agree_with_the_header(rmr):
    from rm_radar_amd import _lib, rows
    text = open(os.path.join(ROOT, "include", "rmr.h")).read()
    value = lambda name: int(re.search(rf"\b{name}\s*=?\s*(\d+)", text).group(1))  # noqa: E731
    assert value("RMR_LINEAR_FEW_ROWS") == _lib.LINEAR_FEW_ROWS
    assert {k: value(f"RMR_LINEAR_{k.upper()}") for k in rows._FORMATS} == rows._FORMATS
    assert {k: value(f"RMR_ACT_{k.upper()}") for k in rows._ACTIVATIONS} == rows._ACTIVATIONS
    assert C.sizeof(_lib.LinearCall) == 88 and C.sizeof(_lib.LinearCfg) == 20


def test_the_held_form_rounds_to_the_nearest_of_its_values():
    """rows_ref.held against a search over all e4m3 values."""
    e4m3 = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double()
    e4m3 = e4m3[torch.isfinite(e4m3)].unique()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 32, generator=g) * torch.exp2(torch.randint(-30, 30, (40, 1), generator=g).float())
    x[0] = 0
    h = ref.held(x)
    for row, got in zip(x.double(), h):
        top = row.abs().max()
        e = -127
        while top > 448 * 2.0 ** e:
            e += 1
        grid = e4m3 * 2.0 ** e
        best = (row[:, None] - grid[None]).abs().min(1).values
        assert torch.equal((row - got).abs(), best) and bool(torch.isin(got, grid).all())
