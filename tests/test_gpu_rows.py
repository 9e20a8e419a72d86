"""The feature cache and the linear layer on the GPU, against plain forms in 64 bits (rows_ref.py)."""
import numpy as np
import pytest
import torch

import rows_ref as ref

pytestmark = pytest.mark.gpu

KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def rmr():
    import rm_radar_amd
    assert rm_radar_amd.device_count() >= 1
    return rm_radar_amd


def make(rows, width, kind, seed, pad=0, offset=0, scale=1.0):
    """[rows, width] of `kind` on the GPU, rows width + pad elements apart, the first one `offset` elements into its storage."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width + pad, generator=g) * scale
    x = x * torch.exp2(torch.randint(-4, 5, (rows, 1), generator=g).float())
    flat = torch.empty(offset + x.numel(), dtype=KINDS[kind], device="cuda")
    flat[offset:] = x.reshape(-1).to(KINDS[kind]).cuda()
    return flat[offset:].view(rows, width + pad)[:, :width]


# ---------------------------------------------------------------------------------------------------------------- cache

@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,width,pad,offset", [(1, 1, 0, 0), (50, 1, 0, 0), (70, 3, 2, 1), (300, 4, 0, 0), (300, 8, 1, 0), (90, 9, 0, 0), (1, 576, 0, 0), (3, 31, 1, 1), (5, 33, 0, 3), (64, 128, 0, 0), (400, 576, 8, 0),
                                                (17, 1001, 3, 5), (4097, 40, 0, 0), (6001, 257, 1, 0), (2, 65536, 0, 0)])
def test_cache_write_and_read(rmr, kind, n, width, pad, offset):
    cap = n + 13
    cache = rmr.FeatureCache(cap, width)
    x = make(n, width, kind, 1, pad, offset)
    slots = torch.randperm(cap, generator=torch.Generator().manual_seed(2))[:n].cuda()
    cache.write(x, slots)
    want = ref.held(x)
    for out in ("f16", "bf16", "f32"):
        room = torch.full((n, width), float("nan"), dtype=KINDS[out], device="cuda")
        assert torch.equal(cache.read(slots, out=room).cpu(), want.to(KINDS[out])), out
    rest = torch.ones(cap, dtype=torch.bool)
    rest[slots.cpu()] = False
    other = torch.arange(cap)[rest].cuda()
    assert (cache.read(other, dtype=torch.float32) == 0).all()   # a new cache holds zeros, slots that were not named keep them


@pytest.mark.parametrize("n", [50, 4096, 4097, 20000])
def test_cache_slots_twice_and_missing(rmr, n):
    """The last row of a slot stays, rows without a slot are left out, a read of a missing slot is zeros."""
    cap, width = n // 2 + 3, 96
    g = torch.Generator().manual_seed(n)
    slots = torch.randint(-3, cap + 3, (n,), generator=g)
    slots[1] = 2 ** 40
    slots[2] = -(2 ** 62)
    cache = rmr.FeatureCache(cap, width)
    first = make(cap, width, "f32", 3)
    cache.write(first, torch.arange(cap).cuda())
    x = make(n, width, "f32", 4)
    for _ in range(2):   # the same again leaves the same
        cache.write(x, slots.cuda())
        want = ref.held(first)
        rows = ref.held(x)
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < cap:
                want[s] = rows[i]
        assert torch.equal(cache.read(torch.arange(cap).cuda(), dtype=torch.float32).cpu().double(), want)
    assert torch.equal(cache.read(slots.cuda(), dtype=torch.float32).cpu().double(), ref.pick(want, slots, cap))


def test_cache_extreme_values(rmr):
    """Infinities and NaN are held as NaN and leave their block's scale alone; the type's largest and smallest values; zeros."""
    x = torch.zeros(12, 64)
    x[0, 3], x[0, 40] = float("inf"), 1.0
    x[1, :] = float("nan")
    x[2, 0], x[2, 1], x[2, 2] = float("-inf"), 3.0e38, -448.0
    x[3, :32], x[3, 32:] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny
    x[4, :] = 2.0 ** -149
    x[5, 0], x[5, 1] = 2.0 ** -126, 2.0 ** -140
    x[6, 0], x[6, 1:] = 448.0, torch.linspace(-448, 448, 63)
    x[7, 0], x[7, 1:] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9)), torch.linspace(-448, 448, 63)
    x[8, :] = torch.linspace(0, 2.0 ** -5, 64)
    x[8, 0] = 448.0
    x[9, :] = torch.arange(64) * 0.0625 + 1   # ties
    x[9, 31] = x[9, 63] = 448.0
    x[10, :] = -0.0
    cache = rmr.FeatureCache(12, 64)
    s = torch.arange(12).cuda()
    cache.write(x.cuda(), s)
    got, want = cache.read(s, dtype=torch.float32).cpu(), ref.held(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    # (the largest f32 is held as 2^128, which reads back as the f32 it rounds to: infinity)
    assert torch.equal(got.nan_to_num(7.0, posinf=9.0), want.float().nan_to_num(7.0, posinf=9.0))
    # half a step of e4m3 relative to the value, or half of the block's smallest step
    fin = torch.isfinite(x)
    top = torch.where(fin, x.abs(), torch.zeros(())).reshape(12, 2, 32).amax(2).repeat_interleave(32, 1).double()
    assert (((want - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + torch.clamp(top * 2 / 448, min=2.0 ** -127) * 2.0 ** -10) | ~fin).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["counted", "mixed", "magnitude"])
def test_cache_every_16_bit_value(rmr, kind, order):
    """All 65536 bit patterns, in blocks of neighbours, of anything beside anything, and of neighbours next to one larger value."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    if order == "mixed":
        bits = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(9))]
    x = bits.view(KINDS[kind]).reshape(-1, 32).clone()
    if order == "magnitude":
        top = torch.where(torch.isfinite(x), x.abs().float(), torch.zeros(())).amax(1)
        x[:, 0] = (top * torch.exp2((torch.arange(len(x)) % 12).float())).clamp_max(6e4).to(x.dtype)
    cache = rmr.FeatureCache(len(x), 32)
    s = torch.arange(len(x)).cuda()
    cache.write(x.cuda(), s)
    got, want = cache.read(s, dtype=torch.float32).cpu(), ref.held(x).float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(7.0, posinf=9.0, neginf=8.0), want.nan_to_num(7.0, posinf=9.0, neginf=8.0))


def test_cache_beyond_32_bits(rmr):
    """Slots whose byte offset passes 2^32."""
    slots, width = 1100000, 4096
    cache = rmr.FeatureCache(slots, width)
    assert cache.nbytes() > 2 ** 32
    s = torch.tensor([0, 524287, 524288, 1048575, 1048576, 1048577, slots - 1]).cuda()
    x = make(7, width, "bf16", 5)
    cache.write(x, s)
    assert torch.equal(cache.read(s, dtype=torch.bfloat16).cpu(), ref.held(x).to(torch.bfloat16))
    layer_w = make(32, width, "f32", 6, scale=width ** -0.5)
    layer = rmr.Linear(layer_w, format="mx8")
    y, bound = ref.linear(ref.held(x), ref.held(layer_w), None, "none", None, torch.float32)
    ref.check(layer.kept(cache, s, out_dtype=torch.float32), y, bound)
    cache.close()


def test_read_leaves_what_is_between_rows(rmr):
    cache = rmr.FeatureCache(10, 37)
    x = make(10, 37, "f16", 7)
    s = torch.arange(10).cuda()
    cache.write(x, s)
    for kind in KINDS.values():
        room = torch.full((10, 50), 5.0, dtype=kind, device="cuda")
        cache.read(s, out=room[:, 3:40])
        assert torch.equal(room[:, 3:40].cpu(), ref.held(x).to(kind))
        assert (room[:, :3] == 5).all() and (room[:, 40:] == 5).all()


# --------------------------------------------------------------------------------------------------------------- linear

SHAPES = [(1, 1, 1), (1, 64, 64), (1, 577, 130), (2, 27, 65), (5, 128, 16), (15, 1001, 77), (16, 256, 192), (17, 320, 64), (33, 72, 257),
          (31, 300, 90), (32, 700, 4200), (33, 64, 64), (64, 512, 512), (65, 136, 129), (100, 640, 1000), (129, 264, 320), (200, 96, 33), (257, 1160, 260), (300, 65, 1100), (513, 200, 600),
          (1500, 384, 1030), (2100, 1000, 250), (3001, 2200, 2900),
          (100, 2100, 200), (40, 4300, 70), (64, 8200, 130)]


@pytest.mark.parametrize("fmt", ["f16", "bf16", "mx8"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_exact_on_integers(rmr, fmt, m, k, n):
    """Small whole numbers: every product and sum is exact, so every value must be equal, whatever the order of the sums.
    mx8 holds whole numbers up to 15 exactly beside a largest value of 15."""
    g = torch.Generator().manual_seed(m * 7 + k * 3 + n)
    x = torch.randint(-3, 4, (m, k), generator=g).float()
    w = torch.randint(-2, 3, (n, k), generator=g).float()
    b = torch.randint(-9, 10, (n,), generator=g).float()
    r = torch.randint(-50, 51, (m, n), generator=g).float()
    kind = KINDS["bf16" if fmt == "bf16" else "f16"]
    layer = rmr.Linear(w.cuda(), b.cuda(), format=fmt)
    got = layer(x.to(kind).cuda(), residual=r.cuda(), out_dtype=torch.float32)
    want = x.double() @ w.double().t() + b.double() + r.double()
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("m,k", [(8193, 1001), (8300, 1001), (40001, 193), (8191, 1003), (300, 4101), (20000, 4101)])
def test_linear_many_rows_of_odd_length(rmr, m, k):
    """Rows that do not start at multiples of 16 bytes, few and many: whole numbers, exact."""
    g = torch.Generator().manual_seed(m + k)
    x = torch.randint(-3, 4, (m, k), generator=g).float().cuda()
    w = torch.randint(-2, 3, (40, k), generator=g).float().cuda()
    got = rmr.Linear(w, format="bf16")(x.bfloat16(), out_dtype=torch.float32)
    assert torch.equal(got, x @ w.t())


@pytest.mark.parametrize("m,k,n", [(20, 5000, 4500), (500, 4200, 200), (700, 1000, 900), (3001, 2200, 2900)])
def test_linear_exact_on_integers_with_16_bit_results(rmr, m, k, n):
    """The block-scaled instructions: products of small whole numbers are not cut, so only the one rounding at the end is left."""
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-3, 4, (m, k), generator=g).float()
    w = torch.randint(-2, 3, (n, k), generator=g).float()
    want = (x.double() @ w.double().t()).to(torch.bfloat16)
    layer = rmr.Linear(w.cuda(), format="mx8")
    assert torch.equal(layer(x.bfloat16().cuda()).cpu(), want)
    cache = rmr.FeatureCache(m, k)
    s = torch.randperm(m, generator=g).cuda()
    cache.write(x.cuda(), s)
    assert torch.equal(layer.kept(cache, s, out_dtype=torch.bfloat16).cpu(), want)


@pytest.mark.parametrize("fmt,out", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("mx8", "bf16"), ("mx8", "f32"), ("mx8", "f16")])
@pytest.mark.parametrize("act,with_r,with_b", [("none", False, True), ("relu", True, True), ("silu", True, False), ("gelu", False, True), ("sigmoid", True, True)])
@pytest.mark.parametrize("m,k,n,pad,offset", [(1, 577, 200, 0, 0), (7, 128, 100, 8, 0), (16, 1000, 96, 0, 8), (50, 333, 65, 3, 1), (300, 576, 300, 0, 0), (1030, 193, 520, 1, 0)])
def test_linear_against_64_bits(rmr, fmt, out, act, with_r, with_b, m, k, n, pad, offset):
    src = {"f16": "f16", "bf16": "bf16", "mx8": out}[fmt]
    x = make(m, k, src, 11, pad, offset)
    w = make(n, k, {"mx8": "f32"}.get(fmt, fmt), 12, scale=k ** -0.5)
    b = torch.randn(n, generator=torch.Generator().manual_seed(13)) if with_b else None
    r = make(m, n, out, 14, pad, offset) if with_r else None
    layer = rmr.Linear(w, b.cuda() if with_b else None, activation=act, format=fmt)
    room = torch.full((m, n + 5), 7.0, dtype=KINDS[out], device="cuda")
    got = layer(x, residual=r, out=room[:, 2:n + 2])
    assert (room[:, :2] == 7).all() and (room[:, n + 2:] == 7).all()
    xd, wd = (ref.held(x), ref.held(w)) if fmt == "mx8" else (x.cpu().double(), w.cpu().double())
    y, bound = ref.linear(xd, wd, b.double() if with_b else None, act, r.cpu().double() if with_r else None, KINDS[out], fmt == "mx8")
    ref.check(got, y, bound)
    aligned = layer(x.contiguous(), residual=r.contiguous() if with_r else None, out_dtype=KINDS[out])
    ref.check(aligned, y, bound)


@pytest.mark.parametrize("m,k,n", [(1, 64, 32), (20, 576, 256), (130, 1001, 70), (700, 200, 515)])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_kept_rows(rmr, m, k, n, out):
    cap = 333
    cache = rmr.FeatureCache(cap, k)
    x = make(cap, k, "bf16", 21)
    cache.write(x, torch.arange(cap).cuda())
    g = torch.Generator().manual_seed(22)
    slots = torch.randint(-2, cap + 2, (m,), generator=g)   # some twice, some that do not exist
    w = make(n, k, "f32", 23, scale=k ** -0.5)
    b = torch.randn(n, generator=g)
    layer = rmr.Linear(w, b, activation="silu", format="mx8")
    r = make(m, n, out, 24)
    got = layer.kept(cache, slots.cuda(), residual=r, out_dtype=KINDS[out])
    y, bound = ref.linear(ref.pick(ref.held(x), slots, cap), ref.held(w), b.double(), "silu", r.cpu().double(), KINDS[out], True)
    ref.check(got, y, bound)


@pytest.mark.parametrize("fmt", ["f16", "mx8"])
@pytest.mark.parametrize("m", [3, 70, 600])
def test_linear_non_finite_values_stay_in_their_row(rmr, fmt, m):
    k, n = 200, 90
    x = make(m, k, "f16", 31)
    x[1, 7], x[m - 1, k - 1] = float("inf"), float("nan")
    w = make(n, k, "f16", 32, scale=k ** -0.5)
    layer = rmr.Linear(w, format=fmt)
    got = layer(x, out_dtype=torch.float32).cpu()
    clean = [i for i in range(m) if i not in (1, m - 1)]
    assert torch.isfinite(got[clean]).all() and not torch.isfinite(got[1]).any() and torch.isnan(got[m - 1]).all()


def test_linear_in_place_residual_and_broadcast_rows(rmr):
    for fmt in ("f16", "mx8"):
        layer = rmr.Linear(make(100, 128, "f16", 41, scale=0.1), format=fmt, activation="gelu")
        one = make(1, 128, "f16", 42)
        x = one.expand(300, 128)                     # one row, 300 times: row pitch 0
        y = make(300, 100, "f16", 43)
        want = layer(x.contiguous(), residual=y.clone())
        got = layer(x, residual=y, out=y)
        assert got is y and torch.equal(y, want)
        assert torch.equal(layer(x.view(3, 100, 128), residual=None)[1], layer(one)[0].expand(100, 100))


def test_linear_zero_rows(rmr):
    layer = rmr.Linear(make(10, 12, "f16", 51), format="f16")
    assert layer(torch.empty(0, 12, dtype=torch.float16, device="cuda")).shape == (0, 10)
    layer8 = rmr.Linear(make(10, 12, "f16", 51), format="mx8")
    cache = rmr.FeatureCache(4, 12)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    cache.write(torch.empty(0, 12, dtype=torch.float16, device="cuda"), none)
    assert layer8.kept(cache, none).shape == (0, 10) and cache.read(none).shape == (0, 12)


def test_weights_from_host_and_device_are_the_same(rmr):
    w = make(130, 200, "f32", 61)
    b = torch.randn(130, generator=torch.Generator().manual_seed(62))
    for fmt, kind in (("f16", torch.float16), ("bf16", torch.bfloat16), ("mx8", torch.float16)):
        x = make(40, 200, "f32", 63).to(kind)
        a = rmr.Linear(w, b.cuda(), format=fmt)(x)
        assert torch.equal(a, rmr.Linear(w.cpu().numpy(), b.numpy(), format=fmt)(x))
        assert torch.equal(a, rmr.Linear(w.t().contiguous().t(), b, format=fmt)(x))


def test_captured_and_replayed(rmr):
    """Write, kept layer, second layer and read in one graph, replayed on new inputs with eager work in between."""
    cap, k, n = 500, 200, 96
    cache = rmr.FeatureCache(cap, k)
    up = rmr.Linear(make(n, k, "f32", 71, scale=k ** -0.5), activation="silu", format="mx8")
    down = rmr.Linear(make(k, n, "f32", 72, scale=n ** -0.5), activation="none", format="mx8")
    x = torch.empty(6000, k, dtype=torch.float16, device="cuda")[:, :k]
    slots = torch.empty(6000, dtype=torch.int64, device="cuda")
    pick = torch.empty(70, dtype=torch.int64, device="cuda")

    def step():
        cache.write(x, slots)
        h = up.kept(cache, pick, out_dtype=torch.float16)
        y = down(h, residual=cache.read(pick))
        return h, y

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(6000, k, generator=g).half())
        slots.copy_(torch.randint(-1, cap, (6000,), generator=g))
        pick.copy_(torch.randint(0, cap, (70,), generator=g))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(1, 5):
        fill(seed)
        graph.replay()
        mine = [t.clone() for t in got]
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(mine, want):
            assert torch.equal(a, b)


def test_on_another_stream(rmr):
    layer = rmr.Linear(make(300, 512, "f16", 81, scale=0.05), format="f16", activation="relu")
    x = make(2000, 512, "f16", 82)
    want = layer(x)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (s1, s2, s1, s2):
        with torch.cuda.stream(s):
            outs.append(layer(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_threads_on_one_layer(rmr):
    """A layer is read-only: calls of different sizes from two threads on two streams do not disturb each other."""
    import threading
    layer = rmr.Linear(make(200, 1500, "f32", 85, scale=0.05), format="mx8", activation="silu")
    xs = [make(m, 1500, "bf16", 86 + m) for m in (50, 400, 3000)]
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for i in order:
                    y = layer(xs[i])
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, want[i]):
                        bad.append(i)

    threads = [threading.Thread(target=work, args=(o,)) for o in ((0, 1, 2), (2, 0, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_results_do_not_depend_on_the_run(rmr):
    """No atomics in the sums: the same call gives the same bits, split over workgroups or not."""
    for m, k, n in ((5, 4096, 4096), (64, 8192, 300), (300, 1000, 700)):
        for fmt in ("bf16", "mx8"):
            layer = rmr.Linear(make(n, k, "bf16", 87, scale=k ** -0.5), format=fmt)
            x = make(m, k, "bf16", 88)
            first = layer(x, out_dtype=torch.float32)
            assert all(torch.equal(layer(x, out_dtype=torch.float32), first) for _ in range(5))


def test_a_cache_that_does_not_fit_leaves_no_error_behind(rmr):
    with pytest.raises(rmr.DeviceError):
        rmr.FeatureCache(2 ** 39, 65536)
    cache = rmr.FeatureCache(4, 40)
    x = make(4, 40, "f16", 89)
    s = torch.arange(4).cuda()
    cache.write(x, s)
    assert torch.equal(cache.read(s).cpu(), ref.held(x).half())


def test_refusals(rmr):
    cache = rmr.FeatureCache(8, 64)
    f16 = rmr.Linear(make(32, 64, "f16", 91), format="f16")
    mx8 = rmr.Linear(make(32, 64, "f16", 91), format="mx8")
    x = make(4, 64, "f16", 92)
    s = torch.arange(4).cuda()
    wide = torch.zeros(200, dtype=torch.int64, device="cuda")
    bad = rmr.InvalidArgument
    for call in (lambda: f16(x.bfloat16()), lambda: f16(x.float()), lambda: f16(x[:, :63]), lambda: f16(x.t()), lambda: f16(x.cpu()),
                 lambda: f16(x.double()), lambda: f16(x, residual=make(4, 32, "f32", 1)), lambda: f16(x, residual=make(3, 32, "f16", 1)),
                 lambda: f16(x, out=torch.empty(5, 32, dtype=torch.float16, device="cuda")), lambda: f16(x, out=torch.empty(4, 32, dtype=torch.float16)),
                 lambda: f16(x, out=x[:, :32]), lambda: f16(x, out=torch.empty(4, 32, dtype=torch.float16, device="cuda"), out_dtype=torch.float32),
                 lambda: f16(x, out=torch.empty(1, 32, dtype=torch.float16, device="cuda").expand(4, 32)),
                 lambda: f16.kept(cache, s), lambda: mx8.kept(rmr.FeatureCache(8, 65), s), lambda: mx8.kept(cache, s.int()), lambda: mx8.kept(cache, s.cpu()),
                 lambda: mx8.kept(cache, s[::2]), lambda: cache.write(x, s[:3]), lambda: cache.write(x[:, :32], s), lambda: cache.write(x.cpu(), s),
                 lambda: cache.write(x.long(), s), lambda: cache.read(s, out=torch.empty(3, 64, device="cuda")), lambda: cache.read(s.view(2, 2)),
                 lambda: cache.read(s, out=torch.empty(1, 64, device="cuda").expand(4, 64)), lambda: cache.read(wide[:4], out=wide.view(torch.float32)[:256].view(4, 64)),
                 lambda: mx8.kept(cache, wide[:4], out=wide.view(torch.float16)[:128].view(4, 32)), lambda: cache.read(s, dtype=torch.int32)):
        with pytest.raises(bad):
            call()
    y = torch.empty(5, 32, dtype=torch.float16, device="cuda")
    with pytest.raises(bad):
        f16(x, residual=y[:4], out=y[1:])
    # the C entry itself: no workspace where one is needed
    from rm_radar_amd import _lib
    import ctypes as C
    x, out = make(400, 64, "f16", 93), torch.empty(400, 32, dtype=torch.float16, device="cuda")
    c = _lib.LinearCall(x.data_ptr(), 0, 64, 400, None, 0, out.data_ptr(), 0, 32, None, 0)
    with pytest.raises(rmr.CapacityError):
        _lib.check(_lib.lib().rmr_linear_run(mx8._h, C.byref(c), None))


# ------------------------------------------------------------------------------------------------------------- together

def test_detector_features_through_cache_and_layers(rmr, tmp_path, monkeypatch):
    """A detector's stage output kept over two frames, embedded in place and projected: as a second head would run."""
    from rm_radar_amd import weights as W
    import netutil
    monkeypatch.setenv("RMR_ARENA_REUSE", "0")
    pack = W.make_synthetic_pack(str(tmp_path / "car.rmrw"), "m", 1, seed=3, cls_bias=-3.0)
    det = rmr.Detector(pack, 1, (1280, 720), 2)
    imgs = [netutil.test_image(i, 720, 1280) for i in range(2)]
    det.infer(imgs)
    feats = [det.read_feature("model.21", i) for i in range(2)]
    h, w, c = feats[0].shape
    cache = rmr.FeatureCache(2 * h * w + 5, c)
    for i in range(2):
        det.keep_feature("model.21", cache, 3 + i * h * w, img=i)
    flat = torch.from_numpy(np.concatenate([f.reshape(h * w, c) for f in feats]))
    held = ref.held(flat)
    got = cache.read(torch.arange(3, 3 + 2 * h * w).cuda(), dtype=torch.float32)
    assert torch.equal(got.cpu().double(), held)
    embed_w, out_w = make(128, c, "f32", 101, scale=c ** -0.5), make(24, 128, "f16", 102, scale=0.1)
    embed = rmr.Linear(embed_w, torch.zeros(128), activation="silu", format="mx8")
    head = rmr.Linear(out_w, activation="sigmoid", format="f16")
    pixels = torch.tensor([3, 3 + h * w - 1, 3 + h * w, 3 + 2 * h * w - 1, 100, 100]).cuda()
    e = embed.kept(cache, pixels)
    y, bound = ref.linear(held[pixels.cpu() - 3], ref.held(embed_w), None, "silu", None, torch.float16, True)
    ref.check(e, y, bound)
    y, bound = ref.linear(e.cpu().double(), out_w.cpu().double(), None, "sigmoid", None, torch.float16)
    ref.check(head(e), y, bound)
    for bad in (lambda: det.keep_feature("model.21", cache, 6 + h * w, img=1), lambda: det.keep_feature("model.21", cache, -1),
                lambda: det.keep_feature("nothing", cache, 0), lambda: det.keep_feature("model.21", cache, 0, img=2),
                lambda: det.keep_feature("model.21", rmr.FeatureCache(2000, c + 1), 0)):
        with pytest.raises(rmr.InvalidArgument):
            bad()
    det.close()
