"""Timing cases of the dense operators that work on a detector's kept features.

Four operators are listed: a linear layer (matrix product with bias, activation and residual in its epilogue) on 16-bit
rows, the same layer on block-scaled 8-bit rows, the layer on rows that a feature cache holds, and the cache itself
(rows quantised as they are written, and read back).

A block-scaled ("mx8") row holds its values in blocks of 32: one power of two 2^e per block and 32 OCP e4m3 values.  e is the
smallest exponent in [-127, 127] with max|v| <= 448 * 2^e over the block's finite values (-127 for a block of zeros), every value
is v / 2^e rounded to nearest even, and a value that is not finite is held as NaN.

``own`` says which side ``prepare`` and ``run`` take: the plain form in elementary torch operations, or this package's
operators.  ``exact`` computes the same from the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_ACTS = ("none", "relu", "silu", "gelu", "sigmoid")


def listed():
    return [
        # one new row through a wide layer: every weight is read for one row, latency and bandwidth count
        dict(name="linear_one_row", op="linear", format="bf16", rows=1, inner=4096, outer=4096, act="silu", residual=True, out="bf16", pad=0),
        # a pointwise layer of the detector's 40 x 40 maps over a batch of 64 images
        dict(name="linear_maps", op="linear", format="f16", rows=102400, inner=384, outer=384, act="silu", residual=True, out="f16", pad=0),
        # sizes that fit no tile, rows that start at odd addresses
        dict(name="linear_ragged", op="linear", format="f16", rows=1777, inner=1001, outer=1237, act="gelu", residual=True, out="f32", pad=3),
        # the largest product: a full batch of rows through a square layer
        dict(name="linear_large", op="linear", format="bf16", rows=8192, inner=8192, outer=8192, act="gelu", residual=False, out="bf16", pad=0),
        # a handful of rows through 8-bit weights, as one row per robot of a frame
        dict(name="linear8_few", op="linear", format="mx8", rows=16, inner=4096, outer=8192, act="none", residual=False, out="bf16", pad=0, source="bf16"),
        # the largest product on 8-bit rows, quantised within the call
        dict(name="linear8_large", op="linear", format="mx8", rows=8192, inner=8192, outer=8192, act="silu", residual=True, out="bf16", pad=0, source="bf16"),
        # the robots of a frame: 20 rows out of the kept features of 64 images' 20 x 20 maps, embedded by a small layer
        dict(name="kept_robots", op="kept", rows=20, inner=576, outer=256, act="silu", residual=False, out="f32", slots=25600),
        # a whole bank of kept rows through a wide layer
        dict(name="kept_bank", op="kept", rows=16384, inner=4096, outer=4096, act="none", residual=False, out="bf16", slots=32768),
        # the deepest 20 x 20 map of one image enters the cache and is read back: latency
        dict(name="cache_frame", op="cache", rows=400, inner=576, source="f16", out="f16", slots=25600, order="run", pad=0),
        # many streams' rows at scattered slots, some of them left out: bandwidth
        dict(name="cache_bank", op="cache", rows=262144, inner=1024, source="bf16", out="bf16", slots=524288, order="shuffled", pad=0),
        # one robot's history of 100 rows
        dict(name="read_track", op="read", rows=100, inner=576, out="f16", slots=25600),
        # scattered rows of an odd width for a long list of slots
        dict(name="read_bank", op="read", rows=200000, inner=1001, out="f32", slots=400000),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread over the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _size(rng, low, high):
    v = _spread(rng, low, high)
    kind = rng.random()
    if kind < 0.4 and v >= 64:
        v = v // 32 * 32
    elif kind < 0.7:
        v |= 1
    return min(high, max(low, v))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear8", "kept", "cache", "read"))
    out = rng.choice(("f16", "bf16", "f32"))
    if op in ("cache", "read"):
        inner = _size(rng, 32, 2048)
        rows = _size(rng, 1, min(262144, 262144 * 1001 // inner))
        case = dict(op=op, rows=rows, inner=inner, out=out, slots=rows + _spread(rng, 1, 262144))
        if op == "cache":
            case.update(source=rng.choice(("f16", "bf16", "f32")), order=rng.choice(("run", "shuffled", "repeated")), pad=rng.choice((0, 0, 8, 3)))
        return case
    rows, inner, outer = _size(rng, 1, 32768), _size(rng, 32, 8192), _size(rng, 32, 8192)
    while rows * inner * outer > 8192 ** 3 // 4:
        rows = max(1, rows // 2)
    case = dict(op=op, rows=rows, inner=inner, outer=outer, act=rng.choice(_ACTS), residual=rng.random() < 0.5, out=out)
    if op == "kept":
        case.update(slots=rows + _spread(rng, 1, 32768))
    elif op == "linear8":
        case.update(op="linear", format="mx8", source=rng.choice(("f16", "bf16", "f32")), pad=rng.choice((0, 0, 8, 3)))
    else:
        case.update(format=rng.choice(("f16", "bf16")), pad=rng.choice((0, 0, 8, 3)))
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs

def _generator(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _features(g, rows, width, dtype, pad=0):
    """Rows as a SiLU layer leaves them, a few channels an order of magnitude larger than the others."""
    x = torch.randn(rows, width + pad, generator=g, device="cuda", dtype=torch.float32)
    x = x * torch.sigmoid(1.702 * x)
    loud = torch.rand(width + pad, generator=g, device="cuda") < 0.02
    x = torch.where(loud, x * 12.0, x).to(dtype)
    return x[:, :width]


def _weights(g, outer, inner):
    w = torch.randn(outer, inner, generator=g, device="cuda", dtype=torch.float32) / math.sqrt(inner)
    bias = torch.randn(outer, generator=g, device="cuda", dtype=torch.float32) * 0.5
    return w, bias


def _slots(g, case):
    n, cap = case["rows"], case["slots"]
    order = case.get("order", "shuffled")
    if order == "run":
        first = int(torch.randint(0, cap - n + 1, (1,), generator=g, device="cuda"))
        return torch.arange(first, first + n, device="cuda", dtype=torch.int64)
    s = torch.randperm(cap, generator=g, device="cuda")[:n]
    if case["op"] == "cache":  # rows that are left out carry no slot
        s = torch.where(torch.rand(n, generator=g, device="cuda") < 0.02, torch.full_like(s, -1), s)
    if order == "repeated" and n > 1:  # a slot that is named twice keeps its last row
        again = torch.rand(n, generator=g, device="cuda") < 0.1
        s = torch.where(again, s.roll(n // 2), s)
    return s.contiguous()


def _inputs(case, seed):
    """Everything a case is made of, the same for every form of it."""
    g = _generator(seed)
    d = dict(case=case)
    if case["op"] in ("linear", "kept"):
        w, d["bias"] = _weights(g, case["outer"], case["inner"])
        d["weight"] = w if case.get("format", "mx8") == "mx8" else w.to(_TYPES[case["format"]])
        if case["residual"]:
            d["residual"] = torch.randn(case["rows"], case["outer"], generator=g, device="cuda", dtype=torch.float32).to(_TYPES[case["out"]])
    if case["op"] == "linear":
        kind = case["source"] if case["format"] == "mx8" else case["format"]
        d["x"] = _features(g, case["rows"], case["inner"], _TYPES[kind], case["pad"])
    elif case["op"] == "cache":
        d["x"] = _features(g, case["rows"], case["inner"], _TYPES[case["source"]], case["pad"])
        d["slots"] = _slots(g, case)
    else:
        d["kept"] = _features(g, case["slots"], case["inner"], torch.bfloat16)
        d["slots"] = _slots(g, case)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    s = dict(case=case)
    for k in ("x", "residual", "slots"):
        if k in d:
            s[k] = d[k]
    if own:
        import rm_radar_amd as rmr
        if "weight" in d:
            s["layer"] = rmr.Linear(d["weight"], d["bias"], activation=case["act"], format=case.get("format", "mx8"))
        if "slots" in d:
            s["cache"] = rmr.FeatureCache(case["slots"], case["inner"])
            if "kept" in d:
                s["cache"].write(d["kept"], torch.arange(case["slots"], device="cuda"))
        return s
    if "weight" in d:
        s["bias"] = d["bias"]
        s["weight"] = d["weight"] if case.get("format", "mx8") != "mx8" else _quantise(d["weight"])
    if "kept" in d:
        s["cache"] = _quantise(d["kept"])
    elif "slots" in d:
        blocks = -(-case["inner"] // 32)
        s["cache"] = (torch.zeros(case["slots"], blocks, 32, device="cuda", dtype=torch.float8_e4m3fn),
                      torch.full((case["slots"], blocks), -127, device="cuda", dtype=torch.int32))
    return s


# ------------------------------------------------------------------------------------------------------------ plain form

def _quantise(x):
    """Rows to blocks of 32: e4m3 values [rows, blocks, 32] and exponents [rows, blocks]."""
    rows, width = x.shape
    blocks = -(-width // 32)
    v = torch.zeros(rows, blocks * 32, device=x.device, dtype=torch.float32)
    v[:, :width] = x.float()
    v = v.view(rows, blocks, 32)
    top = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(2)
    m, e = torch.frexp(top)                      # top = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(top == 0, torch.full_like(e, -127), e.clamp(-127, 127))
    v = torch.where(torch.isfinite(v), torch.ldexp(v.double(), -e[:, :, None]).float(), torch.full_like(v, float("nan")))
    return v.to(torch.float8_e4m3fn), e


def _values(cache, width):
    q, e = cache
    return (q.float() * torch.ldexp(torch.ones((), device=q.device, dtype=torch.float64), e[:, :, None]).float()).flatten(1)[:, :width]


def _activate(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * torch.erfc(v * -math.sqrt(0.5))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    return v


def _linear(x, s):
    case = s["case"]
    w = _values(s["weight"], case["inner"]) if isinstance(s["weight"], tuple) else s["weight"].float()
    y = _activate(x @ w.t() + s["bias"], case["act"])
    if "residual" in s:
        y = y + s["residual"].float()
    return y.to(_TYPES[case["out"]])


def _rows(cache, slots):
    """The rows at `slots`; zeros where there is no such slot."""
    q, e = cache
    good = (slots >= 0) & (slots < q.shape[0])
    at = torch.where(good, slots, torch.zeros_like(slots))
    q8 = torch.where(good[:, None, None], q.view(torch.uint8)[at], torch.zeros((), device=q.device, dtype=torch.uint8))
    return q8.view(torch.float8_e4m3fn), e[at]


def _write(cache, x, slots):
    q, e = _quantise(x)
    good = (slots >= 0) & (slots < cache[0].shape[0])
    last = torch.full((cache[0].shape[0] + 1,), -1, device=x.device, dtype=torch.int64)   # the last row that names each slot
    at = torch.where(good, slots, torch.full_like(slots, cache[0].shape[0]))
    row = torch.arange(slots.numel(), device=x.device)
    last.scatter_reduce_(0, at, row, "amax")
    win = good & (last[at] == row)
    cache[0].view(torch.uint8)[slots[win]] = q.view(torch.uint8)[win]
    cache[1][slots[win]] = e[win]


def run(state):
    case = state["case"]
    op, kind = case["op"], _TYPES[case["out"]]
    if own:
        if op == "linear":
            return state["layer"](state["x"], residual=state.get("residual"), out_dtype=kind)
        if op == "kept":
            return state["layer"].kept(state["cache"], state["slots"], residual=state.get("residual"), out_dtype=kind)
        if op == "cache":
            state["cache"].write(state["x"], state["slots"])
        return state["cache"].read(state["slots"], dtype=kind)
    width = case["inner"]
    if op == "linear":
        x = state["x"]
        return _linear(_values(_quantise(x), width) if case["format"] == "mx8" else x.float(), state)
    if op == "kept":
        return _linear(_values(_rows(state["cache"], state["slots"]), width), state)
    if op == "cache":
        _write(state["cache"], state["x"], state["slots"])
    return _values(_rows(state["cache"], state["slots"]), width).to(kind)


# ----------------------------------------------------------------------------------------------------------------- sizes

def work(case):
    n, k = case["rows"], case["inner"]
    row8 = k + -(-k // 32)                                  # one held row: its values and its exponents
    if case["op"] == "cache":
        return {"bytes": n * (k * _BYTES[case["source"]] + 8 + row8) + n * (8 + row8 + k * _BYTES[case["out"]]), "flops": 0}
    if case["op"] == "read":
        return {"bytes": n * (8 + row8 + k * _BYTES[case["out"]]), "flops": 0}
    m = case["outer"]
    eight = case.get("format", "mx8") == "mx8"
    x = n * (8 + row8) if case["op"] == "kept" else n * k * _BYTES[case["source"] if eight else case["format"]]
    w = m * row8 if eight else m * k * 2
    y = n * m * _BYTES[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": x + w + 4 * m + y, "flops": 2.0 * n * m * k}


# ----------------------------------------------------------------------------------------------------------------- exact

def _held(x):
    """The values a held row stands for, in 64 bits."""
    rows, width = x.shape
    full = width + (-width) % 32
    v = torch.zeros(rows, full, dtype=torch.float64, device=x.device)
    v[:, :width] = x.double()
    step = torch.empty_like(v)
    for first in range(0, full, 32):                        # a block at a time: its power of two
        part = v[:, first:first + 32]
        top = part.abs().nan_to_num(nan=0.0, posinf=0.0, neginf=0.0).amax(1, keepdim=True)
        e = torch.ceil(torch.log2(top / 448.0)).clamp(-127, 127)
        e = e + (torch.exp2(e) * 448.0 < top)               # the logarithm may be off by one next to a border
        lower = torch.exp2(e - 1) * 448.0 >= top
        e = torch.where(lower & (e > -127), e - 1, e)
        e = torch.where(top == 0, torch.full_like(e, -127.0), e)
        step[:, first:first + 32] = torch.exp2(e)
    u = v / step
    grid = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)   # distance of neighbouring e4m3 values
    u = torch.round(u / grid) * grid                        # to nearest, ties to even
    return torch.where(torch.isfinite(v), u * step, torch.full_like(v, float("nan")))[:, :width]


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "cache":
        slots = d["slots"].tolist()
        held = _held(d["x"])
        last = {s: i for i, s in enumerate(slots) if 0 <= s < case["slots"]}
        pick = torch.tensor([last.get(s, -1) for s in slots], device="cuda")
        return torch.where((pick >= 0)[:, None], held[pick.clamp_min(0)], torch.zeros((), dtype=torch.float64, device="cuda"))
    if case["op"] == "read":
        return _held(d["kept"][d["slots"]])
    eight = case.get("format", "mx8") == "mx8"
    x = d["kept"][d["slots"]] if case["op"] == "kept" else d["x"]
    x = _held(x) if eight else x.double()
    w = _held(d["weight"]) if eight else d["weight"].double()
    y = torch.mm(x, w.t().contiguous()) + d["bias"].double()
    act = case["act"]
    if act == "relu":
        y = y.clamp_min(0.0)
    elif act == "silu":
        y = y * torch.special.expit(y)
    elif act == "gelu":
        y = y * torch.special.ndtr(y)
    elif act == "sigmoid":
        y = torch.special.expit(y)
    return y + d["residual"].double() if "residual" in d else y
