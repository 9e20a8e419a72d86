"""Plain 64-bit forms of the feature cache's format and of the linear layer, for the tests."""
import numpy as np
import torch

EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}   # half a subnormal step
# largest slope of each activation
SLOPE = {"none": 1.0, "relu": 1.0, "silu": 1.1, "gelu": 1.13, "sigmoid": 0.25}


def held(x):
    """What a held row stands for: f64 [rows, width] on the CPU."""
    v = x.detach().cpu().double().numpy()
    rows, width = v.shape
    blocks = -(-width // 32)
    p = np.zeros((rows, blocks * 32))
    p[:, :width] = v
    p = p.reshape(rows, blocks, 32)
    fin = np.isfinite(p)
    top = np.where(fin, np.abs(p), 0.0).max(2)
    m, e = np.frexp(top)                         # top = m 2^e, 448 = 0.875 * 2^9
    e = np.where(m > 0.875, e - 8, e - 9)
    e = np.where(top == 0, -127, np.clip(e, -127, 127)).astype(np.int64)
    u = np.where(fin, p, 0.0) / np.exp2(e.astype(np.float64))[:, :, None]
    grid = np.exp2(np.floor(np.log2(np.maximum(np.abs(u), 2.0 ** -6))) - 3)
    u = np.round(u / grid) * grid                # numpy rounds ties to even
    out = np.where(fin, u * np.exp2(e.astype(np.float64))[:, :, None], np.nan)
    return torch.from_numpy(out.reshape(rows, blocks * 32)[:, :width].copy())


def pick(held_rows, slots, cap):
    """Rows by slot, zeros where there is no such slot."""
    s = slots.cpu()
    good = (s >= 0) & (s < cap)
    out = held_rows[torch.where(good, s, torch.zeros_like(s))]
    return torch.where(good[:, None], out, torch.zeros((), dtype=out.dtype))


def activate(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(v * -(0.5 ** 0.5))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    return v


def linear(x, w, bias, act, residual, kind, eight=False):
    """(y, bound) in f64 for f64 operands: the exact layer and how far a right f32 evaluation rounded once to `kind` may be from it.

    A sum of K products in f32, in any order, is off by at most (K + 1) 2^-24 / (1 - ...) of sum |x w|; one more 2^-24 for the bias.  The
    activation passes that on with at most its slope and adds its own evaluation: exp of an argument rounded to 2^-24 |v| 1.5,
    a reciprocal and two products, together under (8 + 2 |v|) 2^-24 of |v| or 1; gelu's erfc is 1.5e-7 off, half of it times |v|.

    eight: the operands are held rows and y has 16 bits.  Then the matrix pipe cuts every product 13 bits below the largest product of
    its group: at most 2^-13 of the largest of all K products each, and that is at most the root of the sum of their squares."""
    u = 2.0 ** -24
    k = x.shape[1]
    s = x @ w.t()
    mass = x.abs() @ w.abs().t()
    if eight and kind != torch.float32:
        cut = k * 2.0 ** -13 * torch.minimum(mass, ((x * x) @ (w * w).t()).sqrt())
    else:
        cut = 0.0
    v = s if bias is None else s + bias
    dv = cut + (k + 2) * 1.01 * u * mass + u * (v.abs() + (0 if bias is None else bias.abs()))
    y = activate(v, act)
    d = SLOPE[act] * dv
    if act in ("silu", "gelu"):
        d = d + (8 + 2 * v.abs().clamp_max(90)) * u * v.abs().clamp_max(1e30) * torch.exp(-v.abs() / 2 * (v < 0)) + (0.8e-7 * v.abs() if act == "gelu" else 0)
    elif act == "sigmoid":
        d = d + (8 + 2 * v.abs().clamp_max(90)) * u * y
    if residual is not None:
        y = y + residual
        d = d + u * y.abs()
    return y, d + (y.abs() + d) * EPS[kind] + TINY[kind]


def check(got, y, bound, what=""):
    g = got.detach().cpu().double()
    nan = torch.isnan(y)
    assert torch.equal(torch.isnan(g), nan), f"{what}: NaN in other places"
    inf = torch.isinf(y)
    # values past the type's range round to infinity
    big = torch.finfo(got.dtype).max
    over = torch.isinf(g) & ~inf
    assert ((y.abs() + bound)[over] >= big).all(), f"{what}: infinite where the value fits"
    assert torch.equal(g[inf], y[inf]), f"{what}: infinities differ"
    ok = ~(nan | inf | over)
    far = ((g - y).abs() - bound)[ok]
    assert far.numel() == 0 or far.max() <= 0, f"{what}: {int((far > 0).sum())} of {far.numel()} values outside their bound, worst by {float(far.max()):.3e}"
