"""Feature cache and linear layer on the GPU: calls and numbers that test_gpu_rows.py leaves open."""
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


@pytest.mark.parametrize("fmt", ["f16", "mx8"])
@pytest.mark.parametrize("m", [1, 20, 70, 700])
@pytest.mark.parametrize("k,n", [(64, 48), (200, 90), (203, 65)])
def test_columns_of_one_buffer(rmr, fmt, m, k, n):
    """x, the residual and y side by side in one wide buffer, as a concatenation holds them."""
    g = torch.Generator().manual_seed(m + k + n)
    wide = torch.randint(-3, 4, (m, k + 2 * n + 9), generator=g).half().cuda()
    w = torch.randint(-2, 3, (n, k), generator=g).float()
    x, r, y = wide[:, 2:k + 2], wide[:, k + 2:k + n + 2], wide[:, k + n + 5:k + 2 * n + 5]
    before = wide.clone()
    want = (x.cpu().double() @ w.double().t() + r.cpu().double()).half()
    assert rmr.Linear(w.cuda(), format=fmt)(x, residual=r, out=y) is y
    assert torch.equal(y.cpu(), want)
    wide[:, k + n + 5:k + 2 * n + 5] = before[:, k + n + 5:k + 2 * n + 5]
    assert torch.equal(wide, before)                      # nothing beside y was written


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(32, 1, 5), (None, 8, 70), (300, 8, 128), (64, 4200, 64)])
def test_gelu_is_right_in_relation_to_its_value(rmr, out, m, k, n):
    """Every f16 value (or m of them) through v / 2 erfc(-v / sqrt 2); the sum is the value itself.  Workgroups of few rows, tiles with
    and without an edge, a K that is split.

    e^(-v v / 2): its argument takes three roundings, 1.5 v v 2^-24 of the result.  Beside that 8 2^-24 for the polynomial in f32 (84 for
    the short one of 16-bit results: 5e-6), 2 each for the reciprocal and the power (one unit in the last place), 4 for the products and
    the difference.  Powers below the smallest
    normal f32 may be taken for zero: they are multiplied by at most |v| / 2."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    every = every[torch.isfinite(every)]
    v = every if m is None else torch.cat([every[every.abs() < 14][::max(1, 45000 // m)][:m - 2], torch.tensor([-4.0, -5.5]).half()])
    x = torch.zeros(len(v), k, dtype=torch.float16)
    x[:, k // 2] = v
    w = torch.zeros(n, k, dtype=torch.float16)
    w[:, k // 2] = 1
    got = rmr.Linear(w, activation="gelu", format="f16")(x.cuda(), out_dtype=KINDS[out]).cpu().double()
    d = v.double()
    y = 0.5 * d * torch.special.erfc(d * -(0.5 ** 0.5))
    u = 2.0 ** -24
    bound = ((16 if out == "f32" else 92) + 1.5 * d.clamp(-40, 0) ** 2) * u * y.abs() + 2.0 ** -127 * d.abs()
    bound = bound + (y.abs() + bound) * ref.EPS[KINDS[out]] + ref.TINY[KINDS[out]]
    far = (got - y[:, None]).abs() - bound[:, None]
    assert far.max() <= 0, f"worst at v = {float(v[far.max(1).values.argmax()])}, by {float(far.max()):.3e}"
