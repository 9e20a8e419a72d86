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
