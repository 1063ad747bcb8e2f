"""Edges of the operators of growing sessions, against the same plain
implementations in 64 bits and with the same bounds as test_session_ops_gpu.py:
zero points over the whole byte."""
import pytest

from conftest import cuda_ok, pkg
from test_session_ops_gpu import _check_w4, _w4_case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not cuda_ok():
        pytest.skip("no CUDA device")


# ---------------------------------------------------------------- w4_linear

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,pad", [(1, 0), (13, 0), (5, 1)])
def test_w4_zero_points_are_any_byte(dtype, group, m, pad):
    """A zero point is a byte; codes only reach 15.  Each value meets every code,
    on rows that are read 16 bytes at a time and (pad) on rows that are not.
    A group's f32 sum holds terms of up to 255 |x|, inside the bound's sum."""
    import torch
    n, k = 512, 16 * group
    c = _w4_case(m, n, k, group, dtype, True, False, seed=group + m)
    edge = torch.tensor([0, 15, 16, 63, 64, 65, 127, 128, 129, 191, 192, 240, 241, 254, 255, 8], dtype=torch.uint8)
    c["zeros"][:16] = edge[(torch.arange(16)[:, None] + torch.arange(16)[None]) % 16]
    c["zeros"][16:] = torch.arange((n - 16) * 16).view(-1, 16) % 256
    x = torch.zeros(m, k + pad, dtype=c["x"].dtype, device="cuda")[:, pad:]
    x.copy_(c["x"])
    out = torch.full((m, n), float("nan"), dtype=c["x"].dtype, device="cuda")
    pkg()._lib.w4_linear(x, c["wq"].cuda(), c["scales"].cuda(), out, zeros=c["zeros"].cuda())
    _check_w4(c, out)
