"""Clamped gates of what is no number: a NaN behind a clamp is still one."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from liyab_amd.kernels import ops as module

    return module


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_alone(ops, dtype):
    n, ff = 5, 70
    gu = torch.randn(n, 2 * ff, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.empty(n, ff, dtype=dtype, device=DEV)
    ops.glu_clamped(want, gu, 1.5, 1.7, 1.0)
    gu[1, 3] = gu[2, ff + 69] = float("nan")
    gu[3, 5], gu[4, ff + 6] = float("inf"), float("-inf")
    out = torch.empty_like(want)
    ops.glu_clamped(out, gu, 1.5, 1.7, 1.0)
    nan = torch.zeros(n, ff, dtype=torch.bool, device=DEV)
    nan[1, 3] = nan[2, 69] = True
    assert torch.equal(torch.isnan(out), nan)
    changed = nan.clone()
    changed[3, 5] = changed[4, 6] = True
    assert torch.equal(out[~changed], want[~changed])
    gu[3, 5], gu[4, ff + 6] = 1.5, -1.5  # what lies beyond the limits is the limit
    ops.glu_clamped(want, gu, 1.5, 1.7, 1.0)
    assert torch.equal(out[3:], want[3:])


@pytest.mark.parametrize("block,dtype", [(16, torch.bfloat16), (64, torch.float32), (64, torch.bfloat16)])
def test_gates_in_the_experts_product(ops, block, dtype):
    n, E, N, K = 40, 2, 72, 64
    g = torch.Generator().manual_seed(2)
    a = torch.randn(n, K, generator=g).to(dtype).to(DEV)
    w0, w1 = ((0.2 * torch.randn(E, N, K, generator=g)).to(dtype).to(DEV) for _ in range(2))
    tiles = ops.moe_tiles(n, E, block)
    rows, group, at = torch.full((tiles, block), -1, dtype=torch.int32), torch.full((tiles,), -1, dtype=torch.int32), 0
    for e in range(E):
        for c in torch.arange(e, n, E, dtype=torch.int32).split(block):
            rows[at, :len(c)], group[at], at = c, e, at + 1
    outs = []
    for bad in (False, True):
        if bad:
            a[7, 11] = float("nan")
        out = torch.zeros(n, N, dtype=dtype, device=DEV)
        ops.moe_product(out, a, w0, w1, rows.to(DEV).flatten(), group.to(DEV), block=block, clamp=(0.7, 1.702, 1.0))
        outs.append(out)
    nan = torch.zeros(n, N, dtype=torch.bool, device=DEV)
    nan[7] = True
    assert torch.equal(torch.isnan(outs[1]), nan) and torch.equal(outs[1][~nan], outs[0][~nan])
