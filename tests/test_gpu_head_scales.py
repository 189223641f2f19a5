"""Quantisation of blocks next to the smallest scale, on the GPU against the nearest values. Marked gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import DEV, ops  # noqa: E402,F401
from test_gpu_head_f8 import SCALES, same  # noqa: E402


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_next_to_the_smallest_scale(ops, block_rows):
    """fp32 blocks whose scale is little above 2^-126, with values beside the middles of two e4m3 numbers: what is
    left of a division there lies below fp32's smallest number."""
    g = torch.Generator().manual_seed(3)
    mid = ((ref.GRID[1:] + ref.GRID[:-1]) / 2)[:126]
    rows = 16 * 128
    scale = torch.ldexp(1 + torch.rand(rows, 1, generator=g, dtype=torch.float64),
                        torch.randint(-126, -110, (rows, 1), generator=g)).float()
    if block_rows == 128:
        scale = scale[::128].repeat_interleave(128, 0)
    x = (mid * scale.double()).float()
    away = torch.randint(-1, 2, x.shape, generator=g)
    x = torch.where(away == 0, x, torch.nextafter(x, torch.where(away > 0, 1.0, -1.0)))
    x = torch.cat([x * torch.where(torch.rand(x.shape, generator=g) < 0.5, 1.0, -1.0), 448 * scale, 0 * scale], 1).to(DEV)
    for name, power in (("f32", False), ("e8m0", True)):
        got = ops.quantize_f8(x, block_rows=block_rows, scale_dtype=SCALES[name])
        values, scales = ref.quantize(x, block_rows, power)
        same(got["scales"], scales)
        same(got["values"], values)
