"""The scale of a 4-bit group: the range times fp32's 1 / 15, rounded to the cache's type,
wherever rows are rounded.  Quotient and product differ by a unit of fp32 for about half of all
ranges, which decides groups whose fifteenth lies between two numbers of the cache's type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from oracle import paged_int4 as o4

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def border_rows(dtype: str, dim: int, group: int) -> torch.Tensor:
    """Rows whose groups' ranges round to other scales when they are divided by 15."""
    g = torch.Generator().manual_seed(group)
    ends = torch.randn(400000, 2, generator=g).to(DT[dtype])
    hi, lo = ends.amax(1).float(), ends.amin(1).float()
    product = ((hi - lo) * torch.tensor(1 / 15)).to(DT[dtype])
    ends = torch.stack([hi, lo], 1)[((hi - lo).double() / 15).float().to(DT[dtype]) != product]
    assert len(ends) > 100
    if dtype == "bf16":
        ends[:2] = torch.tensor([[6.1875, -0.0966796875], [22.5, -15 / 256]])
    n = len(ends) // (dim // group) * (dim // group)
    ends = ends[:n].view(-1, dim // group, 2)
    rows = torch.rand(*ends.shape[:2], group, generator=g) * (ends[..., :1] - ends[..., 1:]) + ends[..., 1:]
    rows = rows.to(DT[dtype]).float().clamp(min=ends[..., 1:], max=ends[..., :1])
    rows[..., 5], rows[..., group - 3] = ends[..., 0], ends[..., 1]
    return rows.flatten(1).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
def test_scales_at_the_border(dtype, dim, group):
    rows = border_rows(dtype, dim, group)
    codes, scales = ab.quantize_kv_int4(rows, group)
    x = rows.float().unflatten(-1, (-1, group))
    want = ((x.amax(-1) - x.amin(-1)) * torch.tensor(1 / 15)).to(DT[dtype])
    assert torch.equal(scales[..., 0], want)
    scale, least, code = o4.levels(rows.float().numpy(), group, dtype)
    np.testing.assert_array_equal(scales[..., 0].float().numpy(), scale)
    np.testing.assert_array_equal(scales[..., 1].float().numpy(), least)
    assert (np.abs(o4.unpack(codes.numpy()) - code) <= 0.5 + 2.0 ** -15).all()
