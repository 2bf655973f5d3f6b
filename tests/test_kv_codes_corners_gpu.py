"""Rotary positions and the quantised cache where results turn on the last bits: factors that 32 bits do not hold."""
import math

import pytest
import torch

from tests.kv_codes_util import code_values
from tests.test_kv_codes_gpu import _freq, _ops
from tests.util import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("factor", [1.2079, 0.1 * math.log(40.0) + 1.0, 0.9, 1.1])
def test_factors_of_64_bits(factor, pairing):
    """A stretched context's factor is taken as it is given: elements whose turned value lies between two codes' middle and what the factor in 32 bits would make of it"""
    from omniserve_amd.backend.lm import code_pools
    rounded = float(torch.tensor(factor, dtype=torch.float32))
    assert rounded != factor
    grid = code_values("cpu")[:127]
    middle = (grid[1:] + grid[:-1]) / 2
    near = (middle / factor).float()
    near = torch.cat([near, *(torch.nextafter(near, torch.full_like(near, s)) for s in (0.0, 1e9))]).double()
    middle = middle.repeat(3)
    x = near[((near * factor - middle) * (near * rounded - middle) < 0)]      # (the two products lie on both sides)
    assert x.numel() >= 10
    x = torch.cat((x, -x))[:127]
    row = torch.zeros(1, 128, dtype=torch.float64)
    row[0, 0], row[0, 1:1 + x.numel()] = 440 / factor, x      # (exponent 0)
    x = torch.cat((row, row), 1).float().to(dev())
    ops, cache = _ops(torch.float32), code_pools(1, 1, 128, 128, dev())
    zero = torch.zeros(1, dtype=torch.int32, device=dev())
    ops.kv_store(x, cache, zero, 0, freq=_freq(64), pos=zero, pairing=pairing, factor=factor)
    want = x[0, :128].double() * factor
    assert int(cache.k_exp[0, 0, 0]) == 127
    got, wide = grid.to(dev())[(cache.k[0, 0, 0] & 127).long()], grid.to(dev())
    best = (want.abs()[:, None] - wide[None]).abs().amin(1)
    assert torch.equal((want.abs() - got).abs(), best)
    # and the queries' f32 results are those of the 64-bit factor, rounded once
    out = ops.rope(x[:, :128].contiguous(), _freq(64), zero, 1, 128, pairing=pairing, factor=factor)
    assert ((out[0].double() - want).abs() <= 1.01 * 2.0 ** -23 * want.abs()).all()
