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


@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("dk,dv,half", [(128, 128, 64), (64, 256, 7), (256, 64, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kept_rows_are_stored_as_a_prompt_is(dtype, dk, dv, half, pairing):
    """Rows named by number, any order, twice and outside x, turned as they are stored: the codes of the same rows stored in order, and empty places stay"""
    from omniserve_amd.backend.lm import code_pools
    ops, H, G, n = _ops(dtype), 3, 2, 23
    gen = torch.Generator(device=dev()).manual_seed(dk + half)
    x = torch.randn(n, (H + G) * dk + G * dv, device=dev(), generator=gen).to(dtype)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())      # noqa: E731
    rows, pos = [22, 0, 5, 5, -1, 23, 7, 1, 9], [100000, 3, 70, 71, 5, 5, 0, -1, 12]
    a, b = code_pools(2, G, dk, dv, dev()), code_pools(2, G, dk, dv, dev())
    slot = [127, 0, 64, 3, 4, 5, 6, 7, 128]
    ops.kv_store(x, a, ints(slot), H, rows=ints(rows), freq=_freq(half), pos=ints(pos), pairing=pairing, factor=1.25)
    good = [i for i in range(9) if 0 <= rows[i] < n]
    ops.kv_store(x[[rows[i] for i in good]], b, ints([slot[i] for i in good]), H, freq=_freq(half), pos=ints([pos[i] for i in good]), pairing=pairing, factor=1.25)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert int((a.k_exp[:, 0] != 27).sum()) == 5      # (seven named rows, one of an empty place and one behind the pools)


def test_drafts_are_kept_as_they_would_have_been_a_prompt():
    """A prompt, a tree of drafted tokens over it, and the ones that were kept: turned for attention, and stored from their unturned rows, so that the cache is the
    one that a longer prompt leaves"""
    from omniserve_amd.backend.lm import code_pools, tree_masks
    from tests.kv_codes_util import attention, attention_bound, decoded
    ops, heads, kv_heads, n = _ops(torch.bfloat16), 8, 2, 100
    gen = torch.Generator(device=dev()).manual_seed(1)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())      # noqa: E731
    qkv, draft = (torch.randn(t, (heads + 2 * kv_heads) * 128, device=dev(), generator=gen).to(torch.bfloat16) for t in (n, 4))
    freq, cache, other, block_table = _freq(64), *(code_pools(3, kv_heads, 128, 128, dev()) for _ in range(2)), ints([[2, 0]])
    slots = lambda at: ints([int(block_table[0, i // 64]) * 64 + i % 64 for i in at])      # noqa: E731
    prompt = torch.cat((qkv, draft[[0, 1, 3]]))
    ops.kv_store(prompt, other, slots(range(n + 3)), heads, freq=freq, pos=ints(list(range(n + 3))))
    ops.kv_store(qkv, cache, slots(range(n)), heads, freq=freq, pos=ints(list(range(n))), q_out=qkv[:, :heads * 128])
    length, first = ints([n]), ints([0, 4])
    mask, depth = (t.to(dev()) for t in tree_masks([-1, 0, 0, 1]))
    pos = length + depth
    turned = ops.rope(draft, freq, pos, heads + kv_heads, 128)
    q, k, v = turned[:, :heads * 128], turned[:, heads * 128:], draft[:, (heads + kv_heads) * 128:]
    o = ops.tree_attn(q, k, v, mask, first, pos, cache, block_table, length, 128 ** -0.5, max_draft=4, max_context=128)
    ref = attention(q.double().view(4, heads, 128), k.double().view(4, kv_heads, 128), v.double().view(4, kv_heads, 128), mask, first.cpu(), pos,
                    *(decoded(c, e) for c, e in zip(cache[:2], cache[2:])), block_table, length, 128 ** -0.5, 1 << 30, 4, heads // kv_heads)
    assert ((o.double().view(4, heads, 128) - ref[0]).abs() <= attention_bound(torch.bfloat16, True, 128, *ref)).all()
    kept = ints([0, 1, 3])
    ops.kv_store(draft, cache, slots(range(n, n + 3)), heads, rows=kept, freq=freq, pos=pos[kept])
    assert all(torch.equal(s, t) for s, t in zip(cache, other))
