"""Rotary positions, and keys and values in a cache of 8-bit floats, against 64 bits."""
import math

import pytest
import torch

from tests.kv_codes_util import CODE_STEP, PAGE, UNIT, code_values, decoded, row_exponent, turned
from tests.util import dev

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


def _ops(dtype):
    from omniserve_amd.backend.lm import lm_ops
    return lm_ops(dtype)


def _freq(half, base=10000.0):
    return torch.tensor([base ** (-i / half) for i in range(half)], dtype=torch.float64, device=dev())


def _positions(n, gen, far=1 << 20):
    pos = torch.randint(0, far, (n,), device=dev(), generator=gen, dtype=torch.int32)
    pos[0] = 0
    if n > 2:
        pos[1] = far - 1
    return pos


def _rope_close(got, x, freq, pos, half, pairing, factor, dtype):
    ref = turned(x, freq, pos, half, pairing, factor)
    # the pair's length bounds both results: sine and cosine in f32, two products and their sum
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if pairing == "halves" else (2 * i, 2 * i + 1)
    size = torch.zeros_like(x)
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * factor
    bound = 1.01 * UNIT[dtype] * ref.abs() + 4 * 2.0 ** -24 * size
    bound[..., 2 * half:] = 0
    assert ((got - ref).abs() <= bound).all(), float((got - ref).abs().max())


@pytest.mark.parametrize("tokens", [1, 5, 70, 1030])
@pytest.mark.parametrize("heads,dk,half", [(1, 64, 32), (5, 128, 64), (12, 128, 16), (3, 256, 128), (7, 80, 20), (2, 96, 3), (40, 128, 32), (1, 6, 2), (3, 128, 1)])
@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("dtype", TYPES)
def test_rope(dtype, pairing, heads, dk, half, tokens):
    gen = torch.Generator(device=dev()).manual_seed(tokens + dk + half)
    x = torch.randn(tokens, heads * dk, device=dev(), generator=gen).to(dtype)
    freq, pos = _freq(half), _positions(tokens, gen)
    keep = x.clone()
    got = _ops(dtype).rope(x, freq, pos, heads, dk, pairing=pairing, factor=1.25)
    assert torch.equal(x, keep) and got.shape == x.shape and got.dtype == dtype
    _rope_close(got.double().view(tokens, heads, dk), x.double().view(tokens, heads, dk), freq, pos, half, pairing, 1.25, dtype)
    # in place, as part of wider rows at an odd distance: the same bits, the neighbours untouched
    wide = torch.full((tokens, heads * dk + 13), 3.0, dtype=dtype, device=dev())
    part = wide[:, 5:5 + heads * dk]
    part.copy_(x)
    assert _ops(dtype).rope(part, freq, pos, heads, dk, pairing=pairing, factor=1.25, out=part) is part
    assert torch.equal(part, got) and bool((wide[:, :5] == 3).all()) and bool((wide[:, 5 + heads * dk:] == 3).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_rope_leaves_empty_places(dtype):
    gen = torch.Generator(device=dev()).manual_seed(3)
    x = torch.randn(9, 4 * 64, device=dev(), generator=gen).to(dtype)
    pos = _positions(9, gen)
    pos[4] = -1
    out = torch.full_like(x, 7.0)
    _ops(dtype).rope(x, _freq(32), pos, 4, 64, out=out)
    assert bool((out[4] == 7).all()) and not bool((out[3] == 7).any())
    keep = x[4].clone()
    _ops(dtype).rope(x, _freq(32), pos, 4, 64, out=x)
    assert torch.equal(x[4], keep) and torch.equal(x[5], out[5])


def test_rope_of_far_positions_turns_by_the_whole_angle():
    """A position that f32 angles would miss by whole turns"""
    pos = torch.tensor([2 ** 31 - 1, 2 ** 30 + 1], dtype=torch.int32, device=dev())
    x = torch.ones(2, 64, device=dev())
    got = _ops(torch.float32).rope(x, _freq(32), pos, 1, 64, pairing="halves")
    # the angle: three roundings of 2^-53 of 2^31 there, one here, times a pair's length
    ref = turned(x.double().view(2, 1, 64), _freq(32), pos, 32, "halves", 1.0).view(2, 64)
    assert ((got.double() - ref).abs() <= 8 * 2.0 ** -24 + 4 * 2.0 ** -22 * 2.0 ** 0.5).all()


def _check_codes(x, codes, exps):
    """x f64 [.., size]: the exponent is the least one, every code the nearest (ties to even) up to the accuracy of 64-bit angles"""
    assert torch.equal(exps.int() - 127, row_exponent(x).int())
    y = x / torch.exp2(exps.double() - 127)[..., None]
    grid = code_values(x.device)
    val = grid[codes.long()]
    bad = ~x.isfinite()
    assert torch.equal(val.isnan(), bad)
    y, val, codes = y[~bad], val[~bad], codes[~bad].long() & 127
    up, down = grid[(codes + 1).clamp(max=126)], grid[(codes - 1).clamp(min=0)]
    mag, m = val.abs(), y.abs()
    eps = 2.0 ** -20 * 2.0 ** -9      # f64 angles of 2^20: 2^-33 of a value up to 448, and far above the smallest step's accuracy
    assert bool(((val >= 0) == (y >= 0))[mag > 0].all())
    assert bool((m <= (mag + up) / 2 + eps)[codes < 126].all()) and bool((m >= (mag + down) / 2 - eps)[codes > 0].all())
    assert bool((m[codes == 0] <= 2.0 ** -10 + eps).all())


def _store(dtype, dk, dv, heads, kv_heads, half, tokens, pairing, seed, with_q=True, spread=0.0):
    gen = torch.Generator(device=dev()).manual_seed(seed)
    ops = _ops(dtype)
    from omniserve_amd.backend.lm import code_pools
    nq, nk, nv = heads * dk, kv_heads * dk, kv_heads * dv
    wide = torch.randn(tokens, nq + nk + nv + 24, device=dev(), generator=gen).mul_(torch.exp(spread * torch.randn(tokens, 1, device=dev(), generator=gen))).to(dtype)
    x = wide[:, 8:8 + nq + nk + nv]
    pages = tokens // PAGE + 3
    cache = code_pools(pages, kv_heads, dk, dv, dev())
    for t in cache[:2]:
        t.fill_(0x55)
    places = torch.randperm(pages * PAGE, device=dev(), generator=gen)
    slot = places[:tokens].int()
    if tokens > 4:
        slot[2], slot[3] = -1, pages * PAGE      # not stored
    freq, pos = (_freq(half), _positions(tokens, gen)) if half else (None, None)
    q = torch.zeros(tokens, nq, dtype=dtype, device=dev()) if with_q and half else None
    before = x.clone()
    ops.kv_store(x, cache, slot, heads, freq=freq, pos=pos, pairing=pairing, factor=1.125, q_out=q)
    assert torch.equal(x, before)
    live = (slot >= 0) & (slot < pages * PAGE)
    page, off = (slot[live] // PAGE).long(), (slot[live] % PAGE).long()
    kx = x[:, nq:nq + nk].double().view(tokens, kv_heads, dk)
    if half:
        kx = turned(kx, freq, pos, half, pairing, 1.125)
    vx = x[:, nq + nk:].double().view(tokens, kv_heads, dv)
    _check_codes(kx[live], cache.k[page, :, off], cache.k_exp[page, :, off])
    _check_codes(vx[live], cache.v[page, :, off], cache.v_exp[page, :, off])
    if q is not None:
        _rope_close(q.double().view(tokens, heads, dk), x[:, :nq].double().view(tokens, heads, dk), freq, pos, half, pairing, 1.125, dtype)
    # nothing else was written
    rest = torch.ones(pages * PAGE, dtype=torch.bool, device=dev())
    rest[slot[live].long()] = False
    for t in cache[:2]:
        assert bool((t.transpose(1, 2).reshape(pages * PAGE, -1)[rest] == 0x55).all())
    # read back: the same values, zeros outside
    k, v = ops.kv_load(cache, slot)
    assert k.dtype == dtype and v.shape == (tokens, nv)
    for y, c, e in ((k, cache.k, cache.k_exp), (v, cache.v, cache.v_exp)):
        want = torch.zeros(tokens, y.shape[1], dtype=torch.float64, device=dev())
        want[live] = decoded(c[page, :, off], e[page, :, off]).flatten(1)
        assert torch.equal(y.double(), want)      # (codes times powers of two are elements)
    return cache


@pytest.mark.parametrize("tokens", [1, 17, 63, 700, 4100])
@pytest.mark.parametrize("dk,dv,heads,kv_heads,half", [(128, 128, 8, 2, 64), (64, 128, 3, 3, 32), (256, 64, 4, 1, 16), (128, 256, 14, 2, 7), (64, 64, 1, 1, 0), (128, 128, 5, 5, 3)])
@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("dtype", TYPES)
def test_store_and_load(dtype, pairing, dk, dv, heads, kv_heads, half, tokens):
    _store(dtype, dk, dv, heads, kv_heads, half, tokens, pairing, tokens + dk, spread=2.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_store_of_special_rows(dtype):
    """Zeros, ties, the largest and smallest rows, one element at the borders of a power of two, NaN and infinities"""
    from omniserve_amd.backend.lm import NOTHING, code_pools
    ops, d = _ops(dtype), 64
    big = torch.finfo(dtype).max
    rows = torch.zeros(10, d, dtype=torch.float64)
    rows[1] = torch.arange(d).double() * 0.0625 + 1.0          # with ties
    rows[2, 3], rows[3, 3] = 448.0, 448.0 * (1 + 2.0 ** -7)     # the last that a power holds, the first that it does not
    rows[4], rows[4, 0] = 2.0 ** -126, 2.0 ** -120              # smaller than any power the cache has
    rows[5] = big
    rows[6], rows[6, 1], rows[6, 2], rows[6, 3] = 1.5, math.inf, -math.inf, math.nan
    rows[7] = math.nan
    rows[8], rows[8, 7] = 2.0 ** -12, 1.0                       # below the smallest code
    rows[9, 5] = -0.0
    x = rows.to(dtype).to(dev())
    cache = code_pools(1, 1, d, d, dev())
    slot = torch.arange(10, dtype=torch.int32, device=dev())
    ops.kv_store(torch.cat((x, -x), 1), cache, slot, 0)
    k, v = ops.kv_load(cache, slot)
    e = cache.k_exp[0, 0, :10].int() - 127
    assert e.tolist()[0] == NOTHING - 127 and e.tolist()[2:4] == [0, 1] and e.tolist()[4] == -100 and e.tolist()[5] == 120 and e.tolist()[7] == -100
    for i in (0, 1, 2, 3, 4, 6, 8, 9):
        _check_codes(x[i].double(), cache.k[0, 0, i], cache.k_exp[0, 0, i])
    assert bool((k[5] == 240 * 2.0 ** 120).all())               # finite stays finite
    assert bool(k[7].isnan().all()) and bool((k[0] == 0).all()) and k[6].isnan().nonzero().flatten().tolist() == [1, 2, 3]
    assert torch.equal(torch.nan_to_num(v.float()), torch.nan_to_num(-k.float()))


def test_store_of_kept_rows():
    """Drafted tokens are stored by row number, in any order; rows outside x are none; queries stay"""
    from omniserve_amd.backend.lm import code_pools
    ops = _ops(torch.bfloat16)
    gen = torch.Generator(device=dev()).manual_seed(8)
    x = torch.randn(11, 2 * 128 + 2 * 128, device=dev(), generator=gen).to(torch.bfloat16)
    cache = code_pools(2, 1, 128, 128, dev())
    rows = torch.tensor([7, 0, 11, -1, 3], dtype=torch.int32, device=dev())
    slot = torch.tensor([64, 5, 6, 7, 127], dtype=torch.int32, device=dev())
    ops.kv_store(x, cache, slot, 2, rows=rows)
    k, v = ops.kv_load(cache, slot)
    for i, r in ((0, 7), (1, 0), (4, 3)):
        page, off = int(slot[i]) // PAGE, int(slot[i]) % PAGE
        _check_codes(x[r, 256:384].double(), cache.k[page, 0, off], cache.k_exp[page, 0, off])
        assert ((v[i].double() - x[r, 384:].double()).abs() <= CODE_STEP * x[r, 384:].double().abs() + 2.0 ** -10 * torch.exp2(cache.v_exp[page, 0, off].double() - 127)).all()
    assert bool((k[2:4] == 0).all())


def test_far_pages():
    """Offsets that pass 32 bits"""
    from omniserve_amd.backend.lm import KvCodes
    ops = _ops(torch.bfloat16)
    pages, G, d = 70000, 4, 128      # 2.3e9 bytes a pool
    cache = KvCodes(*(torch.zeros(pages, G, PAGE, d, dtype=torch.uint8, device=dev()) for _ in range(2)), *(torch.zeros(pages, G, PAGE, dtype=torch.uint8, device=dev()) for _ in range(2)))
    gen = torch.Generator(device=dev()).manual_seed(9)
    x = torch.randn(3, 2 * G * d, device=dev(), generator=gen).to(torch.bfloat16)
    slot = torch.tensor([pages * PAGE - 1, 0, 66000 * PAGE + 5], dtype=torch.int32, device=dev())
    ops.kv_store(x, cache, slot, 0)
    k, v = ops.kv_load(cache, slot)
    for y, at in ((k, 0), (v, G * d)):
        want = x[:, at:at + G * d].double().view(3, G, d)
        step = torch.exp2(row_exponent(want).double())[..., None]
        assert ((y.double().view(3, G, d) - want).abs() <= CODE_STEP * want.abs() + 2.0 ** -10 * step).all()


@pytest.mark.parametrize("tokens", [1, 300])
def test_captured_store_and_load(tokens):
    """Replayed with new inputs, eager work and synchronisations between"""
    from omniserve_amd.backend.lm import code_pools
    ops = _ops(torch.bfloat16)
    gen = torch.Generator(device=dev()).manual_seed(10)
    new = lambda: torch.randn(tokens, 6 * 128, device=dev(), generator=gen).to(torch.bfloat16)      # noqa: E731
    x, pages = new(), tokens // PAGE + 1
    cache, other = code_pools(pages, 1, 128, 128, dev()), code_pools(pages, 1, 128, 128, dev())
    slot = torch.randperm(pages * PAGE, device=dev(), generator=gen)[:tokens].int()
    freq, pos, q = _freq(64), _positions(tokens, gen), torch.zeros(tokens, 4 * 128, dtype=torch.bfloat16, device=dev())

    def step(cache, q):
        ops.kv_store(x, cache, slot, 4, freq=freq, pos=pos, pairing="halves", q_out=q)
        return ops.kv_load(cache, slot)

    step(cache, q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        k, v = step(cache, q)
    for _ in range(4):
        x.copy_(new())
        pos.copy_(_positions(tokens, gen))
        g.replay()
        q2 = torch.zeros_like(q)
        k2, v2 = step(other, q2)
        torch.cuda.synchronize()
        assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(q, q2)


def test_queries_turned_in_place():
    from omniserve_amd.backend.lm import code_pools
    ops = _ops(torch.bfloat16)
    gen = torch.Generator(device=dev()).manual_seed(11)
    x = torch.randn(33, 6 * 128, device=dev(), generator=gen).to(torch.bfloat16)
    freq, pos, slot = _freq(48), _positions(33, gen), torch.arange(33, dtype=torch.int32, device=dev())
    pos[9] = -1
    a, b = code_pools(1, 1, 128, 128, dev()), code_pools(1, 1, 128, 128, dev())
    q = x[:, :512].clone()
    ops.kv_store(x, a, slot, 4, freq=freq, pos=pos, q_out=q)
    y = x.clone()
    ops.kv_store(y, b, slot, 4, freq=freq, pos=pos, q_out=y)
    assert torch.equal(y[:, :512], q) and torch.equal(y[:, 512:], x[:, 512:]) and torch.equal(q[9], x[9, :512])
    assert all(torch.equal(s, t) for s, t in zip(a, b)) and int(a.k[0, 0, 9].max()) == 0      # (an empty place is not stored)
