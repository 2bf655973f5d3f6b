"""Rotary positions, the quantised cache and attention of drafted tokens without a GPU: masks of trees, and which calls are refused before anything is enqueued."""
import pytest
import torch

from omniserve_amd.backend import lm

BF16, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


@pytest.fixture(params=[BF16, F32])
def ops(request):
    return lm.lm_ops(request.param)


def test_masks_of_a_tree():
    mask, depth = lm.tree_masks([-1, 0, 0, 2, -1])
    assert mask.tolist() == [[0b1], [0b11], [0b101], [0b1101], [0b10000]] and depth.tolist() == [0, 1, 1, 2, 0]
    assert mask.dtype == I64 and depth.dtype == I32


def test_masks_of_long_chains():
    """Bits 63, 64 and beyond, across words"""
    mask, depth = lm.tree_masks(list(range(-1, 129)))
    assert mask.shape == (130, 3) and depth.tolist() == list(range(130))
    for i in (0, 62, 63, 64, 127, 128, 129):
        bits = [j for j in range(192) if int(mask[i, j // 64]) >> (j % 64) & 1]
        assert bits == list(range(i + 1))


def test_masks_of_nothing():
    mask, depth = lm.tree_masks([])
    assert mask.shape == (0, 1) and depth.shape == (0,)


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 2, 0], [-2]])
def test_masks_refuse(parents):
    with pytest.raises(ValueError):
        lm.tree_masks(parents)


def test_empty_pools_hold_zeros():
    c = lm.code_pools(2, 3, 128, 64, "cpu")
    assert [tuple(t.shape) for t in c] == [(2, 3, 64, 128), (2, 3, 64, 64), (2, 3, 64), (2, 3, 64)]
    assert all(t.dtype == torch.uint8 for t in c) and int(c.k.max()) == 0 and int(c.k_exp.min()) == 27 == int(c.v_exp.max())


def test_stretched_frequencies():
    """Fast pairs as they are, slow ones divided by the factor, no step between, and the known factor of the scores"""
    import math

    from omniserve_amd.rope import inverse_frequencies, stretched_frequencies
    for dims, base, factor, original in ((128, 10000.0, 16.0, 4096), (64, 500000.0, 8.0, 8192), (2, 10000.0, 4.0, 2048)):
        plain, (got, scale) = inverse_frequencies(dims, base), stretched_frequencies(dims, base, factor, original)
        assert scale == 0.1 * math.log(factor) + 1.0 and len(got) == dims // 2
        share = [(1.0 - g / f) / (1.0 - 1.0 / factor) for f, g in zip(plain, got)]      # 0: kept, 1: divided
        turns = [original * f / (2 * math.pi) for f in plain]
        assert all(-1e-12 <= x <= 1 + 1e-12 for x in share) and share == sorted(share)
        assert all(abs(x) < 1e-12 for x, t in zip(share, turns) if t >= 32.0 * base ** (2.0 / dims))
        assert all(abs(x - 1) < 1e-12 for x, t in zip(share, turns) if t <= base ** (-2.0 / dims))
    assert stretched_frequencies(64, 10000.0, 1.0, 4096)[0] == pytest.approx(inverse_frequencies(64, 10000.0), rel=1e-15) and stretched_frequencies(64, 10000.0, 1.0, 4096)[1] == 1.0
    for bad in ((3, 10000.0, 2.0, 4096), (0, 10000.0, 2.0, 4096), (64, 10000.0, 0.5, 4096), (64, 10000.0, 2.0, 4096, 1.0, 2.0)):
        with pytest.raises(ValueError):
            stretched_frequencies(*bad)


def refuse(match, call, *args, **kw):
    with pytest.raises(ValueError, match=match):
        call(*args, **kw)


def test_rope_refuses(ops):
    t = ops.dtype
    x, freq, pos = torch.zeros(3, 256, dtype=t), torch.ones(32, dtype=torch.float64), torch.zeros(3, dtype=I32)
    refuse("GPU", ops.rope, x, freq, pos, 4, 64)                                   # (all is well but for the device)
    refuse("x:", ops.rope, x, freq, pos, 5, 64)
    refuse("x:", ops.rope, x.to(torch.float16), freq, pos, 4, 64)
    refuse("x:", ops.rope, x.t().contiguous().t(), freq, pos, 4, 64)
    refuse("x:", ops.rope, x[0], freq, pos, 4, 64)
    refuse("freq", ops.rope, x, freq.float(), pos, 4, 64)
    refuse("freq", ops.rope, x, torch.ones(33, dtype=torch.float64), pos, 4, 64)
    refuse("freq", ops.rope, x, freq[:0], pos, 4, 64)
    refuse("pos", ops.rope, x, freq, pos[:2], 4, 64)
    refuse("pos", ops.rope, x, freq, pos.long(), 4, 64)
    refuse("pairing", ops.rope, x, freq, pos, 4, 64, pairing="thirds")
    refuse("heads", ops.rope, x, freq, pos, 0, 64)
    refuse("out", ops.rope, x, freq, pos, 4, 64, out=x[:2])
    refuse("out", ops.rope, x, freq, pos, 4, 64, out=x[:, :255])


def test_store_and_load_refuse(ops):
    t = ops.dtype
    cache = lm.code_pools(2, 2, 64, 128, "cpu")
    x, slot, freq, pos = torch.zeros(3, 4 * 64 + 2 * 64 + 2 * 128, dtype=t), torch.zeros(3, dtype=I32), torch.ones(32, dtype=torch.float64), torch.zeros(3, dtype=I32)
    refuse("GPU", ops.kv_store, x, cache, slot, 4, freq=freq, pos=pos)
    refuse("GPU", ops.kv_store, x, cache, slot, 4)
    refuse("x:", ops.kv_store, x, cache, slot, 5)
    refuse("heads", ops.kv_store, x, cache, slot, -1)
    refuse("slot", ops.kv_store, x, cache, slot[:2], 4)
    refuse("slot", ops.kv_store, x, cache, slot.long(), 4)
    refuse("freq", ops.kv_store, x, cache, slot, 4, freq=freq)
    refuse("freq", ops.kv_store, x, cache, slot, 4, pos=pos)
    refuse("rows", ops.kv_store, x, cache, slot, 4, rows=pos[:2])
    refuse("queries", ops.kv_store, x, cache, slot, 4, freq=freq, pos=pos, rows=pos, q_out=x)
    refuse("queries", ops.kv_store, x, cache, slot, 4, q_out=x)
    refuse("q_out", ops.kv_store, x, cache, slot, 4, freq=freq, pos=pos, q_out=x[:, :255])
    refuse("cache", ops.kv_store, x, cache[:2], slot, 4)
    refuse("pools", ops.kv_store, x, (cache.k[:, :, :32].contiguous(),) + cache[1:], slot, 4)
    refuse("pools", ops.kv_store, x, (cache.k[:1],) + cache[1:], slot, 4)
    refuse("pools", ops.kv_store, x, lm.KvCodes(*(c.view(torch.int8) for c in cache)), slot, 4)
    refuse("exponents", ops.kv_store, x, cache[:2] + (cache.k_exp[:1], cache.v_exp), slot, 4)
    refuse("pools", ops.kv_load, (torch.zeros(2, 2, 64, 96, dtype=torch.uint8),) + cache[1:], slot)
    refuse("GPU", ops.kv_load, cache, slot)
    refuse("slot", ops.kv_load, cache, slot.view(1, 3))
    out = torch.zeros(3, 128, dtype=t), torch.zeros(3, 256, dtype=t)
    refuse("GPU", ops.kv_load, cache, slot, out=out)
    refuse("out", ops.kv_load, cache, slot, out=(out[0][:2], out[1]))
    refuse("out", ops.kv_load, cache, slot, out=(out[0], torch.zeros(3, 257, dtype=t)[:, 1:]))


def test_tree_attention_refuses(ops):
    t = ops.dtype
    cache = lm.code_pools(3, 2, 64, 128, "cpu")
    plain = (torch.zeros(3, 2, 64, 64, dtype=t), torch.zeros(3, 2, 64, 128, dtype=t))
    n = 5
    ok = dict(q=torch.zeros(n, 4 * 64, dtype=t), k=torch.zeros(n, 2 * 64, dtype=t), v=torch.zeros(n, 2 * 128, dtype=t), mask=torch.zeros(n, 1, dtype=I64),
              first=torch.zeros(3, dtype=I32), pos=torch.zeros(n, dtype=I32), cache=cache, bt=torch.zeros(2, 4, dtype=I32), length=torch.zeros(2, dtype=I32), scale=0.1, window=None,
              max_draft=3, max_context=100, out=None)
    bad = lambda match, **kw: refuse(match, ops.tree_attn, **{**ok, **kw})      # noqa: E731
    bad("GPU")
    bad("GPU", cache=plain)
    bad("GPU", window=7, max_draft=64)
    bad("pools", cache=tuple(p.to(torch.float16) for p in plain))
    bad("cache", cache=cache[:3])
    for i in range(4):      # (a view that begins between two 16-byte boundaries)
        odd = torch.zeros(cache[i].numel() + 4, dtype=torch.uint8)[4:].view(cache[i].shape)
        bad("16 bytes", cache=(*cache[:i], odd, *cache[i + 1:]))
    bad("q:", q=torch.zeros(n, 3 * 64, dtype=t))
    bad("q:", q=torch.zeros(n, 4 * 64 + 1, dtype=t))
    bad("q:", q=ok["q"].to(torch.float16))
    bad("k:", k=ok["k"][:, :127])
    bad("k:", k=ok["k"][:4])
    bad("v:", v=torch.zeros(n, 2 * 128 + 1, dtype=t)[:, 1:])
    bad("mask", mask=ok["mask"].int())
    bad("mask", mask=ok["mask"][:4])
    bad("mask", max_draft=65)
    bad("mask", max_draft=-1)
    bad("first", first=torch.zeros(2, dtype=I32))
    bad("pos", pos=ok["pos"].long())
    bad("length", length=torch.zeros(2, dtype=I64))
    bad("bt", bt=torch.zeros(3, 4, dtype=I32))
    bad("bt", bt=torch.zeros(4, 2, dtype=I32).t())
    bad("scale", scale=0.0)
    bad("scale", scale=float("nan"))
    for scale in (-0.1, float("inf"), 1e300, 2.0 ** 61, 2.0 ** -61, 1e-300):
        bad("scale", scale=scale)
    bad("GPU", scale=2.0 ** -60)
    bad("GPU", scale=2.0 ** 60)
    bad("window", window=0)
    bad("window", window=-3)
    bad("max_context", max_context=-1)
    bad("out", out=torch.zeros(n, 4 * 128 - 1, dtype=t))
    bad("out", out=torch.zeros(4, 4 * 128, dtype=t))
    bad("block table", cache=lm.code_pools(0, 2, 64, 128, "cpu"))


def test_library_refuses(ops):
    """The C entries' own checks, which come before any launch"""
    h, f = ops._h, 0.5
    assert h.lm_rope(64, 0, 64, 0, 64, 0, 64, 0, f, 1, 1, 64, None) == -22              # nothing turns
    assert h.lm_rope(64, 0, 64, 0, 64, 33, 64, 0, f, 1, 1, 64, None) == -22
    assert h.lm_rope(64, 0, 64, 0, None, 8, 64, 0, f, 1, 1, 64, None) == -22
    assert h.lm_rope(None, 0, 64, 0, 64, 8, 64, 0, f, 1, 1, 64, None) == -22
    assert h.lm_rope(64, 0, 64, 0, 64, 8, 64, 0, f, -1, 1, 64, None) == -22
    assert h.lm_rope(None, 0, None, 0, 64, 8, 64, 0, f, 0, 1, 64, None) == 0            # no tokens: nothing to do
    store = lambda rows=None, q=None, pages=3, tokens=1, H=2, G=1, dk=64, dv=64, kc=64: h.lm_kv_store(      # noqa: E731
        64, 256, 1, rows, None, 0, None, 0, f, q, 0, 64, kc, 64, 64, 64, pages, tokens, H, G, dk, dv, None)
    assert store(tokens=0) == 0 and store(tokens=-1) == store(dk=96) == store(dv=32) == store(G=0) == store(kc=65) == store(kc=None) == store(pages=1 << 26) == -22
    assert store(q=64, H=0) == store(q=64, rows=64) == -22
    assert h.lm_kv_load(64, 64, 64, 64, 64, 64, 64, 64, 3, 64, 0, 1, 64, 64, None) == 0
    assert h.lm_kv_load(64, 64, 64, 64, 64, 64, 64, 64, 3, None, 1, 1, 64, 64, None) == -22
    assert h.lm_kv_load(64, 65, 64, 64, 64, 64, 64, 64, 3, 64, 1, 1, 64, 64, None) == -22
    tree = lambda B=1, n=1, draft=1, H=2, G=1, dk=64, dv=64, width=2, pages=3, context=100, scale=f, window=1, ldq=128, ke=64, ve=64, q=64: h.lm_tree_attn(      # noqa: E731
        q, ldq, 64, 64, 64, 64, 64, 64, ke, ve, pages, 64, width, width, 64, 64, 64, 64, 1, 64, 128, None, scale, window, B, n, draft, context, H, G, dk, dv, None)
    assert tree(B=0) == tree(n=0) == tree(draft=0) == 0
    for bad in (dict(H=3, G=2), dict(dk=80), dict(dv=192), dict(pages=0), dict(context=-1), dict(width=1 << 26, pages=1 << 20), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2.0 ** -61), dict(scale=2.0 ** 61), dict(window=0),
                dict(ldq=129), dict(ke=72), dict(ve=72), dict(ve=68), dict(ke=None), dict(ve=None), dict(q=None), dict(q=72), dict(B=-1)):
        assert tree(**bad) == -22, bad


def test_scratch_of_cut_keys(ops):
    """Room for pieces of the keys where workgroups are few and contexts long; none for short contexts and for batches that fill the chip several times; no
    more than the pieces there can be"""
    room = ops._h.lm_tree_attn_scratch
    for codes in (0, 1):
        assert room(1, 1, 0, 32, 8, 128, 128, codes) == 0 and room(1, 1, 64, 32, 8, 128, 128, codes) == 0
        assert room(1, 1, 100000, 32, 8, 128, 128, codes) > 0 and room(1, 1, 2 ** 31 - 1, 1, 1, 128, 128, codes) > 0
        assert room(512, 1, 100000, 32, 8, 128, 128, codes) == 0
        # few keys: pieces of four tiles, one more a segment (a tile is 64 keys of codes, 32 of elements; one of drafted tokens), and where each segment is cut
        tiles = 8 * (2000 // (64 if codes else 32) + 1 + 1)
        assert room(1, 1, 2000, 32, 8, 128, 128, codes) == (8 + tiles // 4) * 16 * 130 + 2 * 8
    assert room(0, 1, 10000, 32, 8, 128, 128, 1) == room(1, 0, 10000, 32, 8, 128, 128, 1) == room(1, 1, 10000, 3, 2, 128, 128, 1) == room(1, 1, -1, 32, 8, 128, 128, 1) == 0
