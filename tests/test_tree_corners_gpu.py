"""Attention of drafted tokens where it can go wrong: values that are not finite in every kind of tile, exponents and magnitudes far apart, segments cut
into many pieces, few and many rows alike.  Against 64 bits; infinities and NaN are told apart."""
import math

import pytest
import torch

from tests.kv_codes_util import PAGE, attention, attention_bound
from tests.test_tree_attn_gpu import NO_WINDOW, Case
from tests.util import dev

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DRAFTS = [1, 12, 20, 64, 150]      # rows of 2 heads per kv head: one block of 16, two, and the kernel of many rows with 2, 4 and 8 waves


def _limits(c, window):
    """[tokens, heads, dv]: 0 where every value that a row sees is finite, else what their sum is, whatever the weights: inf, -inf or nan"""
    n, (kpool, vpool) = c.q.shape[0], c.pools()
    out = torch.zeros(n, c.H, c.dv, dtype=torch.float64, device=dev())
    first = c.first.tolist()
    for b, ln in enumerate(c.length.tolist()):
        f0, t = first[b], min(first[b + 1] - first[b], c.max_draft)
        if t <= 0:
            continue
        pages = c.bt[b, :-(-ln // PAGE)].long()
        v = torch.cat((vpool[pages].transpose(1, 2).reshape(-1, c.G, c.dv)[:ln], c.v[f0:f0 + t].double().view(t, c.G, c.dv)))
        p, j = c.pos[f0:f0 + t].long(), torch.arange(t, device=dev())
        bits = (c.mask[f0:f0 + t][:, j // 64] >> (j % 64)) & 1
        where = torch.cat((torch.arange(ln, device=dev()), p))
        seen = torch.cat((torch.ones(t, ln, dtype=torch.bool, device=dev()), bits.bool()), 1) & (where[None] > p[:, None] - window)
        for key in (~v.isfinite()).flatten(1).any(1).nonzero()[:, 0].tolist():
            bad = torch.where(v[key].isfinite(), 0.0, v[key]).repeat_interleave(c.H // c.G, 0)
            out[f0:f0 + t] += torch.where(seen[:, key, None, None], bad[None], 0.0)
    return out


def _check(c, got, window=None):
    """Where nothing but finite values is seen: within the bound of the finite ones; elsewhere the right kind of infinity, or NaN"""
    n, window = c.q.shape[0], window or NO_WINDOW
    want = _limits(c, window)
    assert not bool((c.first[1:] - c.first[:-1] > c.max_draft).any())
    ref = attention(c.q.double().view(n, c.H, c.dk), c.k.double().view(n, c.G, c.dk), c.v.double().view(n, c.G, c.dv).nan_to_num(0, 0, 0), c.mask, c.first.cpu(), c.pos,
                    *(t.nan_to_num(0, 0, 0) for t in c.pools()), c.bt, c.length, c.scale, window, c.max_draft, c.H // c.G)
    got = got.double().view(n, c.H, c.dv)
    sick = want != 0      # (NaN is not 0)
    assert torch.equal(got[sick].isnan(), want[sick].isnan()) and torch.equal(got[sick].nan_to_num(0), want[sick].nan_to_num(0))
    over = ((got - ref[0]).abs() / attention_bound(c.dtype, c.codes, c.dk, *ref))[~sick]
    assert over.numel() == 0 or float(over.max()) <= 1.0, float(over.max())


def _spoil(c, b, key, bad, col=5):
    """a cached value of sequence b"""
    page, at = int(c.bt[b, key // PAGE]), key % PAGE
    c.cache[1][page, 0, at, col] = 0x7f if c.codes else bad


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_bad_value_of_the_last_page_reaches_every_row(dtype, codes, draft):
    """The last context tile, partly filled, holds it; drafted tiles follow"""
    for n in (70, 300, 1001):
        c = Case(dtype, codes, 128, 64, 4, 2, [(n, draft), (n // 2, draft)], seed=draft + n)
        _spoil(c, 0, n - 1, -math.inf)
        _spoil(c, 1, n // 2 - 1, math.inf, 63)
        _check(c, c.run())


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 256)])
@pytest.mark.parametrize("heads", [2, 64])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_bad_value_in_any_of_many_pieces(dtype, bad, heads, dk, dv):
    """One token whose keys are cut into more pieces than a row has lanes when they are joined; the value lies in the partly filled last page, behind all others"""
    c = Case(dtype, False, dk, dv, heads, 2, [(9001, 1)], seed=dk + heads)
    c.scale = 2.0 ** -9      # (weights of one size)
    _spoil(c, 0, 9000, bad)
    _check(c, c.run())


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("context", [70, 3000])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_an_infinite_value_of_no_weight(dtype, codes, context, draft):
    """Scores so far apart that the weight of the infinite value, and the factor of the piece that holds it, are zero in 32 bits: it counts all the same"""
    for scale in (8.0, 30.0):
        c = Case(dtype, codes, 64, 64, 4, 2, [(context, draft), (context - 1, draft)], kind="chain", seed=draft)
        c.scale = scale
        c.v[0, 7], c.v[draft, 100] = math.inf, -math.inf
        if not codes:
            _spoil(c, 0, context - 1, math.inf)
        _check(c, c.run())


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("context,scale", [(300, None), (300, 8.0), (5000, None), (5000, 8.0)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinite_values_in_full_pages(dtype, context, scale, draft):
    """Infinities of elements in pages that every row sees whole: the sum of such a row is infinite, of both signs NaN, and nothing else is touched"""
    c = Case(dtype, False, 128, 64, 4, 2, [(context, draft), (context // 3, draft)], seed=draft)
    c.scale = scale or c.scale
    _spoil(c, 0, 3, math.inf, 0)
    _spoil(c, 0, context // 2, -math.inf, 1)
    _spoil(c, 0, 40, math.inf, 2)
    _spoil(c, 0, context // 2 + 33, -math.inf, 2)
    _spoil(c, 1, 20, math.nan, 9)
    _check(c, c.run())


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("codes", [True, False])
def test_scores_are_summed_in_32_bits(codes, dk, draft):
    """Queries and keys with a few channels much larger than the others, of either sign: the largest products cancel or outweigh the rest, which counts all the same"""
    c = Case(BF16, codes, dk, 64, 4, 2, [(500, draft), (70, draft)], seed=draft + dk)
    q, k = c.q.view(-1, 4, dk), c.k.view(-1, 2, dk)
    q[..., [0, 7, dk - 1]] *= 30
    k[..., [0, 7, dk - 1]] *= 8
    if codes:
        c.cache[0][..., [0, 7, dk - 1]] = torch.where(c.cache[0][..., [0, 7, dk - 1]] > 127, 0xf6, 0x76).to(torch.uint8)
    n = c.q.shape[0]
    ref = attention(c.q.double().view(n, c.H, dk), c.k.double().view(n, c.G, dk), c.v.double().view(n, c.G, 64), c.mask, c.first.cpu(), c.pos, *c.pools(), c.bt, c.length, c.scale,
                    NO_WINDOW, c.max_draft, 2)
    over = (c.run().double().view(n, 4, 64) - ref[0]).abs() / attention_bound(BF16, codes, dk, *ref[:5], 0.0)      # (no term for queries in codes)
    assert float(over.max()) <= 1.0, float(over.max())


@pytest.mark.parametrize("loud", [2.0 ** 16, 2.0 ** 40, 2.0 ** 100, 2.0 ** 120])
@pytest.mark.parametrize("draft", [2, 12, 20, 64, 150])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_loud_drafted_value_is_its_own_affair(dtype, draft, loud):
    """A drafted token of large values, and one of tiny ones, in the same tile as tokens that do not see them, or hardly"""
    for kind in ("tree", "chain"):
        c = Case(dtype, True, 64, 128, 4, 2, [(200, draft), (1500, draft), (0, draft)], kind=kind, seed=draft)
        q, k = c.q.view(-1, 4, 64), c.k.view(-1, 2, 64)
        q[..., 0] = 8
        for b in range(3):
            f0, at = int(c.first[b]), draft // 2
            c.v[f0 + at] *= loud
            c.v[f0 + draft - 1] /= loud
            if b == 1:      # those who see it do so faintly
                k[f0 + at, :, 0] = -40
                continue
            bit = 1 << at % 64
            c.mask[[f0 + i for i in range(draft) if i != at], at // 64] &= ~(bit - (1 << 64) if bit >> 63 else bit)
        _check(c, c.run())


def test_a_drafted_value_of_every_size():
    """Every drafted value has a power of two of its own, from the smallest to the largest, and none sees another"""
    for draft in (7, 32, 150):
        c = Case(BF16, True, 64, 64, 2, 1, [(130, draft)], seed=draft)
        e = torch.linspace(-60, 120, draft, device=dev()).round()
        c.v = (c.v.float().clamp(-4, 4) * torch.exp2(e)[:, None]).to(BF16)
        i = torch.arange(draft)
        c.mask.zero_()
        c.mask[i, i // 64] = torch.ones(draft, dtype=torch.int64, device=dev()) << (i % 64).to(dev())
        _check(c, c.run())
        c.length.zero_()
        _check(c, c.run())


@pytest.mark.parametrize("low,high", [(-40, 100), (-60, 60), (-60, 115), (-100, 10), (0, 115), (-99, 115)])
@pytest.mark.parametrize("first", ["quiet", "loud", "mixed"])
@pytest.mark.parametrize("draft", [1, 20, 64])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quiet_values_beside_loud_ones(dtype, draft, first, low, high):
    """Rows under 2^low and 2^high: the quiet ones take their part of the sum, and keep their results where a window hides the loud"""
    for context in (300, 3000):
        c = Case(dtype, True, 64, 64, 4, 2, [(context, draft), (context // 2, draft)], kind="chain", seed=draft + high)
        for b, n in enumerate(c.length.tolist()):
            loud = torch.arange(n, device=dev()) % 3 == 0
            loud = loud if first == "mixed" else torch.arange(n, device=dev()) < n // 2 if first == "loud" else torch.arange(n, device=dev()) >= n // 2
            for page in range(-(-n // PAGE)):
                at = loud[page * PAGE:(page + 1) * PAGE]
                c.cache[3][int(c.bt[b, page]), :, :at.numel()] = torch.where(at, 127 + high, 127 + low).to(torch.uint8)
        _check(c, c.run())
        if first == "loud":
            _check(c, c.run(window=context // 3), window=context // 3)


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_near_the_largest(dtype, codes, draft):
    """An average of numbers near the type's largest is a number"""
    big = 2.0 ** 126
    for context in (0, 300, 3000):
        c = Case(dtype, codes, 64, 64, 4, 2, [(context, draft), (context // 2, draft)], seed=draft)
        if not codes:
            c.cache[1].copy_((c.cache[1].float().clamp(-1, 1) + torch.sign(c.cache[1].float())) * 0.75 * big)
        c.v = ((c.v.float().clamp(-1, 1) + 2) * 0.6 * big).to(dtype)
        got = c.run()
        assert bool(got.isfinite().all())
        _check(c, got)


@pytest.mark.parametrize("draft", [1, 6, 13, 20, 64])
@pytest.mark.parametrize("window", [1, 40, 64, 65, 130, 1000, 2500])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_windows_over_short_and_long_contexts(dtype, codes, window, draft):
    """Few and many rows, segments in one piece and cut, whose first pages no row sees; a table of page numbers that are none in front of the windows"""
    for kind in ("chain", "tree"):
        c = Case(dtype, codes, 64, 64, 4, 2, [(3000, draft), (300, draft), (64, 1), (129, draft), (0, draft)], kind=kind, seed=window + draft)
        _check(c, c.run(window=window), window)
        want = c.run(window=window)
        for b, n in enumerate(c.length.tolist()):
            c.bt[b, :max(0, n + 1 - window) // PAGE] = -7
        assert torch.equal(c.run(window=window), want)


@pytest.mark.parametrize("draft", [1, 6, 13, 20, 64])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nothing_comes_out_of_places_that_no_row_sees(dtype, codes, bad, draft):
    """Behind the end of the last page and in front of every window, keys, values and exponents of any bits"""
    for window in (None, 120, 2000):
        c = Case(dtype, codes, 128, 64, 4, 2, [(3000, draft), (100, draft), (300, draft), (64, draft)], seed=draft)
        want = c.run(window=window)
        for b, n in enumerate(c.length.tolist()):
            for key in list(range(n, -(-n // PAGE) * PAGE)) + list(range(max(0, n + 1 - (window or n + 1)))):
                page = int(c.bt[b, key // PAGE])
                for i in (0, 1):
                    c.cache[i][page, :, key % PAGE] = 0x7f if codes else bad
                    if codes:
                        c.cache[2 + i][page, :, key % PAGE] = 255 if bad > 0 else 254
        got = c.run(window=window)
        assert torch.equal(got, want) and bool(got.isfinite().all())


@pytest.mark.parametrize("draft", [1, 6, 13, 20, 64, 150])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_values_that_some_rows_see(dtype, codes, bad, draft):
    """A cached value that is not finite (of codes: NaN), seen by the rows whose windows reach it: in the first page of a window, in the last one, in between"""
    for window in (90, 700):
        for back in (0, 1, draft // 2, 64, window - draft // 2 - 1, window - 2):
            c = Case(dtype, codes, 64, 64, 4, 2, [(3000, draft), (800, draft)], kind="chain", seed=window)
            _spoil(c, 0, 2999 - back, bad)
            _spoil(c, 1, 799 - back, bad, 17)
            _check(c, c.run(window=window), window)
