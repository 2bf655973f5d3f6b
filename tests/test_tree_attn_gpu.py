"""Attention of drafted token trees over a paged cache, quantised and not, against 64 bits; and the operators around the cache as a step uses them."""
import math

import pytest
import torch

from tests.kv_codes_util import PAGE, attention, attention_bound, decoded, quantised
from tests.util import dev

pytestmark = pytest.mark.gpu
NO_WINDOW = 1 << 30


def _ops(dtype):
    from omniserve_amd.backend.lm import lm_ops
    return lm_ops(dtype)


def _tree(n, kind, gen):
    if kind == "chain":
        return list(range(-1, n - 1))
    pick = torch.rand(n, generator=gen)
    return [int(float(pick[i]) * (i + 1)) - 1 for i in range(n)]


class Case:
    """seqs: (context tokens, drafted tokens)"""

    def __init__(self, dtype, codes, dk, dv, heads, kv_heads, seqs, kind="tree", seed=0, spare=3, loud=1.0):
        from omniserve_amd.backend.lm import KvCodes, tree_masks
        self.dtype, self.codes, self.dk, self.dv, self.H, self.G = dtype, codes, dk, dv, heads, kv_heads
        gen = torch.Generator(device=dev()).manual_seed(seed)
        host = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device=dev(), generator=gen)      # noqa: E731
        self.gen, self.rnd = gen, rnd
        need = [-(-n // PAGE) for n, _ in seqs]
        total = sum(need) + spare
        if codes:
            (k, ke), (v, ve) = (quantised(rnd(total, kv_heads, PAGE, d) * torch.exp(rnd(total, kv_heads, PAGE, 1)) * loud, dev()) for d in (dk, dv))
            self.cache = KvCodes(k, v, ke, ve)
        else:
            self.cache = tuple((rnd(total, kv_heads, PAGE, d) * loud).to(dtype) for d in (dk, dv))
        order = torch.randperm(total, generator=host).int()
        self.bt = torch.zeros(len(seqs), max(need + [1]) + 2, dtype=torch.int32)
        first, pos, masks, at = [0], [], [], 0
        self.parents = []
        for b, ((n, t), p) in enumerate(zip(seqs, need)):
            self.bt[b, :p] = order[at:at + p]
            at += p
            self.parents.append(_tree(t, kind, host))
            m, depth = tree_masks(self.parents[-1])
            masks.append(m)
            pos += (depth + n).tolist()
            first.append(first[-1] + t)
        words = max([1] + [m.shape[1] for m in masks])
        n = first[-1]
        self.mask = torch.zeros(n, words, dtype=torch.int64)
        for f, m in zip(first, masks):
            self.mask[f:f + m.shape[0], :m.shape[1]] = m
        self.mask, self.bt = self.mask.to(dev()), self.bt.to(dev())
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev())      # noqa: E731
        self.first, self.pos, self.length = ints(first), ints(pos), ints([a for a, _ in seqs])
        self.max_draft, self.max_context = max([t for _, t in seqs]), max([a for a, _ in seqs])
        self.q = rnd(n, heads * dk).to(dtype)
        self.k, self.v = rnd(n, kv_heads * dk).to(dtype), rnd(n, kv_heads * dv).to(dtype)
        self.scale = dk ** -0.5

    def pools(self):
        if not self.codes:
            return [t.double() for t in self.cache]
        return [decoded(c, e) for c, e in zip(self.cache[:2], self.cache[2:])]

    def run(self, window=None, out=None, **kw):
        kw = {"max_draft": self.max_draft, "max_context": self.max_context, **kw}
        return _ops(self.dtype).tree_attn(self.q, self.k, self.v, self.mask, self.first, self.pos, self.cache, self.bt, self.length, self.scale, window=window, out=out, **kw)

    def check(self, got, window=None, max_draft=None):
        n = self.q.shape[0]
        ref = attention(self.q.double().view(n, self.H, self.dk), self.k.double().view(n, self.G, self.dk), self.v.double().view(n, self.G, self.dv), self.mask, self.first.cpu(),
                        self.pos, *self.pools(), self.bt, self.length, self.scale, window or NO_WINDOW, max_draft or self.max_draft, self.H // self.G)
        live = ~ref[4][:, 0, 0].isnan()
        got = got.double().view(n, self.H, self.dv)[live]
        ref = [t[live] for t in ref]
        wrong = ref[0].isnan()
        assert torch.equal(got.isnan() | got.isinf(), wrong | ref[0].isinf())
        bound = attention_bound(self.dtype, self.codes, self.dk, *ref)
        over = ((got - ref[0]).abs() / bound)[ref[0].isfinite()]
        assert over.numel() == 0 or float(over.max()) <= 1.0, float(over.max())


SEQS = {"short": [(0, 1), (1, 3), (63, 2), (64, 1), (65, 4)], "none": [(130, 0), (100, 5), (0, 0), (7, 0)], "many": [(200, 17), (31, 33), (129, 26), (0, 64)],
        "long": [(2500, 7), (1111, 1)], "wide": [(300, 100), (5, 130)]}


@pytest.mark.parametrize("seqs", list(SEQS))
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 256), (256, 64), (256, 256), (128, 64), (64, 128), (256, 128), (128, 256)])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention(dtype, codes, dk, dv, seqs):
    c = Case(dtype, codes, dk, dv, 4, 2, SEQS[seqs], seed=dk + dv)
    c.check(c.run())


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (7, 1), (16, 2), (20, 1), (8, 8), (33, 3)])
@pytest.mark.parametrize("codes", [True, False])
def test_head_groups(codes, heads, kv_heads):
    """Rows that end inside a block, at its end, and fill several"""
    for draft in (1, 5, 16):
        c = Case(torch.bfloat16, codes, 128, 128, heads, kv_heads, [(150, draft), (70, 1)], seed=heads + draft)
        c.check(c.run())


@pytest.mark.parametrize("kind", ["tree", "chain"])
@pytest.mark.parametrize("window", [1, 2, 40, 64, 65, 130, 1000])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows(dtype, codes, window, kind):
    """Context keys that only some of the drafted tokens still see, drafted tokens that their descendants do not"""
    c = Case(dtype, codes, 64, 64, 4, 2, [(300, 20), (64, 50), (0, 9), (129, 1)], kind=kind, seed=window)
    c.check(c.run(window=window), window=window)


@pytest.mark.parametrize("codes", [True, False])
def test_rows_that_see_nothing(codes):
    c = Case(torch.bfloat16, codes, 128, 128, 4, 2, [(0, 6), (50, 4)], seed=1)
    c.mask[2] = 0          # no context, no drafted token
    c.mask[8] = 0          # the context alone
    got = c.run()
    assert bool((got[2] == 0).all())
    c.check(got)


@pytest.mark.parametrize("codes", [True, False])
def test_rows_of_no_sequence_stay(codes):
    """In front of the first sequence, behind the last, and past max_draft; for one part and for several"""
    for seqs in ([(40, 3), (70, 5)], [(3000, 3), (2000, 5)]):
        c = Case(torch.bfloat16, codes, 128, 128, 4, 2, seqs, seed=2)
        c.first[0] = 1
        n = c.q.shape[0]
        c.first[2] = n - 1
        out = torch.full((n, 4 * 128), math.nan, dtype=torch.bfloat16, device=dev())      # (no output is NaN; any number may be one)
        # (the sequences' masks number their tokens from the new first one on)
        got = c.run(out=out, max_draft=3)
        assert got is out
        assert bool(out[0].isnan().all()) and bool(out[n - 1].isnan().all()) and bool(out[6:n - 1].isnan().all())
        assert not bool(out[1:6].isnan().any())
        c.check(got, max_draft=3)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_comes_out_of_masked_places(dtype, codes, bad):
    """NaN and infinities behind the end of a page's sequence, before every window, in drafted tokens that a row does not see"""
    c = Case(dtype, codes, 128, 64, 4, 2, [(100, 12), (300, 9), (0, 40)], seed=4)
    window = 120
    for b, n in enumerate(c.length.tolist()):
        for key in list(range(n, -(-n // PAGE) * PAGE)) + list(range(max(0, n - window - 30))):
            page = int(c.bt[b, key // PAGE])
            for i in (0, 1):
                c.cache[i][page, :, key % PAGE] = 0x7f if codes else bad
                if codes:
                    c.cache[2 + i][page, :, key % PAGE] = 255
    for b, tok in ((0, 5), (1, 8), (2, 3), (2, 35)):      # seen by itself and what descends from it
        row = int(c.first[b]) + tok
        c.k[row, ::3] = bad
        c.v[row, 7] = bad
    # the rows that do see a bad key or value
    sick = torch.zeros(c.q.shape[0], dtype=torch.bool, device=dev())
    for i in range(c.q.shape[0]):
        b = int((c.first.cpu() <= i).sum()) - 1
        for j in range(int(c.first[b]), int(c.first[b + 1])):
            if int(c.mask[i, 0]) >> (j - int(c.first[b])) & 1 and not bool(c.k[j].isfinite().all()):
                sick[i] = True
    got = c.run(window=window)
    assert bool(got[~sick].isfinite().all())
    # every other row: as if the bad places held zeros
    c.k, c.v = c.k.nan_to_num(0, 0, 0), c.v.nan_to_num(0, 0, 0)
    pools = [t.nan_to_num(0, 0, 0) for t in c.pools()]
    n = c.q.shape[0]
    ref = attention(c.q.double().view(n, c.H, c.dk), c.k.double().view(n, c.G, c.dk), c.v.double().view(n, c.G, c.dv), c.mask, c.first.cpu(), c.pos, *pools, c.bt, c.length, c.scale,
                    window, c.max_draft, c.H // c.G)
    far = ((got.double().view(n, c.H, c.dv) - ref[0]).abs() / attention_bound(dtype, codes, c.dk, *ref))[~sick]
    assert float(far.max()) <= 1.0


@pytest.mark.parametrize("codes", [True, False])
def test_values_that_a_row_sees_pass(codes):
    """An infinite value of a key that some rows see: those rows' column is infinite, nothing else"""
    c = Case(torch.bfloat16, codes, 64, 64, 2, 1, [(70, 6)], kind="chain", seed=5)
    c.v[3, 11] = math.inf
    got = c.run()
    c.check(got)
    assert bool(got[3:, 11].isinf().all()) and int((~got.isfinite()).sum()) == 6


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("draft", [1, 6, 20, 40])
@pytest.mark.parametrize("codes", [True, False])
def test_bad_queries_stay_in_their_rows(codes, draft, bad):
    """A query with a non-finite element: its head of its token alone is NaN"""
    c = Case(torch.bfloat16, codes, 128, 64, 4, 2, [(200, draft), (70, draft)], seed=15)
    want = c.run()
    row, head = draft + draft // 2, 3
    c.q[row, head * 128 + 77] = bad
    got = c.run()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[row, head * 64:(head + 1) * 64] = False
    assert bool(got[~keep].isnan().all()) and torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("codes", [True, False])
def test_pages_that_are_not_there(codes):
    """Page numbers outside the pools are not seen; lengths beyond the block table end with it"""
    c = Case(torch.bfloat16, codes, 128, 128, 4, 2, [(300, 4), (200, 3)], seed=6)
    c.bt[0, 1], c.bt[1, 3], c.bt[0, 4] = -1, 1 << 30, c.cache[0].shape[0]
    c.length[1] = 10000
    c.bt[1, 4:] = -5
    c.check(c.run())


@pytest.mark.parametrize("loud", [1e-12, 1e-4, 1e6])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_magnitudes(dtype, loud):
    """Cached values much smaller or larger than the drafted ones, and keys whose scores have any size"""
    c = Case(dtype, True, 128, 128, 4, 1, [(500, 5), (30, 30)], seed=7, loud=loud)
    c.q = (c.q.float() / max(loud, 1.0)).to(dtype)
    c.check(c.run())


def test_far_pages():
    """Offsets that pass 32 bits"""
    from omniserve_amd.backend.lm import KvCodes
    c = Case(torch.bfloat16, True, 128, 128, 4, 4, [(200, 3)], seed=8)
    pages = 70000
    far = [torch.zeros((pages,) + t.shape[1:], dtype=torch.uint8, device=dev()) for t in c.cache]
    at = pages - c.cache[0].shape[0]
    for t, f in zip(c.cache, far):
        f[at:] = t
    want = c.run()
    c.cache, c.bt = KvCodes(*far), c.bt + at
    assert torch.equal(c.run(), want)


@pytest.mark.parametrize("codes", [True, False])
def test_strides_and_streams(codes):
    """Rows of a wider projection, a block table that is part of a wider one, a stream of its own; the same bits"""
    c = Case(torch.bfloat16, codes, 128, 64, 8, 2, [(900, 11), (65, 4)], seed=9)
    want = c.run()
    wide = torch.randn(c.q.shape[0], 8 * 128 + 2 * 128 + 2 * 64 + 8, device=dev()).to(torch.bfloat16)
    wide[:, :1024], wide[:, 1024:1280], wide[:, 1280:1408] = c.q, c.k, c.v
    c.q, c.k, c.v = wide[:, :1024], wide[:, 1024:1280], wide[:, 1280:1408]
    c.bt = torch.cat((c.bt, torch.full_like(c.bt, -1)), 1)[:, :c.bt.shape[1]]
    out = torch.zeros(c.q.shape[0], 8 * 64 + 4, dtype=torch.bfloat16, device=dev())[:, 4:]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run(out=out)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("context", [70, 5000])
def test_captured(context):
    """Replayed with new lengths and inputs, two graphs in turn, eager calls between"""
    a = Case(torch.bfloat16, True, 128, 128, 8, 2, [(context, 9), (context // 2, 4)], seed=10)
    b = Case(torch.bfloat16, True, 128, 128, 8, 2, [(context // 3, 5), (context, 14)], seed=11)
    graphs = []
    for c in (a, b):
        c.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c.run()
        graphs.append((c, g, out))
    for k in range(4):
        for c, g, out in graphs:
            c.q.copy_(c.rnd(*c.q.shape))
            c.length.sub_(3)
            g.replay()
        for c, g, out in graphs:
            want = c.run()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            c.check(out)


def test_repeats_itself():
    c = Case(torch.bfloat16, True, 128, 128, 8, 2, [(3000, 13), (1700, 20)], seed=12)
    want = c.run()
    for _ in range(5):
        assert torch.equal(c.run(), want)


# ---------------------------------------------------------------------------------------------------------------
# together, as a step uses them
# ---------------------------------------------------------------------------------------------------------------
def test_prompt_then_drafts_then_the_kept_ones():
    """A prompt is turned and stored in one launch and read back for its own attention; a tree of drafted tokens is turned, attends to cache and tree, one
    path of it is stored by row number; the next token's attention sees it"""
    from omniserve_amd.backend.lm import code_pools, tree_masks
    from omniserve_amd.rope import inverse_frequencies
    dtype, H, G, d = torch.bfloat16, 8, 2, 128
    ops = _ops(dtype)
    gen = torch.Generator(device=dev()).manual_seed(13)
    rows = lambda n: torch.randn(n, (H + 2 * G) * d, device=dev(), generator=gen).to(dtype)      # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev())      # noqa: E731
    freq = torch.tensor(inverse_frequencies(d, 500000.0, {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192}), dtype=torch.float64, device=dev())
    n, pages = 150, [4, 0, 3, 1]
    cache = code_pools(6, G, d, d, dev())
    table = ints([pages])
    slots = lambda at: ints([pages[i // PAGE] * PAGE + i % PAGE for i in at])      # noqa: E731
    # the prompt
    x = rows(n)
    q = torch.empty(n, H * d, dtype=dtype, device=dev())
    ops.kv_store(x, cache, slots(range(n)), H, freq=freq, pos=ints(list(range(n))), pairing="halves", q_out=q)
    k, v = ops.kv_load(cache, slots(range(3 * PAGE)))
    o = torch.empty(n, H * d, dtype=dtype, device=dev())
    ops.attn_prefill(q, k, v, ints([[0, 1, 2]]), ints([[0, n, 0, 0]]), ints([[0, 0], [0, 128]]), None, o, d ** -0.5, NO_WINDOW, H, G, d, d)
    pools = [decoded(c, e) for c, e in zip(cache[:2], cache[2:])]
    # ... which is the attention of a chain of n drafted tokens whose keys and values are the cache's
    mask, depth = tree_masks(list(range(-1, n - 1)))
    ref = attention(q.double().view(n, H, d), k[:n].double().view(n, G, d), v[:n].double().view(n, G, d), mask.to(dev()), ints([0, n]).cpu(), ints(list(range(n))), *pools, table, ints([0]),
                    d ** -0.5, NO_WINDOW, n, H // G)
    assert ((o.double().view(n, H, d) - ref[0]).abs() <= attention_bound(dtype, False, d, *ref)).all()
    got = ops.tree_attn(q, k[:n], v[:n], mask.to(dev()), ints([0, n]), ints(list(range(n))), cache, table, ints([0]), d ** -0.5, max_draft=n, max_context=0)
    assert ((got.double().view(n, H, d) - ref[0]).abs() <= attention_bound(dtype, True, d, *ref)).all()
    # the drafts
    parents = [-1, 0, 0, 1, 1, 2, 4, 6]
    mask, depth = tree_masks(parents)
    pos = (depth + n).to(dev())
    y = rows(8)
    ops.rope(y, freq, pos, H + G, d, pairing="halves", out=y)
    args = (mask.to(dev()), ints([0, 8]), pos, cache, table, ints([n]), d ** -0.5)
    yq, yk, yv = y[:, :H * d], y[:, H * d:(H + G) * d], y[:, (H + G) * d:]
    got = ops.tree_attn(yq, yk, yv, *args, max_draft=8, max_context=n)
    ref = attention(yq.double().view(8, H, d), yk.double().view(8, G, d), yv.double().view(8, G, d), args[0], args[1].cpu(), pos, *pools, table, ints([n]), d ** -0.5, NO_WINDOW, 8, H // G)
    assert ((got.double().view(8, H, d) - ref[0]).abs() <= attention_bound(dtype, True, d, *ref)).all()
    # 0 - 1 - 4 - 6 are kept
    ops.kv_store(y, cache, slots(range(n, n + 4)), H, rows=ints([0, 1, 4, 6]))
    n += 4
    pools = [decoded(c, e) for c, e in zip(cache[:2], cache[2:])]
    k, v = ops.kv_load(cache, slots(range(n)))
    want = pools[0][table[0].long()].transpose(1, 2).reshape(-1, G * d)[:n]
    assert torch.equal(k.double(), want)
    near = yk[[0, 1, 4, 6]].double().view(4, G, d)
    assert ((want[-4:].view(4, G, d) - near).abs() <= 2.0 ** -4 * near.abs() + 2.0 ** -9 * near.abs().amax(-1, keepdim=True) / 224).all()
    # the next token
    z = rows(1)
    at = ints([n])
    ops.rope(z, freq, at, H + G, d, pairing="halves", out=z)
    zq, zk, zv = z[:, :H * d], z[:, H * d:(H + G) * d], z[:, (H + G) * d:]
    one = torch.ones(1, 1, dtype=torch.int64, device=dev())
    got = ops.tree_attn(zq, zk, zv, one, ints([0, 1]), at, cache, table, at, d ** -0.5, max_draft=1, max_context=n)
    ref = attention(zq.double().view(1, H, d), zk.double().view(1, G, d), zv.double().view(1, G, d), one, ints([0, 1]).cpu(), at, *pools, table, at, d ** -0.5, NO_WINDOW, 1, H // G)
    assert ((got.double().view(1, H, d) - ref[0]).abs() <= attention_bound(dtype, True, d, *ref)).all()


def test_a_chain_is_its_tokens_in_turn():
    """Over a cache of elements: the drafted chain's outputs are those of single tokens appended one after the other (lm_attn_decode, unturned)"""
    dtype, H, G, d, T, n = torch.bfloat16, 8, 2, 128, 5, 200
    c = Case(dtype, False, d, d, H, G, [(n, T)], kind="chain", seed=14)
    got = c.run()
    ops = _ops(dtype)
    kc, vc = (t.clone() for t in c.cache)
    none = torch.zeros(0, dtype=torch.float32, device=dev())
    n_, ref = c.q.shape[0], None
    full = attention(c.q.double().view(n_, H, d), c.k.double().view(n_, G, d), c.v.double().view(n_, G, d), c.mask, c.first.cpu(), c.pos, *c.pools(), c.bt, c.length, c.scale, NO_WINDOW,
                     T, H // G)
    bound = attention_bound(dtype, False, d, *full)
    c.bt[0, -(-n // PAGE)] = c.cache[0].shape[0] - 1 if int((c.bt[0] == c.cache[0].shape[0] - 1).sum()) == 0 else c.cache[0].shape[0] - 2
    for i in range(T):
        row = torch.cat((c.q[i:i + 1], c.k[i:i + 1], c.v[i:i + 1]), 1)
        at = n + i
        slot = torch.tensor([int(c.bt[0, at // PAGE]) * PAGE + at % PAGE], dtype=torch.int32, device=dev())
        ref = torch.empty(1, H * d, dtype=dtype, device=dev())
        ops.attn_decode(row, None, 0.0, none, torch.tensor([at], dtype=torch.int32, device=dev()), slot, kc, vc, c.bt, None, ref, None, 1, c.scale, NO_WINDOW, H, G, d, d)
        assert ((ref[0].double() - got[i].double()).abs().view(H, d) <= 2 * bound[i]).all()


@pytest.mark.parametrize("first", ["zeros", "loud"])
@pytest.mark.parametrize("loud", [2.0 ** 20, 2.0 ** 40, 2.0 ** 80])
@pytest.mark.parametrize("draft", [1, 26, 64])
def test_zeros_beside_loud_values(draft, loud, first):
    """Rows of zeros have the lowest exponent; they take their part of the sum whatever the others' is, in a tile of their own or not, in one piece or several"""
    for context in (300, 3000):
        c = Case(torch.bfloat16, True, 128, 128, 4, 2, [(context, draft), (context, draft)], seed=draft)
        c.cache[3].add_(int(math.log2(loud)))
        zeros = torch.zeros(context, dtype=torch.bool, device=dev())
        zeros[:context // 2] = True
        zeros = zeros if first == "zeros" else ~zeros
        zeros[::3] = True
        for b in range(2):
            for page in range(-(-context // PAGE)):
                at = zeros[page * PAGE:(page + 1) * PAGE].nonzero()[:, 0]
                for t, x in zip((c.cache[1], c.cache[3]), (0, 27)):
                    t[int(c.bt[b, page]), :, at] = x
        c.check(c.run())


@pytest.mark.parametrize("draft", [1, 26, 64])
def test_nothing_but_zeros(draft):
    """Many keys of the lowest exponent, whose scores rise: the sum stays finite"""
    c = Case(torch.bfloat16, True, 128, 128, 4, 2, [(40000, draft)], seed=draft)
    c.cache[1].zero_()
    c.cache[3].fill_(27)
    c.check(c.run())
    c.v *= 2.0 ** 60
    c.check(c.run())


def test_more_sequences_than_a_wave_has_lanes():
    """Segments are dealt out by one wave: 64 sequences, one more and many, some without tokens"""
    for n in (64, 65, 150):
        for draft in (1, 12, 40):
            c = Case(torch.bfloat16, True, 64, 64, 4, 2, [((i * 37) % 700, draft if i % 5 else 0) for i in range(n)], seed=n)
            c.check(c.run())
            c.check(c.run(max_context=5000))


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -12, 1.0])
@pytest.mark.parametrize("draft", [1, 64])
@pytest.mark.parametrize("codes", [True, False])
def test_scales(codes, draft, scale):
    c = Case(torch.bfloat16, codes, 128, 128, 4, 2, [(500, draft), (70, draft)], seed=draft)
    c.scale = scale
    c.check(c.run())
