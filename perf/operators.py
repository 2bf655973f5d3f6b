"""The operators around a quantised key-value cache, as cases: rotary positions, keys and values written as 8-bit floats and read back,
attention of drafted token trees over the cache.

`run` computes them in plain torch operations, or, where `own` is true, by the calls that a program makes of `backend.lm`.  Sizes are those of
the models and benchmarks of this repository (32 or 64 heads over 8 key-value heads of 128, prompts of 333 to 12001 tokens, contexts up to
100000) and of common drafting depths."""
import math
import random

import torch

own = False      # true: run() makes the framework's calls

PAGE = 64
LOW_EXP, HIGH_EXP = -100, 120      # of a cache row's scale
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    llama = dict(heads=32, kv_heads=8, dk=128, dv=128, type="bf16")
    return [
        # a decode step of one sequence far into a long context: nothing but latency
        dict(name="rope 1 token", op="rope", tokens=1, heads=40, dk=128, dims=128, pairing="halves", scaling="bands", factor=1.0, far=131072, type="bf16"),
        # a long prompt's queries and keys, neighbouring pairs of half the head, attention scaled up for the stretched context
        dict(name="rope 12001 tokens, half the head", op="rope", tokens=12001, heads=40, dk=128, dims=64, pairing="neighbours", scaling="stretched", factor=1.2079, far=131072,
             type="bf16"),
        # one decode step of 16 sequences: their new keys and values, read back as the next layer's check of them would
        dict(name="store 16 single tokens", op="store", tokens=16, dims=128, pairing="halves", scaling="bands", factor=1.0, far=8192, **llama),
        # a batch of seven prompts: turned, stored, and read back for the prompts' own attention
        dict(name="store 7 x 333", op="store", tokens=2331, dims=128, pairing="halves", scaling="none", factor=1.0, far=333, **llama),
        # a long prompt of a wide model
        dict(name="store 12001 tokens", op="store", tokens=12001, dims=128, pairing="halves", scaling="bands", factor=1.0, far=12001, heads=64, kv_heads=8, dk=128, dv=128, type="bf16"),
        # the context of one prompt portion that continues a conversation
        dict(name="load 1501 tokens", op="load", tokens=1501, kv_heads=8, dk=128, dv=128, type="bf16"),
        # a whole long context
        dict(name="load 100000 tokens", op="load", tokens=100000, kv_heads=8, dk=128, dv=128, type="bf16"),
        # one user without drafts
        dict(name="attend 1 token", op="tree", seqs=1, draft=1, shape="chain", low=1501, high=1501, codes=True, window=0, **llama),
        # a decode step of a full batch, no drafts
        dict(name="attend 61 single tokens", op="tree", seqs=61, draft=1, shape="chain", low=300, high=4000, codes=True, window=0, **llama),
        # trees of 26 drafted tokens for a medium batch
        dict(name="attend 16 trees of 26", op="tree", seqs=16, draft=26, shape="tree", low=500, high=4000, codes=True, window=0, **llama),
        # the same kind of step over a cache that is not quantised
        dict(name="attend 8 trees of 13, bf16 cache", op="tree", seqs=8, draft=13, shape="tree", low=1000, high=3000, codes=False, window=0, **llama),
        # wide trees over long documents
        dict(name="attend 4 trees of 64, 32768 tokens", op="tree", seqs=4, draft=64, shape="tree", low=32000, high=32768, codes=True, window=0, **llama),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rope", "store", "load", "tree", "tree"))
    kind = "f32" if rng.random() < 0.15 else "bf16"
    dk = rng.choice((64, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 7, 8))
    turned = dict(pairing=rng.choice(("halves", "neighbours")), scaling=rng.choice(("none", "bands", "stretched")), factor=rng.choice((1.0, 1.2079)), far=_log(rng, 64, 1000000))
    if op == "rope":
        dk = rng.choice((64, 80, 96, 128, 256))
        return dict(op=op, tokens=_log(rng, 1, 8000), heads=heads + kv_heads, dk=dk, dims=rng.choice((dk, dk // 2, 32)), type=kind, **turned)
    if op == "store":
        return dict(op=op, tokens=_log(rng, 1, 8000), heads=heads, kv_heads=kv_heads, dk=dk, dv=rng.choice((64, 128, dk)), dims=rng.choice((dk, dk // 2, 32)), type=kind, **turned)
    if op == "load":
        return dict(op=op, tokens=_log(rng, 1, 40000), kv_heads=kv_heads, dk=dk, dv=rng.choice((64, 128, dk)), type=kind)
    seqs, draft = _log(rng, 1, 40), _log(rng, 1, 64)
    high = _log(rng, 64, max(100, min(32768, 2000000 // (seqs * draft))))
    return dict(op=op, seqs=seqs, draft=draft, shape=rng.choice(("tree", "chain")), low=rng.randint(0, high), high=high, codes=rng.random() < 0.7,
                window=rng.choice((0, 0, 0, rng.randint(1, high + draft))), heads=heads, kv_heads=kv_heads, dk=dk, dv=rng.choice((64, 128, dk)), type=kind)


def _frequencies(c):
    """Rotation per position of the dims / 2 pairs, in 64 bits: as they are, in three bands of wavelengths (the long ones slowed down by 8), or
    stretched by 16 with a ramp over the pair's turns in the original context."""
    f = [10000.0 ** (-2.0 * i / c["dims"]) for i in range(c["dims"] // 2)]
    if c["scaling"] == "none":
        return f
    original, factor, slow, fast = (8192, 8.0, 1.0, 4.0) if c["scaling"] == "bands" else (4096, 16.0, 1.0, 32.0)
    turns = [original * x / (2 * math.pi) for x in f]
    if c["scaling"] == "bands":
        keep = [min(1.0, max(0.0, (t - slow) / (fast - slow))) for t in turns]
    else:
        pair = lambda t: c["dims"] * math.log(original / (t * 2 * math.pi)) / (2 * math.log(10000.0))      # noqa: E731
        a, b = math.floor(pair(fast)), math.ceil(pair(slow))
        keep = [1.0 - min(1.0, max(0.0, (i - a) / max(b - a, 1e-3))) for i in range(len(f))]
    return [x * k + x / factor * (1.0 - k) for x, k in zip(f, keep)]


def _sizes(c):
    """(context tokens, drafted tokens) of every sequence: fixed by the case, so that its work is"""
    r = random.Random("%d %d %d %d" % (c["seqs"], c["draft"], c["low"], c["high"]))
    return [(r.randint(c["low"], c["high"]), c["draft"] if i == 0 else r.randint(max(1, c["draft"] - 3), c["draft"])) for i in range(c["seqs"])]


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e of whole e in f32, exact"""
    return ((e + 127) << 23).view(torch.float32)


def _codes(x):
    """8-bit floats (4 exponent bits, 3 of fraction) of rows of f32 and the rows' exponents: 2^e is the least that brings the row below 448"""
    m, q = torch.frexp(x.abs().amax(-1))
    e = (q - 9 + (m > 0.875).int()).clamp(LOW_EXP, HIGH_EXP)
    e = torch.where(m == 0, torch.full_like(e, LOW_EXP), e)
    return (x * _pow2(-e)[..., None]).to(torch.float8_e4m3fn), e


def _values(codes, exps):
    return codes.view(torch.float8_e4m3fn).float() * _pow2(exps.int() - 127)[..., None]


def _pools(c, pages, rnd):
    """[pages][kv heads][64][size] of keys and values: keys with a few channels much larger than the others, values without"""
    loud = 1.0 + 7.0 * (torch.arange(c["dk"], device="cuda") % 37 == 5)
    k, v = rnd(pages, c["kv_heads"], PAGE, c["dk"]) * loud / math.sqrt(1.0 + 63.0 / 37), rnd(pages, c["kv_heads"], PAGE, c["dv"])
    if not c.get("codes", True):
        return k.to(DTYPES[c["type"]]), v.to(DTYPES[c["type"]])
    (kc, ke), (vc, ve) = _codes(k), _codes(v)
    return kc.view(torch.uint8), vc.view(torch.uint8), (ke + 127).to(torch.uint8), (ve + 127).to(torch.uint8)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, dtype = case, DTYPES[case["type"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)      # noqa: E731
    s = dict(case)
    if c["op"] in ("rope", "store"):
        s["freq"] = torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda")
        last = max(c["far"], 1)
        at = [host.randrange(last) for _ in range(c["tokens"])] if c["tokens"] <= 64 else [(host.randrange(last) + i) % last for i in range(c["tokens"])]
        s["pos"] = _ints(at)
    if c["op"] == "rope":
        s["x"] = rnd(c["tokens"], c["heads"] * c["dk"]).to(dtype)
    elif c["op"] == "store":
        n = c["tokens"]
        width = (c["heads"] + c["kv_heads"]) * c["dk"] + c["kv_heads"] * c["dv"]
        s["x"] = (rnd(n, width) * torch.exp(0.5 * rnd(n, 1))).to(dtype)
        pages = n // PAGE + 2
        s["cache"] = _pools(c, pages, rnd)
        number = torch.randperm(pages, device="cuda", generator=gen).int()
        at = torch.arange(n, device="cuda", dtype=torch.int32) + host.randrange(PAGE)
        s["slot"] = number[(at // PAGE).long()] * PAGE + at % PAGE
        s["q"] = torch.empty(n, c["heads"] * c["dk"], dtype=dtype, device="cuda")
    elif c["op"] == "load":
        pages = c["tokens"] // PAGE + 2
        s["cache"] = _pools(c, pages, rnd)
        number = torch.randperm(pages, device="cuda", generator=gen).int()
        at = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
        s["slot"] = number[(at // PAGE).long()] * PAGE + at % PAGE
    else:
        sizes = _sizes(c)
        need = [-(-n // PAGE) for n, _ in sizes]
        total = sum(need) + 1
        s["cache"] = _pools(c, total, rnd)
        order = list(range(total))
        host.shuffle(order)
        table, first, pos, masks, at = [], [0], [], [], 0
        for (n, t), p in zip(sizes, need):
            table.append(order[at:at + p] + [0] * (max(need + [1]) - p))
            at += p
            seen, depth = [], []
            for i in range(t):
                parent = i - 1 if c["shape"] == "chain" else host.randint(-1, i - 1) if i < 4 else host.randint(i // 3, i - 1)
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
                depth.append(depth[parent] + 1 if parent >= 0 else 0)
            pos += [n + d for d in depth]
            masks += [m - (1 << 64) if m >> 63 else m for m in seen]
            first.append(first[-1] + t)
        n = first[-1]
        s["q"] = rnd(n, c["heads"] * c["dk"]).to(dtype)
        s["k"], s["v"] = rnd(n, c["kv_heads"] * c["dk"]).to(dtype), rnd(n, c["kv_heads"] * c["dv"]).to(dtype)
        s["table"], s["first"], s["pos"], s["length"] = _ints(table), _ints(first), _ints(pos), _ints([x for x, _ in sizes])
        s["mask"] = torch.tensor(masks, dtype=torch.int64, device="cuda").view(n, 1)
        s["scale"], s["longest"] = c["dk"] ** -0.5, max(x for x, _ in sizes)
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _turned(x, s, heads):
    """rows [T][heads][dk] in f32, their first dims turned by position"""
    T, half = x.shape[0], s["dims"] // 2
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]
    x = x.float().view(T, heads, s["dk"])
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    if s["pairing"] == "halves":
        a, b = turn[..., :half], turn[..., half:]
        turn = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turn, rest), -1)


def _plain_rope(s):
    return _turned(s["x"], s, s["heads"]).to(s["x"].dtype).flatten(1)


def _plain_load(s):
    k, v, ke, ve = s["cache"]
    page, off = (s["slot"] // PAGE).long(), (s["slot"] % PAGE).long()
    out = [_values(c[page, :, off], e[page, :, off]).to(DTYPES[s["type"]]).flatten(1) for c, e in ((k, ke), (v, ve))]
    return tuple(out)


def _plain_store(s):
    H, G = s["heads"], s["kv_heads"]
    qk = _turned(s["x"][:, :(H + G) * s["dk"]], s, H + G)
    v = s["x"][:, (H + G) * s["dk"]:].float().view(-1, G, s["dv"])
    page, off = (s["slot"] // PAGE).long(), (s["slot"] % PAGE).long()
    s["q"].copy_(qk[:, :H].flatten(1))
    for x, c, e in ((qk[:, H:], s["cache"][0], s["cache"][2]), (v, s["cache"][1], s["cache"][3])):
        code, exp = _codes(x)
        c[page, :, off] = code.view(torch.uint8)
        e[page, :, off] = (exp + 127).to(torch.uint8)
    return (s["q"],) + _plain_load(s)


def _plain_tree(s):
    G, dk, dv = s["kv_heads"], s["dk"], s["dv"]
    group = s["heads"] // G
    first, length, B = s["first"].long(), s["length"], s["length"].numel()
    n, longest, T = s["q"].shape[0], s["longest"], s["draft"]
    table = s["table"].long()
    rows = []
    for i, d in ((0, dk), (1, dv)):
        x = s["cache"][i][table]
        x = _values(x, s["cache"][2 + i][table]) if s["codes"] else x.float()
        rows.append(x.transpose(1, 2).reshape(B, G, -1, d)[:, :, :longest])      # [B, G, keys, size]
    seq = torch.searchsorted(first, torch.arange(n, device="cuda"), right=True) - 1
    at = torch.arange(n, device="cuda") - first[seq]
    pad = lambda x: torch.zeros((B, T) + x.shape[1:], dtype=torch.float32, device="cuda").index_put((seq, at), x.float())      # noqa: E731
    for i, x in ((0, s["k"].view(n, G, dk)), (1, s["v"].view(n, G, dv))):
        rows[i] = torch.cat((rows[i], pad(x).transpose(1, 2)), 2)
    q = pad(s["q"].view(n, G, group, dk)).permute(0, 2, 1, 3, 4).reshape(B, G, T * group, dk)
    keys = torch.arange(longest, device="cuda")
    bits = torch.zeros((B, T), dtype=torch.int64, device="cuda").index_put((seq, at), s["mask"][:, 0])
    pos = torch.zeros((B, T), dtype=torch.int32, device="cuda").index_put((seq, at), s["pos"])
    low = pos - (s["window"] if s["window"] else 1 << 30)      # the newest position that is not seen any more
    context = (keys < length[:, None, None]) & (keys > low[..., None])
    drafted = (bits[..., None] >> torch.arange(T, device="cuda") & 1).bool() & (pos[:, None, :] > low[..., None])
    seen = torch.cat((context, drafted), -1).repeat_interleave(group, 1)[:, None]      # [B, 1, T * group, keys]
    x = torch.matmul(q, rows[0].transpose(2, 3)) * s["scale"]
    x = torch.where(seen, x, torch.full_like(x, float("-inf")))
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows[1]) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(B, G, T, group, dv).permute(0, 2, 1, 3, 4)[seq, at]
    return o.reshape(n, -1).to(s["q"].dtype)


def run(state):
    s = state
    if not own:
        return {"rope": _plain_rope, "store": _plain_store, "load": _plain_load, "tree": _plain_tree}[s["op"]](s)
    from omniserve_amd.backend.lm import lm_ops
    ops = lm_ops(DTYPES[s["type"]])
    if s["op"] == "rope":
        return ops.rope(s["x"], s["freq"], s["pos"], s["heads"], s["dk"], pairing=s["pairing"], factor=s["factor"])
    if s["op"] == "store":
        ops.kv_store(s["x"], s["cache"], s["slot"], s["heads"], freq=s["freq"], pos=s["pos"], pairing=s["pairing"], factor=s["factor"], q_out=s["q"])
        return (s["q"],) + tuple(ops.kv_load(s["cache"], s["slot"]))
    if s["op"] == "load":
        return tuple(ops.kv_load(s["cache"], s["slot"]))
    return ops.tree_attn(s["q"], s["k"], s["v"], s["mask"], s["first"], s["pos"], s["cache"], s["table"], s["length"], s["scale"],
                         window=s["window"] or None, max_draft=s["draft"], max_context=s["longest"])


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    c, size = case, DTYPES[case["type"]].itemsize
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dk"] * size + 4 * c["tokens"], "flops": 3 * n * c["dims"]}
    if c["op"] in ("store", "load"):
        n = c["tokens"]
        kv = n * c["kv_heads"] * (c["dk"] + c["dv"])
        codes = kv + 2 * n * c["kv_heads"]
        if c["op"] == "load":
            return {"bytes": codes + kv * size + 4 * n, "flops": kv}
        q = n * c["heads"] * c["dk"]
        # the queries read and written, keys and values read, their codes written; the codes read back and the values written
        return {"bytes": 2 * q * size + kv * size + codes + codes + kv * size + 8 * n, "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["dims"] + 3 * kv}
    each = (c["dk"] + c["dv"] + 2) if c["codes"] else (c["dk"] + c["dv"]) * size
    total = flops = 0
    for length, draft in _sizes(c):
        keys = min(length, c["window"] + draft) if c["window"] else length
        seen = min(length, c["window"]) if c["window"] else length
        total += keys * c["kv_heads"] * each + draft * (c["heads"] + c["kv_heads"]) * (c["dk"] + c["dv"]) * size + 16 * draft + 4 * (-(-keys // PAGE))
        flops += 2 * draft * (seen + 1) * c["heads"] * (c["dk"] + c["dv"])
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_turn(s, first_head, heads):
    x = s["x"].double()[:, first_head * s["dk"]:(first_head + heads) * s["dk"]].reshape(-1, heads, s["dk"]).clone()
    half = s["dims"] // 2
    angle = s["pos"].double().unsqueeze(1) * s["freq"].unsqueeze(0)
    # the pair (a, b) as a complex number, times factor * e^(i angle)
    a = slice(0, half) if s["pairing"] == "halves" else slice(0, 2 * half, 2)
    b = slice(half, 2 * half) if s["pairing"] == "halves" else slice(1, 2 * half, 2)
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(angle, s["factor"]), angle).unsqueeze(1)
    x[..., a], x[..., b] = z.real, z.imag
    return x


def _exact_rounded(x):
    """x as the cache gives it back: on the grid of 8-bit floats under the row's power of two"""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0))
    e = e + (top > 448.0 * torch.exp2(e)).double() - (top <= 448.0 * torch.exp2(e - 1)).double()      # (the logarithm's own rounding)
    e = e.clamp(LOW_EXP, HIGH_EXP)
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _exact_code(c):
    """the number that each 8-bit pattern stands for"""
    c = c.long()
    e, f = c >> 3 & 15, (c & 7).double()
    size = torch.where(e == 0, f * 2.0 ** -9, (8.0 + f) * torch.exp2((e - 10).double()))
    return torch.where(c > 127, -size, size)


def _exact_cache(s, i, page, off=None):
    x = s["cache"][i][page] if off is None else s["cache"][i][page, :, off]
    if not s.get("codes", True):
        return x.double()
    e = s["cache"][2 + i][page] if off is None else s["cache"][2 + i][page, :, off]
    return _exact_code(x) * torch.exp2(e.double() - 127)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rope":
        return _exact_turn(s, 0, s["heads"]).flatten(1)
    if s["op"] == "store":
        H, G = s["heads"], s["kv_heads"]
        v = s["x"].double()[:, (H + G) * s["dk"]:].reshape(-1, G, s["dv"])
        return (_exact_turn(s, 0, H).flatten(1), _exact_rounded(_exact_turn(s, H, G)).flatten(1), _exact_rounded(v).flatten(1))
    if s["op"] == "load":
        page, off = s["slot"].long() // PAGE, s["slot"].long() % PAGE
        return tuple(_exact_cache(s, i, page, off).flatten(1) for i in (0, 1))
    H, G, out = s["heads"], s["kv_heads"], []
    first, length = s["first"].tolist(), s["length"].tolist()
    for b, n in enumerate(length):
        lo, hi = first[b], first[b + 1]
        pages = s["table"][b, :-(-n // PAGE)].long()
        tokens = torch.arange(hi - lo, device="cuda")
        mine = s["pos"][lo:hi].long()
        oldest = mine - (s["window"] if s["window"] else 1 << 40) + 1
        spot = torch.cat((torch.arange(n, device="cuda"), mine))
        seen = torch.cat((torch.ones(hi - lo, n, dtype=torch.bool, device="cuda"), (s["mask"][lo:hi] >> tokens) % 2 != 0), 1) & (spot >= oldest[:, None])
        for h in range(H):
            g = h * G // H
            part = []
            for i, x, d in ((0, s["k"], s["dk"]), (1, s["v"], s["dv"])):
                old = _exact_cache({**s, "cache": [t[:, g:g + 1] for t in s["cache"]]}, i, pages).reshape(-1, d)[:n]
                part.append(torch.cat((old, x[lo:hi, g * d:(g + 1) * d].double())))
            z = (part[0] @ s["q"][lo:hi, h * s["dk"]:(h + 1) * s["dk"]].double().T).T * s["scale"]
            w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            out.append(torch.nan_to_num(w) @ part[1])
    at, rows = 0, []
    for b in range(len(length)):
        rows.append(torch.cat(out[at:at + H], 1))
        at += H
    return torch.cat(rows)
