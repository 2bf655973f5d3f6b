"""The quantised key-value cache, rotary positions and attention of drafted tokens, in 64 bits."""
import math

import torch

PAGE = 64
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # half a step, relative
CODE_STEP = 2.0 ** -4                                               # half a step of the codes, relative


def code_values(device):
    """the 256 codes' values, from the format: 4 exponent bits (bias 7), 3 of fraction, no infinities"""
    out = []
    for c in range(256):
        e, f = c >> 3 & 15, c & 7
        v = math.ldexp(8 + f, e - 10) if e else math.ldexp(f, -9)
        out.append((math.nan if c & 127 == 127 else v) * (-1 if c & 128 else 1))
    return torch.tensor(out, dtype=torch.float64, device=device)


def decoded(codes, exps):
    return code_values(codes.device)[codes.long()] * torch.exp2(exps.double() - 127)[..., None]


def row_exponent(x):
    """least e with max |x| <= 448 * 2^e over the finite values of the rows, from -100 on (f64 in)"""
    top = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(-1)
    m, q = torch.frexp(top)
    e = q - 9 + (m > 0.875).int()
    return torch.where(top == 0, torch.full_like(e, -100), e.clamp(-100, 120))


def turned(x, freq, pos, half, pairing, factor):
    """x [T, heads, dk] f64"""
    x = x.clone()
    angle = pos.double()[:, None] * freq[None]
    c, s = (angle.cos() * factor)[:, None], (angle.sin() * factor)[:, None]
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if pairing == "halves" else (2 * i, 2 * i + 1)
    y, z = x[..., a], x[..., b]
    x[..., a], x[..., b] = y * c - z * s, z * c + y * s
    return x


def quantised(x, device):
    """x [.., size] f32 -> (codes, exponent bytes) of valid cache rows, nearest code by search"""
    e = row_exponent(x.double())
    y = x.double() / torch.exp2(e.double())[..., None]
    grid = code_values(device)[:127]
    at = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, 126)
    near = torch.where(y.abs() - grid[at - 1] < grid[at] - y.abs(), at - 1, at)
    return (near | (y < 0).long() << 7).to(torch.uint8), (e + 127).to(torch.uint8)


def attention(q, k, v, mask, first, pos, kpool, vpool, bt, length, scale, window, max_draft, groups):
    """-> (output, sum p |v|, largest scale * sum |q| |k|, largest p * row's max |v|, seen keys, largest scale * max |q| * sum |k|), all of [tokens, heads, ..]; pools [pages, G, 64, size] f64;
    rows of no sequence are NaN"""
    n, H, dk = q.shape
    G, dv = kpool.shape[1], vpool.shape[3]
    out = torch.full((n, H, dv), math.nan, dtype=torch.float64, device=q.device)
    size = out.clone()
    sums, peak, count, coarse = (out[..., :1].clone() for _ in range(4))
    for b, ln in enumerate(length.tolist()):
        f0 = int(first[b])
        T = min(int(first[b + 1]) - f0, max_draft)
        if T <= 0:
            continue
        ln = min(ln, bt.shape[1] * PAGE)
        np_ = -(-ln // PAGE)
        pages = bt[b, :np_].long()
        real = ((pages >= 0) & (pages < kpool.shape[0])).repeat_interleave(PAGE)[:ln]
        at = pages.clamp(0, max(kpool.shape[0] - 1, 0))
        kk = torch.cat((kpool[at].transpose(0, 1).reshape(G, -1, dk)[:, :ln], k[f0:f0 + T].transpose(0, 1)), 1)
        vv = torch.cat((vpool[at].transpose(0, 1).reshape(G, -1, dv)[:, :ln], v[f0:f0 + T].transpose(0, 1)), 1)
        p = pos[f0:f0 + T].long()
        j = torch.arange(T, device=q.device)
        bits = (mask[f0:f0 + T][:, j // 64] >> (j % 64)) & 1
        where = torch.cat((torch.arange(ln, device=q.device), p))
        seen = torch.cat((real[None].expand(T, ln), bits.bool()), 1) & (where[None] > p[:, None] - window)
        for h in range(H):
            g = h // groups
            row = q[f0:f0 + T, h]
            x = (row[:, None] * torch.where(seen[..., None], kk[g][None], 0.0)).sum(-1) * scale
            x = torch.where(seen, x, -math.inf)
            w = torch.exp(x - x.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            w = torch.where(seen, w, 0.0)
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
            val = torch.where(seen[..., None], vv[g][None], 0.0)
            out[f0:f0 + T, h] = (w[..., None] * val).sum(1)
            size[f0:f0 + T, h] = (w[..., None] * val.abs()).sum(1)
            mag = kk[g].abs().nan_to_num(nan=0.0, posinf=0.0)
            sums[f0:f0 + T, h, 0] = torch.where(seen, row.abs() @ mag.T, 0.0).amax(-1) * scale
            coarse[f0:f0 + T, h, 0] = torch.where(seen, row.abs().amax(-1, keepdim=True) * mag.sum(-1), 0.0).amax(-1) * scale
            peak[f0:f0 + T, h, 0] = (w * val.abs().amax(-1)).amax(-1)
            count[f0:f0 + T, h, 0] = seen.sum(-1).double()
    return out, size, sums, peak, count, coarse


def attention_bound(dtype, codes, dk, ref, size, sums, peak, count, coarse):
    """How far lm_tree_attn may be from 64 bits: the result's rounding; then relative to sum p |v|: scores are sums of dk products in f32 (twice that
    for the order, and the conversion to a power of two), whose error enters every p and the total; a weight is 11 bits where values are codes (half a step
    2^-12, twice for the total's that is not rounded) and 16 of two bf16, or f32; exponentials and f32 sums of all keys.  An f16
    weight is at least 2^7 for the largest (times its values' power of two, at most 2^-7 of the row's largest value), and off by 2^-25 where it is small: 2^-32 of that.  Many rows over codes: a query element is two codes,
    q = 2^e (hi + lo / 16), max |q| > 224 * 2^e; hi is off by at most half a step, 2^-4 of it or (below 2^-6) 2^-10, lo is 16 times that, at most 256, and off by 2^-10 where it is below
    2^-6 and not at all where its 4 bits hold the rest (bf16 has 8): the element by 2^-14 * 2^e < 2^-21 max |q|; that times |k|, in every p and the total."""
    weight = (2.0 ** -12 if codes else 2.0 ** -16) if dtype == torch.bfloat16 else 2.0 ** -23
    rel = 2 * (dk + 4) * 2.0 ** -24 * (sums + 1.0) + weight + (count + 8) * 2.0 ** -24 + 2.0 ** -21
    rel = rel + (2 * 2.0 ** -21 * coarse if codes and dtype == torch.bfloat16 else 0.0)
    lost = count * 2.0 ** -32 * peak * 448 / 224 if codes and dtype == torch.bfloat16 else 0.0
    return 1.01 * UNIT[dtype] * ref.abs() + rel * size + lost + 1e-30
