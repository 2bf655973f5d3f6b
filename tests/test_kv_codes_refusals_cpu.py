"""Calls of the operators around the quantised cache that their kernels do not take are ValueErrors before anything is enqueued: addresses, rows that overlap, too
many heads."""
import pytest
import torch

from omniserve_amd.backend import lm

BF16, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


@pytest.fixture(params=[BF16, F32])
def ops(request):
    return lm.lm_ops(request.param)


def refuse(match, call, *args, **kw):
    with pytest.raises(ValueError, match=match):
        call(*args, **kw)


def off(shape, by, dtype=torch.uint8):
    """zeros that begin `by` elements behind an aligned address"""
    n = torch.Size(shape).numel()
    return torch.zeros(n + by, dtype=dtype)[by:].view(shape)


def overlapping(rows, width, step, dtype):
    return torch.zeros((rows - 1) * step + width, dtype=dtype).as_strided((rows, width), (step, 1))


def test_pools_off_their_alignment(ops):
    cache = lm.code_pools(2, 1, 64, 64, "cpu")
    x, slot = torch.zeros(3, 128, dtype=ops.dtype), torch.zeros(3, dtype=I32)
    for i in (0, 1):
        for by, store, load in ((1, "8 bytes", "16 bytes"), (4, "8 bytes", "16 bytes"), (8, "GPU", "16 bytes"), (16, "GPU", "GPU")):
            odd = (*cache[:i], off(cache[i].shape, by), *cache[i + 1:])
            refuse(store, ops.kv_store, x, odd, slot, 0)
            refuse(load, ops.kv_load, odd, slot)


def test_results_that_overlap(ops):
    t = ops.dtype
    x, freq, pos = torch.zeros(3, 256, dtype=t), torch.ones(32, dtype=torch.float64), torch.zeros(3, dtype=I32)
    refuse("overlap", ops.rope, x, freq, pos, 4, 64, out=torch.zeros(1, 256, dtype=t).expand(3, 256))
    refuse("overlap", ops.rope, x, freq, pos, 4, 64, out=overlapping(3, 256, 255, t))
    refuse("GPU", ops.rope, x, freq, pos, 4, 64, out=overlapping(3, 256, 256, t))
    refuse("GPU", ops.rope, x[:1], freq, pos[:1], 4, 64, out=torch.zeros(1, 256, dtype=t).expand(1, 256))
    refuse("GPU", ops.rope, torch.zeros(1, 256, dtype=t).expand(3, 256), freq, pos, 4, 64)      # (inputs may)
    cache = lm.code_pools(2, 1, 64, 64, "cpu")
    y = torch.zeros(3, 4 * 64 + 128, dtype=t)
    refuse("overlap", ops.kv_store, y, cache, pos, 4, freq=freq, pos=pos, q_out=torch.zeros(1, 256, dtype=t).expand(3, 256))
    refuse("overlap", ops.kv_load, cache, pos, out=(torch.zeros(3, 64, dtype=t), torch.zeros(1, 64, dtype=t).expand(3, 64)))


def test_too_many_heads(ops):
    t = ops.dtype
    x, freq, pos = torch.zeros(1, 4097 * 2, dtype=t), torch.ones(1, dtype=torch.float64), torch.zeros(1, dtype=I32)
    refuse("heads", ops.rope, x, freq, pos, 4097, 2)
    refuse("GPU", ops.rope, x, freq, pos, 4096, 2)
    cache = lm.code_pools(1, 1, 64, 64, "cpu")
    y = torch.zeros(1, 4096 * 64 + 128, dtype=t)
    refuse("heads", ops.kv_store, y, cache, pos, 4096)
    refuse("GPU", ops.kv_store, y, cache, pos, 4095)
    wide = lm.code_pools(1, 4097, 64, 64, "cpu")
    refuse("heads", ops.kv_load, wide, pos)


def test_attention_that_overlaps_or_is_too_large(ops):
    t, n = ops.dtype, 5
    cache = lm.code_pools(3, 2, 64, 128, "cpu")
    ok = dict(q=torch.zeros(n, 4 * 64, dtype=t), k=torch.zeros(n, 2 * 64, dtype=t), v=torch.zeros(n, 2 * 128, dtype=t), mask=torch.zeros(n, 1, dtype=I64),
              first=torch.zeros(3, dtype=I32), pos=torch.zeros(n, dtype=I32), cache=cache, bt=torch.zeros(2, 4, dtype=I32), length=torch.zeros(2, dtype=I32), scale=0.1, window=None,
              max_draft=3, max_context=100, out=None)
    bad = lambda match, **kw: refuse(match, ops.tree_attn, **{**ok, **kw})      # noqa: E731
    bad("overlap", bt=torch.zeros(1, 4, dtype=I32).expand(2, 4))
    bad("overlap", bt=overlapping(2, 4, 3, I32))
    bad("overlap", out=torch.zeros(1, 4 * 128, dtype=t).expand(n, 4 * 128))
    bad("GPU", out=overlapping(n, 4 * 128, 4 * 128, t))
    words = (1 << 24) // 4 // 64 + 1
    bad("max_draft", mask=torch.zeros(n, words, dtype=I64), max_draft=64 * words)
    bad("GPU", mask=torch.zeros(n, words, dtype=I64), max_draft=64 * (words - 1))
