"""Chunks written to the pages of their sequences, caches read back, and the step that chains them."""

from __future__ import annotations

import math

import pytest
import torch

from aws_training_study_amd.pcp_attention import (
    CacheReader,
    ChunkAttentionKernel,
    ChunkCacheWriter,
    ChunkStep,
    KVCacheWriter,
    PageAllocator,
    QueryKeyRotation,
    RotaryEmbedding,
    build_page_pool,
    empty_token_scales,
)
from chunk_model import BF16, FP8, Cache, attention, config, quantised, rows, starts_of

pytestmark = pytest.mark.gpu


def bits(x):
    return x.view(torch.uint8) if x.element_size() == 1 else x.view(torch.int16)


def fresh_tokens(cache, lengths, fresh):
    """K and V rows of the new tokens of ``cache``'s sequences, in order."""
    return tuple(torch.cat([cache.tokens[b][which][n - f:n] for b, (n, f) in enumerate(zip(lengths, fresh))])
                 for which in range(2))


WRITES = {
    "one_each": (dict(d=256, hkv=2, hq=32, kv=FP8, block=512), [1, 600, 513, 64], [1] * 4),
    "ragged": (dict(d=128, hkv=4, hq=28, kv=FP8), [100, 5, 64, 333, 7], [30, 0, 64, 100, 1]),
    "ragged_bf16": (dict(d=128, hkv=4, hq=28), [100, 5, 64, 333, 7], [30, 0, 64, 100, 1]),
    "striped": (dict(pcp=4, il=16, block=128, d=64, hkv=2, hq=8, kv=FP8), [700, 77], [700, 13]),
    "uneven": (dict(pcp=3, il=48, block=192, d=64, hkv=8, hq=24, kv=FP8), [500, 145], [45, 145]),
    "striped_bf16": (dict(pcp=5, il=32, block=64, d=256, hkv=1, hq=4), [333, 9], [333, 9]),
    "many_rows": (dict(d=64, hkv=2, hq=8, kv=FP8, bucket=8192), [8000, 5000], [8000, 4900]),
    "many_sequences": (dict(d=64, hkv=3, hq=6, kv=FP8, bucket=256), [5 + 3 * i % 200 for i in range(150)],
                       [i % 5 for i in range(150)]),
}


@pytest.mark.parametrize("name,scales", [(name, s) for name, (options, *_) in WRITES.items()
                                         for s in (("plain", "token", "tensor") if "kv" in options else ("plain",))])
def test_pages_of_a_chunk(name, scales, cuda_device):
    """The written slots hold the model's bits, every other byte of the pool and the scales stays."""
    options, lengths, fresh = WRITES[name]
    cfg = config(**options)
    cache = Cache(cfg, lengths, 1, scales="none" if scales == "plain" else scales,
                  table_dtype=torch.int64 if scales == "token" else torch.int32)
    before = cache.pool.clone()  # with the older tokens only
    kept = None if cache.token_scales is None else cache.token_scales.clone()
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        page, slot = (x[n - f:] for x in cache.index[b])
        bits(before)[page, :, :, slot] = 0x55
        if kept is not None:
            kept[page, :, :, slot] = -1.0
    first = 2
    k, v = (torch.cat((torch.full_like(x[:1], math.nan).repeat(first, 1, 1), x, x[:3])) for x in
            fresh_tokens(cache, lengths, fresh))
    _, table, kw = cache.call(cuda_device)
    pool = before.reshape(cache.num_pages, -1).to(cuda_device)
    if kept is not None:
        kw["token_scales"] = kept.to(cuda_device)
    ChunkCacheWriter(cfg)(k.to(cuda_device), v.to(cuda_device), pool, table,
                          torch.tensor(lengths, dtype=torch.int32, device=cuda_device),
                          chunk_starts=starts_of(fresh, first).to(cuda_device), **kw)
    torch.cuda.synchronize()
    assert torch.equal(bits(pool.cpu()), bits(cache.pages()))
    if kept is not None:
        assert torch.equal(kw["token_scales"].cpu().view(torch.int32), cache.token_scales.view(torch.int32))


def test_strided_rows_and_equal_chunks(cuda_device):
    """K and V as columns of one projection, the same number of rows for each sequence."""
    cfg = config(d=128, hkv=4, hq=28, kv=FP8)
    lengths, fresh = [40, 3, 300], [3] * 3
    cache = Cache(cfg, lengths, 2, scales="token")
    k, v = fresh_tokens(cache, lengths, fresh)
    qkv = torch.cat((torch.zeros(9, 28, 128, dtype=torch.bfloat16), k, v), dim=1).to(cuda_device)
    _, table, kw = cache.call(cuda_device)
    pool = cache.pages().clone()
    for b, n in enumerate(lengths):
        page, slot = (x[n - 3:] for x in cache.index[b])
        bits(pool).view(cache.num_pages, 2, 4, -1, 128)[page, :, :, slot] = 0
    pool = pool.to(cuda_device)
    ChunkCacheWriter(cfg)(qkv[:, 28:32], qkv[:, 32:], pool, table,
                          torch.tensor(lengths, dtype=torch.int32, device=cuda_device), **kw)
    torch.cuda.synchronize()
    assert torch.equal(bits(pool.cpu()), bits(cache.pages()))


def test_rows_without_a_place(cuda_device):
    """Positions below zero or past the cache and entries of no page: nothing is written for them."""
    cfg = config(d=64, hkv=2, hq=8, kv=FP8, bucket=128)
    table = torch.tensor([[[0, 1]], [[2, 99]], [[-3, 3]]], dtype=torch.int32, device=cuda_device)
    pool = torch.zeros((4, cfg.page_elements), device=cuda_device).to(torch.float8_e4m3fn)
    scales = empty_token_scales(cfg, cuda_device, num_pages=4)
    gen = torch.Generator().manual_seed(3)
    k, v = (rows(gen, 12, 2, 64).to(cuda_device) for _ in range(2))
    # sequence 0: positions -2 .. 1 and 126 .. 129 would be its rows; 1: 62 .. 65; 2: 62 .. 65
    lengths = torch.tensor([2, 66, 66], dtype=torch.int32, device=cuda_device)
    ChunkCacheWriter(cfg)(k, v, pool, table, lengths, token_scales=scales)
    torch.cuda.synchronize()
    got = pool.view(torch.uint8).view(4, 2, 2, 64, 64).cpu()
    want = torch.zeros_like(got)
    codes = [quantised(x.cpu())[0].view(torch.uint8) for x in (k, v)]
    for which in range(2):
        want[0, which, :, 0:2] = codes[which][2:4].transpose(0, 1)
        want[2, which, :, 62:64] = codes[which][4:6].transpose(0, 1)
        want[3, which, :, 0:2] = codes[which][10:12].transpose(0, 1)
    assert torch.equal(got, want)
    assert int((scales != 0).sum()) == 6 * 2 * 2
    before = pool.clone()
    ChunkCacheWriter(cfg)(k, v, pool, table, torch.full((3,), 3000, dtype=torch.int32, device=cuda_device),
                          token_scales=scales)
    torch.cuda.synchronize()
    assert torch.equal(bits(before), bits(pool))


def test_scales_of_unusual_rows(cuda_device):
    """Zeros, the smallest and largest values, infinities and NaN."""
    cfg = config(d=64, hkv=1, hq=1, kv=FP8, bucket=64)
    k = torch.zeros(8, 1, 64)
    k[1, 0, 3] = 1.0
    k[2, 0] = 2.0**-130
    k[3, 0] = torch.finfo(torch.bfloat16).max
    k[4, 0, :5] = torch.tensor([math.inf, -math.inf, math.nan, 3.0, -1.5])
    k[5, 0] = math.inf
    k[6, 0] = torch.linspace(-1, 1, 64)
    k[7, 0, 0], k[7, 0, 1] = 2.0**-60, -(2.0**-68)
    k = k.to(torch.bfloat16)
    pool = torch.zeros((1, cfg.page_elements), device=cuda_device).to(torch.float8_e4m3fn)
    scales = empty_token_scales(cfg, cuda_device, num_pages=1)
    table = torch.zeros((1, 1), dtype=torch.int32, device=cuda_device)
    ChunkCacheWriter(cfg)(k.to(cuda_device), k.to(cuda_device), pool, table,
                          torch.tensor([8], dtype=torch.int32, device=cuda_device), token_scales=scales)
    torch.cuda.synchronize()
    codes, want = quantised(k)
    got = pool.view(2, 64, 64)[:, :8].cpu()
    for which in range(2):
        assert torch.equal(scales[0, which, 0, :8].cpu(), want[:, 0])
        nan = torch.isnan(codes[:, 0].float())
        assert torch.equal(torch.isnan(got[which].float()), nan)
        assert torch.equal(bits(got[which])[~nan], bits(codes[:, 0])[~nan])


@pytest.mark.parametrize("options,length,scales", [
    *((dict(d=256, hkv=2, hq=32, kv=FP8, block=512, pcp=4), 1700, s) for s in ("plain", "token", "tensor")),
    *((dict(d=128, hkv=4, hq=28, kv=FP8, pcp=3, il=48, block=192), 445, s) for s in ("plain", "token", "tensor")),
    (dict(d=64, hkv=2, hq=8, kv=BF16, pcp=4, il=16, block=128), 700, "plain"),
    (dict(d=128, hkv=3, hq=6, kv=BF16), 1, "plain"),
])
def test_reading_back(options, length, scales, cuda_device):
    cfg = config(bucket=2048, **options)
    cache = Cache(cfg, [length], 4, scales="none" if scales == "plain" else scales, table_dtype=torch.int64)
    pool, table, kw = cache.call(cuda_device)
    reader = CacheReader(cfg)
    for first, count in ((0, length), (length // 3, length // 2), (length - 1, 1), (0, 0)):
        got = reader(pool, table if first else table[0], first_pos=first, num_tokens=count, **kw)
        torch.cuda.synchronize()
        for x, value in zip(got, cache.values[0]):
            # one product in 32 bits (exact in 64: 4 bits of code, 24 of scale), rounded to 16 bits
            want = value[first:first + count].float().to(torch.bfloat16).transpose(0, 1)
            assert torch.equal(x.cpu(), want)
    # past the tokens: zeros where there is no page or no cache
    cache.table[0, 0, 0] = cache.num_pages
    got = reader(pool, cache.table.to(cuda_device), first_pos=0, num_tokens=min(length, 16), **kw)[0]
    assert not bool(got.any())
    assert not bool(reader(pool, table, first_pos=2048 * 50, num_tokens=3, **kw)[1].any())


def test_a_cache_of_token_scales_becomes_one_of_tensor_scales(cuda_device):
    """Read back, then filled anew for the prefill's kernel."""
    cfg = config(d=256, hkv=2, hq=32, kv=FP8, block=512, pcp=4, bucket=2048)
    cache = Cache(cfg, [2048], 5, scales="token")
    pool, table, kw = cache.call(cuda_device)
    k, v = CacheReader(cfg)(pool, table, num_tokens=2048, **kw)
    again, k_scale, v_scale, _ = build_page_pool(cfg, k, v, table[0].clamp_max(cfg.num_pages - 1))
    want, want_k, want_v, _ = build_page_pool(
        cfg, *(x.float().to(torch.bfloat16).transpose(0, 1).contiguous().to(cuda_device) for x in cache.values[0]),
        table[0].clamp_max(cfg.num_pages - 1))
    torch.cuda.synchronize()
    assert (k_scale, v_scale) == (want_k, want_v)


def test_far_pages(cuda_device):
    """A chunk written to and read from pages whose bytes lie past 2^32."""
    cfg = config(d=256, hq=32, hkv=2, block=512, bucket=1024)
    pages = 4200
    pool = torch.empty((pages, cfg.page_elements), dtype=torch.bfloat16, device=cuda_device)
    table = torch.tensor([[[pages - 1, pages - 2]]], dtype=torch.int32, device=cuda_device)
    gen = torch.Generator().manual_seed(6)
    k, v = (rows(gen, 600, 2, 256).to(cuda_device) for _ in range(2))
    ChunkCacheWriter(cfg)(k, v, pool, table, torch.tensor([600], dtype=torch.int32, device=cuda_device))
    got = CacheReader(cfg)(pool, table, num_tokens=600)
    torch.cuda.synchronize()
    assert torch.equal(got[0], k.transpose(0, 1)) and torch.equal(got[1], v.transpose(0, 1))


# ---- a run of them together ---------------------------------------------------------


@pytest.mark.parametrize("kv,scales", [(FP8, "token"), (FP8, "plain"), (BF16, "plain")])
@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 28, 4), (256, 32, 2)])
def test_step_equals_its_parts(d, hq, hkv, kv, scales, cuda_device):
    """Rotation and write in one launch: the pages, scales and rows of the separate calls."""
    cfg = config(d=d, hq=hq, hkv=hkv, kv=kv, block=128)
    rotary = RotaryEmbedding(d // 2, base=5.0e5, pairs="interleaved" if d == 128 else "half")
    lengths, fresh = [60, 9, 1, 300], [20, 0, 1, 70]
    n = sum(fresh) + 5
    gen = torch.Generator().manual_seed(7)
    qkv = rows(gen, n, hq + 2 * hkv, d).to(cuda_device)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    weight = (1 + 0.2 * torch.randn(d, generator=gen)).to(cuda_device)
    cache = Cache(cfg, lengths, 8, scales="token" if scales == "token" else "none")
    lens, starts = torch.tensor(lengths, dtype=torch.int32, device=cuda_device), starts_of(fresh).to(cuda_device)
    weights = dict(q_weight=weight, k_weight=weight)

    pool, table, kw = cache.call(cuda_device)
    turned, turned_k = QueryKeyRotation(cfg, rotary)(q, k, lengths=lens, chunk_starts=starts, **weights)
    ChunkCacheWriter(cfg)(turned_k, v, pool, table, lens, chunk_starts=starts, **kw)
    want, want_lse = ChunkAttentionKernel(cfg)(turned, pool, table, lens, chunk_starts=starts, return_lse=True, **kw)

    pool2, _, kw2 = cache.call(cuda_device)
    step = ChunkStep(cfg, rotary)
    out, lse = step(q, k, v, pool2, table, lens, chunk_starts=starts, return_lse=True, **weights, **kw2)
    torch.cuda.synchronize()
    mine = slice(0, sum(fresh))
    assert torch.equal(bits(pool), bits(pool2))
    if kw:
        assert torch.equal(kw["token_scales"].view(torch.int32), kw2["token_scales"].view(torch.int32))
    assert torch.equal(out[mine], want[mine]) and torch.equal(lse[mine], want_lse[mine])


@pytest.mark.parametrize("kv", [FP8, BF16])
def test_token_by_token_as_the_prompt_at_once(kv, cuda_device):
    """Two sequences grow from nothing on pages handed out as they go, one token at a time
    in a graph; their prompts at once give the same rows to rounding, and the model's."""
    cfg = config(pcp=2, il=64, d=128, hq=16, hkv=2, kv=kv, block=64, bucket=512)
    rotary = RotaryEmbedding(128)
    total = [70, 131]
    gen = torch.Generator().manual_seed(9)
    tokens = [(rows(gen, n, 16, 128), rows(gen, n, 2, 128), rows(gen, n, 2, 128)) for n in total]
    pages = 2 * cfg.num_pages
    alloc = PageAllocator(cfg, cuda_device, num_pages=pages)
    table = torch.full((2, 2, cfg.max_local_blocks), -1, dtype=torch.int32, device=cuda_device)
    dtype = torch.float8_e4m3fn if kv == FP8 else torch.bfloat16
    pool = torch.full((pages, cfg.page_elements), math.nan, device=cuda_device).to(dtype)
    scales = empty_token_scales(cfg, cuda_device, num_pages=pages) if kv == FP8 else None
    step = ChunkStep(cfg, rotary)
    q, k, v = (torch.zeros((2, h, 128), dtype=torch.bfloat16, device=cuda_device) for h in (16, 2, 2))
    lengths = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    graph = step.graphed(q, k, v, pool, table, lengths, token_scales=scales)
    steps = max(total)
    grown = [torch.zeros((n, 16, 128), dtype=torch.bfloat16) for n in total]
    for t in range(steps):
        for b, n in enumerate(total):
            at = min(t, n - 1)
            alloc.allocate(at, 1, table[b])
            for x, y in zip((q, k, v), tokens[b]):
                x[b] = y[at].to(cuda_device)
        lengths.copy_(torch.tensor([min(t + 1, n) for n in total], dtype=torch.int32))
        out = graph.replay()
        for b, n in enumerate(total):
            if t < n:
                grown[b][t] = out[b].cpu()
    pool2 = torch.full((pages, cfg.page_elements), math.nan, device=cuda_device).to(dtype)
    scales2 = empty_token_scales(cfg, cuda_device, num_pages=pages) if kv == FP8 else None
    packed = [torch.cat([t[i] for t in tokens]).to(cuda_device) for i in range(3)]
    lens, starts = torch.tensor(total, dtype=torch.int32, device=cuda_device), starts_of(total).to(cuda_device)
    whole = step(*packed, pool2, table, lens, chunk_starts=starts, token_scales=scales2)
    torch.cuda.synchronize()
    assert torch.equal(bits(pool), bits(pool2))
    turned, turned_k = QueryKeyRotation(cfg, rotary)(packed[0], packed[1], lengths=lens, chunk_starts=starts)
    keys = turned_k.cpu().split(total)
    cache = Cache(cfg, total, 10, scales="token" if kv == FP8 else "none",
                  tokens=[(keys[b], tokens[b][2]) for b in range(2)])
    want, _, bound, _ = attention(cfg, cache, turned.cpu(), total, total)
    for got in (whole.cpu(), torch.cat(grown)):
        assert ((got.double() - want).abs() - bound).max().item() <= 0


def test_the_prefills_writer_and_the_chunks_agree(cuda_device):
    """One sequence: the same bits from KVCacheWriter and ChunkCacheWriter with given scales."""
    cfg = config(pcp=4, il=64, d=256, hq=32, hkv=2, kv=FP8, block=128, bucket=1024)
    gen = torch.Generator().manual_seed(11)
    k, v = (rows(gen, 2, 300, 256).to(cuda_device) for _ in range(2))
    table = torch.randperm(cfg.num_pages, generator=gen).to(torch.int32).reshape(4, -1).to(cuda_device)
    pools = [torch.zeros((cfg.num_pages, cfg.page_elements), device=cuda_device).to(torch.float8_e4m3fn)
             for _ in range(2)]
    KVCacheWriter(cfg)(k, v, pools[0], table, first_pos=100, k_scale=0.05, v_scale=0.07)
    ChunkCacheWriter(cfg)(k.transpose(0, 1), v.transpose(0, 1), pools[1], table,
                          torch.tensor([400], dtype=torch.int32, device=cuda_device), k_scale=0.05, v_scale=0.07)
    torch.cuda.synchronize()
    assert torch.equal(bits(pools[0]), bits(pools[1]))
