"""Attention of chunks of new tokens over paged caches, against a 64-bit model.

Every slot that no token owns holds NaN, so a key read by mistake shows.
"""

from __future__ import annotations

import math

import pytest
import torch

from aws_training_study_amd.pcp_attention import (
    ChunkAttentionKernel,
    KVCacheWriter,
    build_page_pool,
    make_history_attention_kernel,
)
from chunk_model import BF16, FP8, Cache, attention, config, rows, starts_of

pytestmark = pytest.mark.gpu


def run(kernel, cache, q, lengths, fresh, device, *, first=0, starts=True, out=None, **kw):
    pool, table, scales = cache.call(device)
    chunk_starts = starts_of(fresh, first).to(device) if starts else None
    got = kernel(q.to(device), pool, table, torch.tensor(lengths, dtype=torch.int32, device=device),
                 chunk_starts=chunk_starts, out=out, return_lse=True, **scales, **kw)
    torch.cuda.synchronize()
    return tuple(x.cpu() for x in got)


def check(got, expected, rows_of=slice(None)):
    out, lse = (x[rows_of] for x in got)
    want, want_lse, bound, lse_bound = (x[rows_of] for x in expected)
    worst = ((out.double() - want).abs() - bound).max().item()
    assert worst <= 0, f"output off by {worst} more than its bound"
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    off = ((lse.double() - want_lse)[~empty].abs() - lse_bound[~empty])
    assert off.numel() == 0 or off.max().item() <= 0


CASES = {
    # one token of one sequence, of several, with one key, at page and tile ends
    "one": (dict(), [1], [1]),
    "one_each": (dict(), [1, 2, 63, 64, 65, 127, 128, 129, 700], [1] * 9),
    "one_each_d128_fp8": (dict(d=128, kv=FP8, hq=28, hkv=4, block=128), [300, 1, 64, 511], [1] * 4),
    "one_each_d256_fp8": (dict(d=256, kv=FP8, hq=32, hkv=2, block=512, bucket=2048), [2048, 31, 513], [1] * 3),
    "one_each_d256_bf16": (dict(d=256, hq=32, hkv=2, block=64), [1000, 31, 513], [1] * 3),
    "one_head_each": (dict(d=128, hq=6, hkv=6), [77, 200], [1, 1]),
    "many_sequences": (dict(hq=4, hkv=1, bucket=256), [(7 * i) % 250 + 1 for i in range(150)], [1] * 150),
    # a long walk over few rows
    "long": (dict(d=64, block=256, bucket=20000), [19997], [1]),
    "long_striped": (dict(pcp=5, il=32, block=64, d=128, kv=FP8, hq=10, hkv=2, bucket=9000), [8765], [2]),
    "one_long_many_short": (dict(d=128, kv=FP8, hq=16, hkv=2, block=128, bucket=9000), [9, 8990, 1, 30, 8], [1] * 5),
    # chunks of several tokens
    "few_rows": (dict(hq=16, hkv=1), [300, 150, 77], [2, 3, 4]),
    "ragged": (dict(d=128, hq=8, hkv=4, block=128), [500, 64, 1, 333, 90, 2], [70, 0, 1, 5, 33, 2]),
    "ragged_fp8_d256": (dict(d=256, kv=FP8, hq=32, hkv=2), [200, 300, 5], [11, 40, 5]),
    "ragged_bf16_d256": (dict(d=256, hq=16, hkv=4), [190, 260, 5], [11, 60, 5]),
    "striped_chunk": (dict(pcp=4, il=16, block=128, hq=8, hkv=2), [777, 100], [130, 100]),
    "striped_uneven": (dict(pcp=3, il=48, block=192, hq=24, hkv=8, kv=FP8), [500, 144, 145], [45, 144, 3]),
    "striped_rank_without_tokens": (dict(pcp=16, il=64, hq=8, hkv=2, block=64), [70, 65], [70, 1]),
    # whole prompts
    "prompts": (dict(d=128, hq=16, hkv=2, block=64), [129, 1, 64, 300, 257], [129, 1, 64, 300, 257]),
    "prompts_fp8_d256": (dict(d=256, kv=FP8, hq=32, hkv=2, block=128), [200, 65], [200, 65]),
    "prompts_fp8_d64": (dict(d=64, kv=FP8, hq=24, hkv=8, block=64), [200, 65], [200, 65]),
    # rows enough to fill the GPU several times over (walks are not cut into ranges)
    "many_rows": (dict(d=64, hq=32, hkv=2, bucket=640), [600, 520, 1], [600, 520, 1]),
    "many_rows_fp8": (dict(d=128, kv=FP8, hq=32, hkv=2, bucket=1280), [640, 1280, 3], [500, 620, 1]),
    # rows enough for the kernel that shares its tiles, with walks that are cut and not
    "many_d64_long": (dict(d=64, hq=64, hkv=2, block=128, bucket=1280), [1000, 90], [70, 20]),
    "many_d128_fp8_long": (dict(d=128, kv=FP8, hq=64, hkv=2, bucket=1280), [700], [70]),
    "many_d128_striped": (dict(pcp=3, il=48, block=192, d=128, hq=64, hkv=2), [300, 0, 200], [70, 0, 31]),
    "many_d256": (dict(d=256, hq=64, hkv=2, bucket=640), [600, 33], [70, 33]),
    "many_d256_fp8": (dict(pcp=2, il=32, block=64, d=256, kv=FP8, hq=64, hkv=2, bucket=640), [600, 33], [70, 33]),
    "many_empty_rows": (dict(d=128, hq=64, hkv=2), [5, 0, 70], [60, 3, 71]),
    # more new tokens than the cache holds (rows that see nothing), empty caches
    "empty_rows": (dict(d=128, hq=8, hkv=2), [5, 0, 0, 130], [9, 3, 0, 131]),
    "empty_rows_fp8": (dict(d=256, kv=FP8, hq=32, hkv=2), [2, 0], [4, 1]),
}


@pytest.mark.parametrize("name,scales", [(name, s) for name, (options, *_) in CASES.items()
                                         for s in (("plain", "token", "tensor") if "kv" in options else ("plain",))])
def test_against_the_model(name, scales, cuda_device):
    options, lengths, fresh = CASES[name]
    cfg = config(**options)
    kind = "none" if scales == "plain" else scales
    print(f"case {name} {scales}", flush=True)
    cache = Cache(cfg, lengths, 5, scales=kind, table_dtype=torch.int64 if len(lengths) % 2 else torch.int32)
    q = rows(torch.Generator().manual_seed(6), sum(fresh), cfg.num_q_heads, cfg.head_dim)
    got = run(ChunkAttentionKernel(cfg), cache, q, lengths, fresh, cuda_device)
    check(got, attention(cfg, cache, q, lengths, fresh))


@pytest.mark.parametrize("name", ["one_each", "one_each_d256_fp8", "long", "prompts_fp8_d256"])
def test_without_starts(name, cuda_device):
    """Sequences of as many rows each give the bits of the same call with starts."""
    options, lengths, _ = CASES[name]
    each = 1 if name.startswith(("one", "long")) else 65
    lengths, fresh = [max(n, each) for n in lengths], [each] * len(lengths)
    cfg = config(**options)
    cache = Cache(cfg, lengths, 7)
    q = rows(torch.Generator().manual_seed(8), sum(fresh), cfg.num_q_heads, cfg.head_dim)
    kernel = ChunkAttentionKernel(cfg)
    got = run(kernel, cache, q, lengths, fresh, cuda_device, starts=False)
    check(got, attention(cfg, cache, q, lengths, fresh))


def test_rows_of_no_sequence_stay(cuda_device):
    cfg = config(d=128, hq=16, hkv=2)
    lengths, fresh = [300, 40, 64], [30, 0, 7]
    cache = Cache(cfg, lengths, 9)
    q = rows(torch.Generator().manual_seed(10), 5 + sum(fresh) + 20, cfg.num_q_heads, cfg.head_dim)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=cuda_device)
    got = run(ChunkAttentionKernel(cfg), cache, q, lengths, fresh, cuda_device, first=5, out=out)
    mine = slice(5, 5 + sum(fresh))
    check(got, attention(cfg, cache, q, lengths, fresh, first=5), mine)
    assert bool((got[0][:5] == 7.0).all()) and bool((got[0][5 + sum(fresh):] == 7.0).all())


def test_no_rows(cuda_device):
    cfg = config()
    cache = Cache(cfg, [10], 11)
    q = torch.empty((0, cfg.num_q_heads, cfg.head_dim), dtype=torch.bfloat16)
    out, lse = run(ChunkAttentionKernel(cfg), cache, q, [10], [0], cuda_device)
    assert out.shape == q.shape and lse.shape == (0, cfg.num_q_heads)


@pytest.mark.parametrize("dtype,bad", [(torch.int32, [-1, -7, 10**6]), (torch.int64, [-1, 2**32, 2**40 + 1])])
@pytest.mark.parametrize("fresh", [[1], [90], [600]])
def test_entries_of_no_page(dtype, bad, fresh, cuda_device):
    """Keys of a table entry that names no page are seen by nobody."""
    cfg = config(pcp=2, il=64, block=64, d=128, hq=8, hkv=2, bucket=1024)
    lengths = [900]
    cache = Cache(cfg, lengths, 12, table_dtype=dtype)
    hidden = torch.zeros(900, dtype=torch.bool)
    for i, value in enumerate(bad):
        rank, block = i % 2, 1 + i
        cache.table[0, rank, block] = value
        for p in range(900):
            chunk = p // 64
            hidden[p] |= chunk % 2 == rank and (chunk // 2) == block
    q = rows(torch.Generator().manual_seed(13), sum(fresh), cfg.num_q_heads, cfg.head_dim)
    got = run(ChunkAttentionKernel(cfg), cache, q, lengths, fresh, cuda_device)
    check(got, attention(cfg, cache, q, lengths, fresh, hidden=[hidden]))


def test_lengths_beyond_the_cache(cuda_device):
    """Positions past the table see the cache that there is."""
    cfg = config(bucket=256, d=64)
    cache = Cache(cfg, [256], 14)
    q = rows(torch.Generator().manual_seed(15), 3, cfg.num_q_heads, cfg.head_dim)
    got = run(ChunkAttentionKernel(cfg), cache, q, [2000], [3], cuda_device)
    check(got, attention(cfg, cache, q, [2000], [3]))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d,kv", [(64, BF16), (128, BF16), (256, BF16), (128, FP8), (256, FP8)])
@pytest.mark.parametrize("fresh", [3, 100, 300])
def test_a_later_token_that_is_not_finite(bad, d, kv, fresh, cuda_device):
    """Rows before a token with a K or V that is not finite keep their results."""
    cfg = config(d=d, kv=kv, hq=16, hkv=2, block=128)
    n = max(150, fresh + 50)
    gen = torch.Generator().manual_seed(16)
    k, v = rows(gen, n, cfg.num_kv_heads, d), rows(gen, n, cfg.num_kv_heads, d)
    q = rows(gen, fresh, cfg.num_q_heads, d)
    clean = Cache(cfg, [n], 17, scales="token" if kv == FP8 else "none", tokens=[(k, v)])
    expected = attention(cfg, clean, q, [n], [fresh])
    spoiled_v = v.clone()
    spoiled_v[n - 2, :, 5] = bad
    spoiled_v[n - 2, 1, d - 1] = bad
    cache = Cache(cfg, [n], 17, scales="token" if kv == FP8 else "none", tokens=[(k, spoiled_v)])
    got = run(ChunkAttentionKernel(cfg), cache, q, [n], [fresh], cuda_device)
    check(got, expected, slice(0, fresh - 2))
    # the rows that see it: that column is lost, the others are right
    assert not bool(torch.isfinite(got[0][fresh - 2:, :, 5]).any())
    others = torch.ones(d, dtype=torch.bool)
    others[[5, d - 1]] = False
    if kv == BF16:  # (in an e4m3 cache the row's scale comes from the finite values, which changed)
        off = (got[0][fresh - 2:].double() - expected[0][fresh - 2:]).abs() - expected[2][fresh - 2:]
        assert off[..., others].max().item() <= 0
    # a K that is not finite: the rows that see it are lost, the others right
    spoiled_k = k.clone()
    spoiled_k[n - 2] = math.nan
    cache = Cache(cfg, [n], 17, scales="token" if kv == FP8 else "none", tokens=[(spoiled_k, v)])
    got = run(ChunkAttentionKernel(cfg), cache, q, [n], [fresh], cuda_device)
    check(got, expected, slice(0, fresh - 2))
    assert bool(torch.isnan(got[0][fresh - 2:]).all())


def test_far_pages(cuda_device):
    """Pages whose bytes lie past 2^32."""
    cfg = config(d=256, hq=32, hkv=2, block=512, bucket=2048)
    lengths, fresh = [1500], [1]
    cache = Cache(cfg, lengths, 18)
    pages = 4200  # 1 MiB each
    shift = pages - cache.num_pages
    assert pages * cfg.page_elements * 2 > 2**32
    pool = torch.empty((pages, cfg.page_elements), dtype=torch.bfloat16, device=cuda_device)
    pool[shift:] = cache.pages().to(cuda_device)
    table = torch.where(cache.table >= 0, cache.table + shift, cache.table).to(cuda_device)
    kernel = ChunkAttentionKernel(cfg)
    for f in (1, 40):
        q = rows(torch.Generator().manual_seed(19), f, cfg.num_q_heads, cfg.head_dim)
        got = kernel(q.to(cuda_device), pool, table, torch.tensor(lengths, dtype=torch.int32, device=cuda_device),
                     return_lse=True)
        torch.cuda.synchronize()
        check(tuple(x.cpu() for x in got), attention(cfg, cache, q, lengths, [f]))


def test_large_scores(cuda_device):
    """Scores of hundreds: the running maximum keeps the exponentials in range."""
    cfg = config(d=128, hq=8, hkv=2, block=64)
    lengths, fresh = [400, 70], [50, 1]
    gen = torch.Generator().manual_seed(20)
    tokens = [((30 * rows(gen, n, 2, 128).float()).to(torch.bfloat16), rows(gen, n, 2, 128)) for n in lengths]
    cache = Cache(cfg, lengths, 21, tokens=tokens)
    q = rows(gen, sum(fresh), 8, 128)
    got = run(ChunkAttentionKernel(cfg), cache, q, lengths, fresh, cuda_device)
    check(got, attention(cfg, cache, q, lengths, fresh))


@pytest.mark.parametrize("name", ["one_long_many_short", "ragged_fp8_d256", "long"])
def test_the_same_bits_each_time(name, cuda_device):
    options, lengths, fresh = CASES[name]
    cfg = config(**options)
    cache = Cache(cfg, lengths, 22)
    q = rows(torch.Generator().manual_seed(23), sum(fresh), cfg.num_q_heads, cfg.head_dim)
    kernel = ChunkAttentionKernel(cfg)
    first = run(kernel, cache, q, lengths, fresh, cuda_device)
    for _ in range(3):
        again = run(kernel, cache, q, lengths, fresh, cuda_device)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_streams_of_their_own(cuda_device):
    """Calls in flight on two streams do not share partial results."""
    cfg = config(d=128, kv=FP8, hq=16, hkv=2, block=256, bucket=20000)
    kernel = ChunkAttentionKernel(cfg)
    problems = []
    for i, n in enumerate((19000, 12345)):
        cache = Cache(cfg, [n], 24 + i)
        q = rows(torch.Generator().manual_seed(26 + i), 1, cfg.num_q_heads, cfg.head_dim)
        pool, table, kw = cache.call(cuda_device)
        problems.append((q.to(cuda_device), pool, table, torch.tensor([n], dtype=torch.int32, device=cuda_device), kw))
    alone = []
    for q, pool, table, lengths, kw in problems:
        alone.append(kernel(q, pool, table, lengths, **kw))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    for _ in range(20):
        outs = []
        for s, (q, pool, table, lengths, kw) in zip(streams, problems):
            with torch.cuda.stream(s):
                outs.append(kernel(q, pool, table, lengths, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))


@pytest.mark.parametrize("fresh", [[1, 1, 1], [3, 0, 40]])
def test_graphs_follow_lengths(fresh, cuda_device):
    """Two graphs replayed in turn, with eager calls between, follow the tensors they captured."""
    cfg = config(d=128, kv=FP8, hq=16, hkv=2, block=128, bucket=6000)
    full = [6000, 500, 4000]
    cache = Cache(cfg, full, 28, scales="token")
    pool, table, kw = cache.call(cuda_device)
    kernel = ChunkAttentionKernel(cfg)
    starts = starts_of(fresh).to(cuda_device)
    graphs = []
    for seed in (29, 30):
        q = rows(torch.Generator().manual_seed(seed), sum(fresh), 16, 128).to(cuda_device)
        lengths = torch.tensor([3000, 77, 100], dtype=torch.int32, device=cuda_device)
        graphs.append((q, lengths, kernel.graphed(q, pool, table, lengths, chunk_starts=starts, return_lse=True, **kw)))
    for lens in ([3000, 77, 100], [6000, 500, 4000], [40, 41, 3999]):
        for q, lengths, graph in graphs:
            lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        replayed = [graph.replay() for _, _, graph in graphs]
        for (q, lengths, _), (out, lse) in zip(graphs, replayed):
            want, want_lse = kernel(q, pool, table, lengths, chunk_starts=starts, return_lse=True, **kw)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_a_capture_of_the_callers_own(cuda_device):
    """Two plain calls captured by hand on one stream and replayed on two at once."""
    cfg = config(d=128, kv=FP8, hq=16, hkv=2, block=256, bucket=20000)
    kernel = ChunkAttentionKernel(cfg)
    cache = Cache(cfg, [19000], 31)
    pool, table, kw = cache.call(cuda_device)
    lengths = torch.tensor([19000], dtype=torch.int32, device=cuda_device)
    captured = []
    for seed in (32, 33):
        q = rows(torch.Generator().manual_seed(seed), 1, 16, 128).to(cuda_device)
        want = kernel(q, pool, table, lengths, **kw)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernel(q, pool, table, lengths, **kw)
        captured.append((graph, out, want, q))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (graph, *_) in zip(streams, captured):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _ in captured)


def test_over_a_prefills_cache(cuda_device):
    """One token over the pool that the producer filled: the history kernel's result
    for that query, as every key of the history lies before it."""
    cfg = config(pcp=4, il=64, block=128, d=256, hq=32, hkv=2, kv=FP8, bucket=2048)
    gen = torch.Generator().manual_seed(34)
    k, v = rows(gen, 2, 2048, 256), rows(gen, 2, 2048, 256)
    table = torch.randperm(cfg.num_pages, generator=gen).to(torch.int32).reshape(4, -1).to(cuda_device)
    pool, k_scale, v_scale, valid = build_page_pool(cfg, k.to(cuda_device), v.to(cuda_device), table)
    q = rows(gen, cfg.current_len, 32, 256).to(cuda_device)
    history = make_history_attention_kernel(cfg)
    stacked = q.view(1, 4, 64, 32, 256).permute(1, 3, 0, 2, 4).reshape(4, 32, 64, 256).contiguous()
    want, want_lse = history(stacked, pool, table, page_valid_len=valid, k_scale=k_scale, v_scale=v_scale,
                             precision="bf16", return_lse=True)
    kernel = ChunkAttentionKernel(cfg)
    lengths = torch.tensor([2048], dtype=torch.int32, device=cuda_device)
    for row in (0, 100, 255):
        out, lse = kernel(q[row:row + 1], pool, table, lengths, k_scale=k_scale, v_scale=v_scale, return_lse=True)
        rank, tok = row // 64, row % 64
        torch.cuda.synchronize()
        # the same products rounded at other places: P's and the outputs' roundings
        assert (out[0].float() - want[rank, :, tok].float()).abs().max().item() < 2e-2
        assert (lse[0] - want_lse[rank, :, tok]).abs().max().item() < 1e-3
    # and a token appended by the producer of the prefill
    more = config(pcp=4, il=64, block=128, d=256, hq=32, hkv=2, kv=FP8, bucket=2048 + 256)
    table2 = torch.full((4, more.max_local_blocks), -1, dtype=torch.int32, device=cuda_device)
    table2[:, :table.shape[1]] = table
    pool2 = torch.cat((pool, torch.zeros_like(pool[:1])))
    table2[0, table.shape[1]] = pool.shape[0]
    k1, v1 = (rows(gen, 2, 1, 256).to(cuda_device) for _ in range(2))
    KVCacheWriter(more)(k1, v1, pool2, table2, first_pos=2048, k_scale=k_scale, v_scale=v_scale)
    out, lse = ChunkAttentionKernel(more)(q[:1], pool2, table2, lengths + 1, k_scale=k_scale, v_scale=v_scale,
                                          return_lse=True)
    # the new key's score joins the history's log-sum-exp
    code = (k1[:, 0].float() / k_scale).to(torch.float8_e4m3fn).double() * k_scale
    s = (q[0].double().view(2, 16, 256) * code[:, None]).sum(-1).reshape(-1) / 16.0
    want = torch.logaddexp(want_lse[0, :, 0].double(), s)
    assert (lse[0].double() - want).abs().max().item() < 1e-3
