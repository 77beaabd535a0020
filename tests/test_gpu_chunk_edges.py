"""Calls of the serving operators at the edges of what they take: outputs that are inputs or
share their memory, scores near the type's end, chunks unlike their average, two threads on
one stream."""

from __future__ import annotations

import math
import threading

import pytest
import torch

from aws_training_study_amd.pcp_attention import ChunkAttentionKernel, ChunkStep, QueryKeyRotation, RotaryEmbedding
from chunk_model import FP8, HALF_STEP, Cache, attention, config, rows, starts_of
from test_gpu_chunk_attention import check, run

pytestmark = pytest.mark.gpu


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


# ---- memory that inputs and outputs share ------------------------------------------


@pytest.mark.parametrize("pairs,weights", [("half", True), ("interleaved", False)])
def test_rotation_in_place_within_one_projection(pairs, weights, cuda_device):
    cfg = config(hq=8, hkv=2, d=128)
    op = QueryKeyRotation(cfg, RotaryEmbedding(64, pairs=pairs))
    projected = rows(torch.Generator().manual_seed(1), 37, 12, 128).to(cuda_device)
    positions = torch.arange(5, 42, dtype=torch.int64, device=cuda_device)
    kw = dict(positions=positions)
    if weights:
        kw.update(q_weight=torch.rand(128, device=cuda_device), k_weight=torch.rand(128, device=cuda_device))
    want = op(projected[:, :8], projected[:, 8:10], **kw)
    for _ in range(2):  # (the second on the native path)
        mine = projected.clone()
        q, k = mine[:, :8], mine[:, 8:10]
        got = op(q, k, q_out=q, k_out=k, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(mine[:, 10:], projected[:, 10:])
    # contiguous rows in place
    q, k = projected[:, :8].contiguous(), projected[:, 8:10].contiguous()
    op(q, k, q_out=q, k_out=k, **kw)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rotations_into_others_memory_are_refused(cuda_device):
    cfg = config(hq=4, hkv=4, d=64)
    op = QueryKeyRotation(cfg, RotaryEmbedding(64))
    step = ChunkStep(cfg, RotaryEmbedding(64))
    lengths = [9]
    pool, table, _ = Cache(cfg, lengths, 2).call(cuda_device)
    lengths = int32(lengths, cuda_device)
    buffer = rows(torch.Generator().manual_seed(3), 30, 4, 64).to(cuda_device)
    q, k, v = buffer[:9], buffer[10:19], buffer[20:29]
    cache = (pool, table, lengths)
    for _ in range(2):  # the general path, then the native one
        for bad in (dict(q_out=buffer[1:10]), dict(q_out=k), dict(k_out=buffer[11:20]), dict(k_out=q),
                    dict(q_out=buffer[20:29], k_out=buffer[21:30]),
                    dict(q_out=torch.as_strided(buffer, (9, 4, 64), (128, 0, 1)))):
            with pytest.raises(ValueError, match="_out"):
                op(q, k, lengths=lengths, **bad)
        for bad in (buffer[1:10], k, v, buffer[15:24]):
            with pytest.raises(ValueError, match="q_out"):
                step.prepare(q, k, v, *cache, q_out=bad)
        op(q, k, lengths=lengths, q_out=torch.empty_like(q))
        step.prepare(q.clone(), k, v, *cache, q_out=torch.empty_like(q))


def test_weights_at_odd_places_are_refused(cuda_device):
    cfg = config(hq=4, hkv=2, d=64)
    op = QueryKeyRotation(cfg, RotaryEmbedding(64))
    q, k = (rows(torch.Generator().manual_seed(4), 3, h, 64).to(cuda_device) for h in (4, 2))
    positions = int32([0, 1, 2], cuda_device)
    store = torch.ones(80, device=cuda_device)
    for _ in range(2):
        op(q, k, positions=positions, q_weight=store[4:68], k_weight=store.bfloat16()[4:68].float())
        for w in (store[1:65], store.bfloat16()[2:66]):
            with pytest.raises(ValueError, match="must start at a multiple of"):
                op(q, k, positions=positions, q_weight=w)
            with pytest.raises(ValueError, match="must start at a multiple of"):
                op(q, k, positions=positions, k_weight=w)


@pytest.mark.parametrize("options,lengths,fresh", [
    (dict(d=256, kv=FP8, hq=32, hkv=2, block=512, bucket=4096), [4000, 31], [1, 1]),  # ranges
    (dict(d=128, hq=4, hkv=4), [100, 31], [1, 1]),
    (dict(d=128, hq=8, hkv=1), [300, 77], [3, 3]),
    (dict(d=64, hq=16, hkv=2, bucket=512), [500, 300], [200, 300]),
    (dict(d=256, hq=32, hkv=2, bucket=640), [640, 640, 5], [600, 640, 5]),
])
def test_attention_into_q(options, lengths, fresh, cuda_device):
    cfg = config(**options)
    cache = Cache(cfg, lengths, 5)
    q = rows(torch.Generator().manual_seed(6), sum(fresh), cfg.num_q_heads, cfg.head_dim)
    kernel = ChunkAttentionKernel(cfg)
    want = run(kernel, cache, q, lengths, fresh, cuda_device)
    check(want, attention(cfg, cache, q, lengths, fresh))
    mine = q.to(cuda_device)
    got = run(kernel, cache, mine, lengths, fresh, cuda_device, out=mine)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # ... but not into a part of it
    pool, table, scales = cache.call(cuda_device)
    both = torch.empty((q.shape[0] + 1, *q.shape[1:]), dtype=q.dtype, device=cuda_device)
    with pytest.raises(ValueError, match="out must be its own input"):
        kernel(both[:-1], pool, table, int32(lengths, cuda_device), chunk_starts=starts_of(fresh).to(cuda_device),
               out=both[1:], **scales)


# ---- objects that go before their work --------------------------------------------------


def test_a_graph_outlives_the_rotation_it_recorded(cuda_device):
    cfg = config(hq=4, hkv=2, d=64)
    rotary = RotaryEmbedding(64, base=12345.0)
    q, k = (rows(torch.Generator().manual_seed(20), 9, h, 64).to(cuda_device) for h in (4, 2))
    positions = torch.arange(100, 109, dtype=torch.int32, device=cuda_device)
    want = [x.clone() for x in QueryKeyRotation(cfg, rotary)(q, k, positions=positions)]
    op = QueryKeyRotation(cfg, rotary)
    op(q, k, positions=positions)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, k, positions=positions)
    del op
    others = [torch.zeros(32, dtype=torch.float64, device=cuda_device) for _ in range(64)]
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        others[0].add_(1.0)


def test_a_first_call_under_capture_is_refused(cuda_device):
    cfg = config(hq=4, hkv=2, d=64)
    op = QueryKeyRotation(cfg, RotaryEmbedding(64, base=54321.0))
    q, k = (rows(torch.Generator().manual_seed(21), 3, h, 64).to(cuda_device) for h in (4, 2))
    positions = torch.arange(3, dtype=torch.int32, device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before a capture"):
            op(q, k, positions=positions)
        positions.add_(0)
    op(q, k, positions=positions)


# ---- scores --------------------------------------------------------------------------


@pytest.mark.parametrize("d,hq,fresh", [(64, 8, 1), (256, 8, 1), (256, 8, 100), (128, 8, 100), (64, 8, 5),
                                        (64, 32, 300), (128, 32, 300), (256, 32, 300)])
def test_scores_near_the_types_lowest(d, hq, fresh, cuda_device):
    """Scores of -2^120: all the same, so that each row is the mean of what it sees.

    P is 1 or one power of two, the sums of n of them are exact but for 2^-24 a
    term in the product with V; the result is rounded once."""
    cfg = config(d=d, hq=hq, hkv=2, bucket=512)
    n = 333
    gen = torch.Generator().manual_seed(7)
    k, v = torch.zeros(n, 2, d, dtype=torch.bfloat16), rows(gen, n, 2, d)
    k[:, :, 0] = -(2.0**62)
    cache = Cache(cfg, [n], 8, tokens=[(k, v)])
    q = torch.zeros(fresh, hq, d, dtype=torch.bfloat16)
    q[:, :, 0] = 2.0**62
    out, lse = run(ChunkAttentionKernel(cfg), cache, q, [n], [fresh], cuda_device)
    for i in range(fresh):
        seen = n - fresh + i + 1
        value = v[:seen].double().repeat_interleave(hq // 2, dim=1)
        mean, size = value.mean(dim=0), value.abs().mean(dim=0)
        worst = ((out[i].double() - mean).abs() - HALF_STEP * mean.abs() - 2 * seen * 2.0**-24 * size).max().item()
        assert worst <= 2.0**-40, worst
        assert (lse[i].double() / (-(2.0**124) * cfg.softmax_scale) - 1).abs().max().item() <= 2.0**-20


@pytest.mark.parametrize("hq", [4, 64])
def test_scores_of_minus_infinity(hq, cuda_device):
    """Rows whose scores are all -inf are zeros, as rows that see nothing; their neighbours are as ever."""
    cfg = config(d=128, hq=hq, hkv=2)
    lengths, fresh = [90, 70], [2, 70]
    cache = Cache(cfg, lengths, 9)
    q = rows(torch.Generator().manual_seed(10), 72, hq, 128)
    want = run(ChunkAttentionKernel(cfg), cache, q, lengths, fresh, cuda_device)
    k, v = cache.tokens[0]
    k = k.clone()
    k[:, :, 0] = -math.inf
    cache2 = Cache(cfg, lengths, 9, tokens=[(k, v), cache.tokens[1]])
    q2 = q.clone()
    q2[:2, :, 0] = 1.0
    out, lse = run(ChunkAttentionKernel(cfg), cache2, q2, lengths, fresh, cuda_device)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())
    check((out, lse), attention(cfg, cache2, q2, lengths, fresh), slice(2, None))
    check(want, attention(cfg, cache, q, lengths, fresh))


# ---- chunks unlike their average -------------------------------------------------------


UNEVEN = [
    # one prompt among many single tokens: on average few rows
    (dict(d=128, kv=FP8, hq=16, hkv=2, bucket=512), [1 + 5 * i for i in range(80)] + [500], [1] * 80 + [150]),
    (dict(d=256, hq=8, hkv=1, bucket=512), [300] + [1 + 3 * i for i in range(70)], [200] + [1] * 70),
    # one single token among prompts, and sequences without rows between
    (dict(d=64, hq=8, hkv=2, bucket=512), [500, 130, 9, 200], [300, 0, 1, 200]),
    # more sequences than a wave has lanes, many rows of each
    (dict(d=128, hq=8, hkv=1, bucket=256), [40 + i for i in range(140)], [5 + i % 9 for i in range(140)]),
    (dict(d=256, kv=FP8, hq=16, hkv=2, bucket=256), [40 + i for i in range(70)], [(i % 3) * 4 for i in range(70)]),
    # more sequences than the registers keep: of few rows, cut into ranges or not, and of many
    (dict(d=64, hq=2, hkv=1, bucket=1024), [1 + (37 * i) % 90 for i in range(299)] + [1000], [i % 3 for i in range(300)]),
    (dict(d=64, hq=2, hkv=1, bucket=128), [1 + (37 * i) % 90 for i in range(300)], [1] * 300),
    (dict(d=64, hq=8, hkv=1, bucket=1024), [20 + (37 * i) % 90 for i in range(299)] + [900], [6] * 300),
    # equal rows of many sequences without ranges
    (dict(d=64, hq=32, hkv=4, bucket=256), [100 + i for i in range(130)], [32] * 130),
]


@pytest.mark.parametrize("options,lengths,fresh,scales", [(*case, s) for case in UNEVEN
                                                          for s in (("none", "token") if "kv" in case[0] else ("none",))])
def test_uneven_chunks(options, lengths, fresh, scales, cuda_device):
    cfg = config(**options)
    print(f"{options} {len(lengths)} sequences", flush=True)
    cache = Cache(cfg, lengths, 11, scales=scales)
    q = rows(torch.Generator().manual_seed(12), sum(fresh), cfg.num_q_heads, cfg.head_dim)
    expected = attention(cfg, cache, q, lengths, fresh)
    kernel = ChunkAttentionKernel(cfg)
    check(run(kernel, cache, q, lengths, fresh, cuda_device), expected)
    if len(set(fresh)) == 1:
        check(run(kernel, cache, q, lengths, fresh, cuda_device, starts=False), expected)


# ---- two calls at once -------------------------------------------------------------------


def test_threads_on_one_stream(cuda_device):
    """Calls of two threads may be queued between each other's launches: their partial results
    are kept apart."""
    cfg = config(d=128, kv=FP8, hq=16, hkv=2, block=128, bucket=9000)
    lengths = [8990, 70]
    cache = Cache(cfg, lengths, 13)
    pool, table, scales = cache.call(cuda_device)
    table_lengths = int32(lengths, cuda_device)
    kernel = ChunkAttentionKernel(cfg)
    qs = [rows(torch.Generator().manual_seed(s), 2, 16, 128).to(cuda_device) for s in (14, 15)]
    assert kernel.workspace_bytes(2, 2, False) > 0
    want = [kernel(q, pool, table, table_lengths, **scales) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        results = [kernel(qs[i], pool, table, table_lengths, **scales) for _ in range(200)]
        torch.cuda.synchronize()
        if not all(torch.equal(r, want[i]) for r in results):
            wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
