"""Norms and rotation of Q and K against a 64-bit model."""

from __future__ import annotations

import math

import pytest
import torch

from aws_training_study_amd.pcp_attention import QueryKeyRotation, RotaryEmbedding, stacked_query
from chunk_model import HALF_STEP, config, rows, starts_of

pytestmark = pytest.mark.gpu


def model(x, positions, rotary, weight, eps):
    """(rotated rows, bound of their error), float64.

    In 32 bits a norm's factor is off by at most 2^-20 relative to it (a sum of up
    to 256 squares, a division and a root), an angle's cosine and sine by 2^-20
    (the reduced angle is rounded to 32 bits, 2^-25 of a turn), each product by
    2^-24; the result is rounded to BF16 once.
    """
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + eps) * weight.double()
    dim = rotary.rotary_dim
    i = torch.arange(dim // 2)
    a, b = (i, i + dim // 2) if rotary.pairs == "half" else (2 * i, 2 * i + 1)
    angle = positions.double()[:, None, None] * rotary.frequencies()
    cos, sin = rotary.amplitude * torch.cos(angle), rotary.amplitude * torch.sin(angle)
    out, size = x.clone(), x.abs()
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = abs(rotary.amplitude) * (x[..., a].abs() + x[..., b].abs())
    return out, HALF_STEP * out.abs() + 2.0**-19 * size


def check(got, expected):
    want, bound = expected
    worst = ((got.cpu().double() - want).abs() - bound).max().item()
    assert worst <= 0, f"off by {worst} more than its bound"


ROTARIES = {
    "half": RotaryEmbedding(64),
    "interleaved": RotaryEmbedding(64, pairs="interleaved", base=500000.0),
    "part": RotaryEmbedding(16, base=1.0e7),
    "part_interleaved": RotaryEmbedding(48, pairs="interleaved"),
    "linear": RotaryEmbedding(64, scaling="linear", factor=4.0),
    "base": RotaryEmbedding(32, scaling="base", factor=8.0),
    "by_parts": RotaryEmbedding(64, scaling="by_parts", factor=16.0, original_len=4096,
                                amplitude=1.0 + 0.1 * math.log(16.0)),
}


@pytest.mark.parametrize("weights", ["none", "both", "q", "float32"])
@pytest.mark.parametrize("name", ROTARIES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (28, 4, 128), (5, 5, 256)])
def test_rows_at_positions(hq, hkv, d, name, weights, cuda_device):
    rotary = ROTARIES[name]
    cfg = config(hq=hq, hkv=hkv, d=d)
    gen = torch.Generator().manual_seed(1)
    n = 37
    qkv = rows(gen, n, hq + 2 * hkv, d)
    positions = torch.randint(0, 1 << 20, (n,), generator=gen, dtype=torch.int64)
    positions[:4] = torch.tensor([0, 1, 2**31 - 1, 131072])
    wq, wk = (1 + 0.3 * torch.randn(d, generator=gen) for _ in range(2))
    if weights != "float32":
        wq, wk = wq.to(torch.bfloat16), wk.to(torch.bfloat16)
    wq, wk = (None if weights == "none" else wq), (None if weights in ("none", "q") else wk)
    op = QueryKeyRotation(cfg, rotary, norm_eps=1e-5)
    on_gpu = qkv.to(cuda_device)
    to = lambda w: None if w is None else w.to(cuda_device)  # noqa: E731
    for dtype in (torch.int64, torch.int32):
        q, k = op(on_gpu[:, :hq], on_gpu[:, hq:hq + hkv], positions=positions.to(cuda_device, dtype),
                  q_weight=to(wq), k_weight=to(wk))
        torch.cuda.synchronize()
        check(q, model(qkv[:, :hq], positions, rotary, wq, 1e-5))
        check(k, model(qkv[:, hq:hq + hkv], positions, rotary, wk, 1e-5))
    # in place, in the projection's own rows, V left as it is
    q, k = on_gpu[:, :hq], on_gpu[:, hq:hq + hkv]
    before = (op(q, k, positions=positions.to(cuda_device), q_weight=to(wq), k_weight=to(wk)), on_gpu.clone())
    op(q, k, positions=positions.to(cuda_device), q_weight=to(wq), k_weight=to(wk), q_out=q, k_out=k)
    torch.cuda.synchronize()
    assert torch.equal(q, before[0][0]) and torch.equal(k, before[0][1])
    assert torch.equal(on_gpu[:, hq + hkv:], before[1][:, hq + hkv:])


@pytest.mark.parametrize("lengths,fresh,first", [
    ([1], [1], 0), ([700, 3, 9, 64], [1, 1, 1, 1], 0), ([5, 0, 30, 1], [5, 0, 30, 1], 3),
    ([7 * i + 1 for i in range(130)], [i % 3 for i in range(130)], 1), ([2], [5], 0),
])
def test_rows_of_a_chunk(lengths, fresh, first, cuda_device):
    cfg = config(hq=8, hkv=2, d=128)
    rotary = ROTARIES["half"]
    op = QueryKeyRotation(cfg, rotary)
    n = first + sum(fresh) + 4
    gen = torch.Generator().manual_seed(2)
    q, k = rows(gen, n, 8, 128), rows(gen, n, 2, 128)
    q_out, k_out = (torch.full_like(x, 9.0).to(cuda_device) for x in (q, k))
    op(q.to(cuda_device), k.to(cuda_device), lengths=torch.tensor(lengths, dtype=torch.int32, device=cuda_device),
       chunk_starts=starts_of(fresh, first).to(cuda_device), q_out=q_out, k_out=k_out)
    torch.cuda.synchronize()
    positions = torch.tensor([m - f + i for m, f in zip(lengths, fresh) for i in range(f)])
    mine = slice(first, first + sum(fresh))
    for got, x in ((q_out, q), (k_out, k)):
        check(got[mine], model(x[mine], positions, rotary, None, 0.0))
        assert bool((got[:first] == 9.0).all()) and bool((got[first + sum(fresh):] == 9.0).all())
    if len(set(fresh)) == 1:
        each, _ = op(q[mine].to(cuda_device), k[mine].to(cuda_device),
                     lengths=torch.tensor(lengths, dtype=torch.int32, device=cuda_device))
        assert torch.equal(each, q_out[mine])


@pytest.mark.parametrize("pcp,il,hq,hkv,d", [(4, 16, 8, 2, 64), (1, 64, 5, 5, 256), (3, 48, 28, 4, 128)])
def test_laid_out_for_a_prefill(pcp, il, hq, hkv, d, cuda_device):
    cfg = config(pcp=pcp, il=il, block=64 if il != 48 else 192, hq=hq, hkv=hkv, d=d).with_overrides(
        current_len=pcp * il * 3)
    n = cfg.current_len
    gen = torch.Generator().manual_seed(3)
    qkv = rows(gen, n, hq + 2 * hkv, d)
    weight = (1 + 0.3 * torch.randn(d, generator=gen)).to(torch.bfloat16)
    rotary = RotaryEmbedding(d, base=1.0e6)
    on_gpu = qkv.to(cuda_device)
    q, k, v = on_gpu[:, :hq], on_gpu[:, hq:hq + hkv], on_gpu[:, hq + hkv:]
    op = QueryKeyRotation(cfg, rotary)
    first = 130001
    stacked, kv = op.prefill(q, k, v, first_pos=first, q_weight=weight.to(cuda_device),
                             k_weight=weight.to(cuda_device))
    rotated, rotated_k = op(q, k, positions=torch.arange(first, first + n, device=cuda_device),
                            q_weight=weight.to(cuda_device), k_weight=weight.to(cuda_device))
    torch.cuda.synchronize()
    positions = torch.arange(first, first + n)
    check(rotated, model(qkv[:, :hq], positions, rotary, weight, 1e-6))
    assert torch.equal(stacked, stacked_query(rotated.transpose(0, 1).contiguous(), cfg))
    assert torch.equal(kv[0], rotated_k.transpose(0, 1))
    assert torch.equal(kv[1], v.transpose(0, 1))


def test_many_rows_take_several_heads_a_wave(cuda_device):
    """Enough tokens that a wave goes through several groups of a token's heads."""
    cfg = config(hq=28, hkv=4, d=128)
    rotary = ROTARIES["half"]
    gen = torch.Generator().manual_seed(4)
    n = 3001
    q, k = rows(gen, n, 28, 128), rows(gen, n, 4, 128)
    positions = torch.randint(0, 1 << 17, (n,), generator=gen)
    weight = (1 + 0.3 * torch.randn(128, generator=gen)).to(torch.bfloat16)
    got_q, got_k = QueryKeyRotation(cfg, rotary)(
        q.to(cuda_device), k.to(cuda_device), positions=positions.to(cuda_device), q_weight=weight.to(cuda_device),
        k_weight=weight.to(cuda_device))
    torch.cuda.synchronize()
    check(got_q, model(q, positions, rotary, weight, 1e-6))
    check(got_k, model(k, positions, rotary, weight, 1e-6))


def test_values_that_are_not_finite_stay_in_their_row(cuda_device):
    cfg = config(hq=8, hkv=2, d=64)
    op = QueryKeyRotation(cfg, ROTARIES["half"])
    gen = torch.Generator().manual_seed(5)
    q, k = rows(gen, 9, 8, 64), rows(gen, 9, 2, 64)
    positions = torch.arange(9, device=cuda_device)
    weight = torch.ones(64, device=cuda_device)
    clean = op(q.to(cuda_device), k.to(cuda_device), positions=positions, q_weight=weight, k_weight=weight)
    q[4, 3, 7], k[2, 1, 60] = math.nan, math.inf
    got = op(q.to(cuda_device), k.to(cuda_device), positions=positions, q_weight=weight, k_weight=weight)
    torch.cuda.synchronize()
    for x, y, at in ((got[0], clean[0], (4, 3)), (got[1], clean[1], (2, 1))):
        other = torch.ones(x.shape[:2], dtype=torch.bool, device=cuda_device)
        other[at] = False
        assert torch.equal(x[other], y[other])


def test_a_graph_follows_lengths(cuda_device):
    cfg = config(hq=8, hkv=2, d=128)
    op = QueryKeyRotation(cfg, ROTARIES["half"])
    gen = torch.Generator().manual_seed(6)
    q, k = rows(gen, 3, 8, 128).to(cuda_device), rows(gen, 3, 2, 128).to(cuda_device)
    lengths = torch.tensor([5, 9, 700], dtype=torch.int32, device=cuda_device)
    op(q, k, lengths=lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(q, k, lengths=lengths)
    for step in range(3):
        lengths += 1
        graph.replay()
        want = op(q, k, lengths=lengths)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), step
