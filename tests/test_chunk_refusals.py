"""What the serving operators refuse, before anything is launched (no GPU needed)."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from aws_training_study_amd import _native
from aws_training_study_amd.pcp_attention import (
    CacheReader,
    ChunkAttentionKernel,
    ChunkCacheWriter,
    QueryKeyRotation,
    RotaryEmbedding,
    empty_token_scales,
)
from aws_training_study_amd.pcp_attention.rotary import _check_output, _own_places, _rows, _share_memory
from chunk_model import FP8, config

HEADER = Path(__file__).resolve().parents[1] / "include" / "pcp_attention_hip.h"


@pytest.fixture(scope="module")
def lib():
    return _native.load_library()


@pytest.mark.parametrize("name,mirror", [("pcpa_chunk", _native.PcpaChunk), ("pcpa_rows", _native.PcpaRows),
                                         ("pcpa_rotary", _native.PcpaRotary)])
def test_struct_layout(name, mirror):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER.read_text(), re.S).group(1)
    fields = re.findall(r"^\s*(?:const )?(int32_t|int64_t|float|double|void)(\*?) (\w+);", body, re.M)
    assert [f[2] for f in fields] == [n for n, _ in mirror._fields_]
    sizes = {"int32_t": 4, "int64_t": 8, "float": 4}
    for (kind, star, _), (_, ctype) in zip(fields, mirror._fields_):
        assert ctypes.sizeof(ctype) == (8 if star else sizes[kind])


def params(**kw):
    p = dict(abi_version=_native.ABI_VERSION, pcp_size=4, num_q_heads=8, num_kv_heads=2, head_dim=64, local_q_len=64,
             block_size=128, max_local_blocks=4, num_pages=16, q_dtype=1, kv_dtype=2, out_dtype=1,
             softmax_scale=0.125, k_scale=1.0, v_scale=1.0, flags=0)
    p.update(kw)
    return ctypes.byref(_native.PcpaParams(**p))


def chunk(**kw):
    c = dict(interleave=64, batch=3, num_tokens=6, reserved=0, lengths=16, starts=None)
    c.update(kw)
    return ctypes.byref(_native.PcpaChunk(**c))


def rows(data=16, token=512, head=64):
    return ctypes.byref(_native.PcpaRows(data, token, head))


def rotary(**kw):
    r = dict(rotary_dim=64, interleaved=0, weight_dtype=1, amplitude=1.0, norm_eps=1e-6, turns=16, q_weight=None,
             k_weight=None)
    r.update(kw)
    return ctypes.byref(_native.PcpaRotary(**r))


BAD_CHUNKS = [(dict(interleave=0), -3), (dict(batch=0), -3), (dict(num_tokens=-1), -3), (dict(num_tokens=7), -3),
              (dict(reserved=1), -3), (dict(lengths=18), -6), (dict(starts=18), -6),
              (dict(num_tokens=3 << 28), -8), (dict(interleave=1 << 30), -8)]


@pytest.mark.parametrize("change,status", BAD_CHUNKS)
def test_chunks_refused_by_every_entry(lib, change, status):
    c = chunk(**change)
    assert lib.pcpa_chunk_attention(params(), c, 16, 16, None, 16, 16, None, None, 0, None) == status
    assert lib.pcpa_chunk_workspace_bytes(params(), c) == status
    assert lib.pcpa_chunk_write(params(), c, rows(), rows(), 16, 16, None, None) == status
    assert lib.pcpa_chunk_prepare(params(), c, rotary(), rows(), rows(), rows(), rows(), 16, 16, None, None) == status
    assert lib.pcpa_rotate(params(), c, rotary(), 16, 32, 0, rows(), rows(), None, rows(), rows(), None, 0,
                           None) == status


@pytest.mark.parametrize("args,status", [
    (dict(q=None), -1), (dict(pages=None), -1), (dict(table=None), -1), (dict(out=None), -1), (dict(q=24), -6),
    (dict(out=24), -6), (dict(pages=24), -6), (dict(table=18), -6), (dict(lse=18), -6), (dict(scales=24), -6),
    (dict(workspace=24), -6), (dict(bytes=-1), -10),
])
def test_attention_pointers(lib, args, status):
    a = dict(q=16, pages=16, scales=None, table=16, out=16, lse=None, workspace=None, bytes=0)
    a.update(args)
    assert lib.pcpa_chunk_attention(params(), chunk(), *a.values(), None) == status


def test_scales_go_with_an_e4m3_pool_and_no_others(lib):
    for p, status in ((params(kv_dtype=1), -4), (params(k_scale=0.5), -9), (params(v_scale=0.5), -9)):
        assert lib.pcpa_chunk_attention(p, chunk(), 16, 16, 16, 16, 16, None, None, 0, None) == status
        assert lib.pcpa_chunk_write(p, chunk(), rows(), rows(), 16, 16, 16, None) == status
        assert lib.pcpa_cache_read(p, 64, 0, 6, 16, 16, 16, 16, 16, None) == status


def test_launches_of_too_many_threads(lib):
    p = params(head_dim=256, num_q_heads=2, max_local_blocks=1 << 18)
    c = chunk(batch=1, num_tokens=(1 << 30) - 256)
    assert lib.pcpa_rotate(p, c, rotary(), 16, 32, 0, rows(), rows(), None, rows(), rows(), None, 0, None) == -8
    assert lib.pcpa_chunk_write(p, c, rows(), rows(), 16, 16, None, None) == -8
    assert lib.pcpa_cache_read(p, 64, 0, (1 << 30) - 256, 16, 16, None, 16, 16, None) == -8
    few = chunk(batch=(1 << 30) - 256, num_tokens=(1 << 30) - 256)
    assert lib.pcpa_chunk_attention(p, few, 16, 16, None, 16, 16, None, None, 0, None) == -8


def test_parameters_are_checked(lib):
    assert lib.pcpa_chunk_attention(params(head_dim=96), chunk(), 16, 16, None, 16, 16, None, None, 0, None) == -5
    assert lib.pcpa_chunk_attention(None, chunk(), 16, 16, None, 16, 16, None, None, 0, None) == -1
    assert lib.pcpa_chunk_attention(params(), None, 16, 16, None, 16, 16, None, None, 0, None) == -1
    assert lib.pcpa_chunk_attention(params(), chunk(lengths=None), 16, 16, None, 16, 16, None, None, 0, None) == -1
    # a cache of more positions than 32-bit indexes hold
    big = params(max_local_blocks=1 << 23, num_pages=16)
    assert lib.pcpa_chunk_write(big, chunk(), rows(), rows(), 16, 16, None, None) == -8


@pytest.mark.parametrize("change,status", [
    (dict(rotary_dim=8), -3), (dict(rotary_dim=80), -3), (dict(rotary_dim=-16), -3), (dict(turns=None), -1),
    (dict(turns=20), -6), (dict(amplitude=math.nan), -9), (dict(norm_eps=-1.0), -9), (dict(weight_dtype=2), -4),
    (dict(q_weight=17), -6), (dict(weight_dtype=3, k_weight=18), -6), (dict(q_weight=20), -6),
    (dict(weight_dtype=3, q_weight=24), -6), (dict(norm_eps=0.0), -9), (dict(norm_eps=2.0**-127), -9),
])
def test_rotations_refused(lib, change, status):
    r = rotary(**change)
    assert lib.pcpa_rotate(params(), chunk(), r, None, 0, 0, rows(), rows(), None, rows(), rows(), None, 0,
                           None) == status
    assert lib.pcpa_chunk_prepare(params(), chunk(), r, rows(), rows(), rows(), rows(), 16, 16, None, None) == status


def test_rotation_arguments(lib):
    def call(positions=None, bits=0, first=0, c=None, q=None, k=None, v=None, qo=None, ko=None, vo=None, striped=0):
        return lib.pcpa_rotate(params(), c or chunk(), rotary(), positions, bits, first, q or rows(), k or rows(), v,
                               qo or rows(), ko or rows(), vo, striped, None)

    assert call(positions=16) == -1            # positions without their width
    assert call(bits=32) == -1                 # and the other way round
    assert call(positions=16, bits=16) == -3
    assert call(positions=20, bits=64) == -6
    assert call(c=chunk(lengths=None)) == -1
    assert call(bits=-1) == -3                 # first_pos: one sequence
    assert call(bits=-1, first=-1, c=chunk(batch=1)) == -3
    assert call(bits=-1, first=2**63 - 3, c=chunk(batch=1)) == -3
    assert call(striped=1) == -3               # striped rows have no lengths
    assert call(bits=-1, c=chunk(batch=1), striped=1) == -3  # 6 rows are no whole stripe
    assert call(v=rows()) == -1 and call(vo=rows()) == -1
    for bad in (rows(data=24), rows(token=508), rows(head=60)):
        assert call(q=bad) == -6 and call(ko=bad) == -6 and call(v=bad, vo=rows()) == -6
    assert call(q=rows(data=None)) == -1


def test_read_arguments(lib):
    def call(il=64, first=0, count=4, table=16, pages=16, k=16, v=16):
        return lib.pcpa_cache_read(params(), il, first, count, table, pages, None, k, v, None)

    assert call(il=0) == -3 and call(first=-1) == -3 and call(count=-1) == -3
    assert call(first=2**63 - 2) == -3
    assert call(table=None) == -1 and call(pages=None) == -1 and call(k=None) == -1 and call(v=None) == -1
    assert call(k=24) == -6 and call(v=8) == -6 and call(pages=8) == -6


# ---- the Python entries ------------------------------------------------------------


@pytest.mark.parametrize("change,message", [
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=80), "rotary_dim"),
    (dict(base=0.0), "base"), (dict(factor=math.inf), "factor"), (dict(pairs="pairs"), "pairs"),
    (dict(scaling="other"), "scaling"), (dict(scaling="by_parts"), "original_len"),
    (dict(scaling="by_parts", original_len=8, slow_turns=4.0, fast_turns=4.0), "slow_turns"),
    (dict(amplitude=math.nan), "amplitude"),
])
def test_embeddings_refused(change, message):
    options = dict(rotary_dim=64)
    options.update(change)
    with pytest.raises(ValueError, match=message):
        QueryKeyRotation(config(), RotaryEmbedding(**options))


def test_norm_eps_refused():
    with pytest.raises(ValueError, match="norm_eps"):
        QueryKeyRotation(config(), RotaryEmbedding(64), norm_eps=-1.0)
    for small in (0.0, 2.0**-127):
        with pytest.raises(ValueError, match="norm_eps"):
            QueryKeyRotation(config(), RotaryEmbedding(64), norm_eps=small)


def test_frequencies():
    plain = RotaryEmbedding(64, base=1.0e4).frequencies()
    assert plain[0] == 1.0 and math.isclose(plain[-1], 1.0e4 ** (-62 / 64))
    assert torch.allclose(RotaryEmbedding(64, scaling="linear", factor=4.0).frequencies(), plain / 4, rtol=1e-15)
    stretched = RotaryEmbedding(64, scaling="base", factor=4.0).frequencies()
    assert stretched[0] == 1.0 and math.isclose(stretched[-1], plain[-1] / 4, rel_tol=1e-12)
    parts = RotaryEmbedding(64, scaling="by_parts", factor=4.0, original_len=2048).frequencies()
    turns = 2048 * plain / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32])
    assert torch.allclose(parts[turns <= 1], plain[turns <= 1] / 4, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert bool(between.any()) and bool(((parts < plain) & (parts > plain / 4))[between].all())


def test_cpu_tensors_are_refused():
    cfg = config(kv=FP8)
    q, k = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    lengths = torch.ones(3, dtype=torch.int32)
    pool = torch.zeros(4, cfg.page_elements).to(torch.float8_e4m3fn)
    table = torch.zeros((3, 1, cfg.max_local_blocks), dtype=torch.int32)
    with pytest.raises(ValueError, match="q must be a bfloat16 GPU tensor"):
        ChunkAttentionKernel(cfg)(q, pool, table, lengths)
    with pytest.raises(ValueError, match="k must be a bfloat16 GPU tensor"):
        ChunkCacheWriter(cfg)(k, k, pool, table, lengths)
    with pytest.raises(ValueError, match="q must be a bfloat16 GPU tensor"):
        QueryKeyRotation(cfg, RotaryEmbedding(64))(q, k, lengths=lengths)
    with pytest.raises(ValueError, match="GPU tensor"):
        CacheReader(cfg)(pool, table[0], num_tokens=3)


def test_token_scales_of_a_bf16_cache_are_refused():
    with pytest.raises(ValueError, match="fp8_e4m3fn"):
        empty_token_scales(config(), "cpu")
    assert empty_token_scales(config(kv=FP8), "cpu", num_pages=3).shape == (3, 2, 2, 64)


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU, to reach the checks behind that one."""

    is_cuda = property(lambda self: True)


def test_rows_that_the_kernels_cannot_address():
    base = torch.zeros(4, 8, 72, dtype=torch.bfloat16)
    ok = base[:, :, :64].as_subclass(_Gpu)
    _rows("q", ok, 8, 64, 4)
    for bad in (base[:, :, 4:68], torch.zeros(4, 8, 68, dtype=torch.bfloat16)[:, :, :64],
                torch.zeros(4, 64, 8, dtype=torch.bfloat16).transpose(1, 2)):
        with pytest.raises(ValueError, match="16 bytes"):
            _rows("q", bad.as_subclass(_Gpu), 8, 64, 4)
    for bad in (ok.float(), ok[:3], ok[:, :7], ok[:, :, :32], ok[0]):
        with pytest.raises(ValueError, match="must be a bfloat16 GPU tensor"):
            _rows("q", bad, 8, 64, 4)


def test_outputs_whose_rows_overlap():
    base = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    _own_places("out", base)
    _own_places("out", base.transpose(0, 1))
    for bad in (base[:1].expand(4, 8, 64), base[:, :1].expand(4, 8, 64), base.as_strided((4, 8, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            _own_places("out", bad)


# ---- chunks of a call ---------------------------------------------------------------


def test_lengths_and_starts():
    from aws_training_study_amd.pcp_attention.rotary import _check_lengths

    cpu = torch.device("cpu")
    lengths = torch.ones(3, dtype=torch.int32)
    assert _check_lengths(lengths, None, 3, 6, cpu) == 3
    assert _check_lengths(lengths, torch.zeros(4, dtype=torch.int32), 3, 7, cpu) == 3
    with pytest.raises(ValueError, match="pass chunk_starts"):
        _check_lengths(lengths, None, 3, 7, cpu)
    for bad in (lengths.long(), lengths[:2], torch.ones(6, dtype=torch.int32)[::2], lengths.view(1, 3)):
        with pytest.raises(ValueError, match="lengths must be"):
            _check_lengths(bad, None, 3, 6, cpu)
    for bad in (lengths, torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="chunk_starts must be"):
            _check_lengths(lengths, bad, 3, 6, cpu)


def test_shared_memory():
    """Which rows of two views share memory, against the addresses themselves."""
    store = torch.zeros(4096, dtype=torch.bfloat16)

    def view(at, n, heads, d, token, head):
        return torch.as_strided(store, (n, heads, d), (token, head, 1), at)

    def addresses(t):
        n, heads, d = t.shape
        return {t.storage_offset() + i * t.stride(0) + h * t.stride(1) + x
                for i in range(n) for h in range(heads) for x in range(d)}

    views = [view(*v) for v in [(0, 4, 2, 8, 64, 8), (16, 4, 2, 8, 64, 8), (8, 4, 2, 8, 64, 8), (48, 4, 3, 8, 64, 8),
                                (56, 4, 1, 8, 64, 8), (256, 4, 2, 8, 64, 8), (0, 1, 2, 8, 64, 8), (16, 1, 4, 8, 0, 8),
                                (1000, 4, 2, 8, 16, 8), (1064, 4, 2, 8, 16, 8), (1024, 4, 2, 8, 16, 8)]]
    for a in views:
        for b in views:
            shared = bool(addresses(a) & addresses(b))
            assert _share_memory(a, b) or not shared
            if a.stride(0) == b.stride(0) and a.shape[0] == b.shape[0]:  # (told apart exactly)
                assert _share_memory(a, b) == shared, (a.storage_offset(), b.storage_offset())
    _check_output("out", views[0], views[0], views[1])
    for own, other in ((views[2], views[1]), (views[0], views[2])):
        with pytest.raises(ValueError, match="out must be its own input"):
            _check_output("out", views[0], own, other)
