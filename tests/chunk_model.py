"""Plain 64-bit models of the serving operators, and caches to try them on.

The caches are built with the layout functions of the host side, one position
at a time, and everything that no token owns holds NaN: the pool's other slots,
their scales, the pages of no table entry.
"""

from __future__ import annotations

import math

import torch

from aws_training_study_amd.pcp_attention import PCPAttentionConfig
from aws_training_study_amd.pcp_attention.layout import owner_and_local_position

FP8, BF16 = "fp8_e4m3fn", "bfloat16"
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2  # relative rounding of a BF16 result


def config(pcp=1, il=64, block=64, bucket=1024, hq=8, hkv=2, d=64, kv=BF16) -> PCPAttentionConfig:
    stride = pcp * il
    bucket = -(-bucket // stride) * stride
    return PCPAttentionConfig(pcp_size=pcp, current_len=stride, max_history_len=bucket, actual_history_len=bucket,
                              block_size=block, interleave_size=il, num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                              backend="hip", kv_dtype=kv).validate()


def rows(gen, *shape):
    """BF16 rows of N(0, 1) values with a factor of their own."""
    factor = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=gen))
    return (torch.randn(*shape, generator=gen) * factor).to(torch.bfloat16)


def quantised(x, scale=None):
    """(codes, scales) of rows: ``scale`` for all, or the row's own over its finite values."""
    x = x.float()
    if scale is None:
        finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros(()))
        scale = (finite.amax(dim=-1) / torch.tensor([448.0])).clamp_min(2.0**-80)
    else:
        scale = torch.full(x.shape[:-1], scale)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


class Cache:
    """Pages of several sequences on the CPU: tables, pool, scales, and what the codes stand for (float64)."""

    def __init__(self, cfg, lengths, seed, *, scales="none", table_dtype=torch.int32, spare=3, tokens=None):
        gen = torch.Generator().manual_seed(seed)
        self.cfg, self.lengths, self.scales_kind = cfg, list(lengths), scales
        self.k_scale, self.v_scale = (0.11, 0.13) if scales == "tensor" else (1.0, 1.0)
        hkv, d, block = cfg.num_kv_heads, cfg.head_dim, cfg.block_size
        places = []
        used = set()
        for b, n in enumerate(self.lengths):
            at = [owner_and_local_position(p, cfg.pcp_size, cfg.interleave_size) for p in range(n)]
            places.append([(r, local // block, local % block) for r, local in at])
            used.update((b, r, blk) for r, blk, _ in places[-1])
        used = sorted(used)
        self.num_pages = len(used) + spare
        order = torch.randperm(self.num_pages, generator=gen)[: len(used)].tolist()
        self.table = torch.full((len(self.lengths), cfg.pcp_size, cfg.max_local_blocks), -1, dtype=table_dtype)
        pages = {}
        for entry, page in zip(used, order):
            self.table[entry] = pages[entry] = page
        self.pool = torch.full((self.num_pages, 2, hkv, block, d), math.nan).to(
            torch.float8_e4m3fn if cfg.kv_dtype == FP8 else torch.bfloat16)
        self.token_scales = None
        if scales == "token":
            self.token_scales = torch.full((self.num_pages, 2, hkv, block), math.nan)
        self.tokens, self.values = [], []
        self.index = []
        for b, n in enumerate(self.lengths):
            k, v = (rows(gen, n, hkv, d), rows(gen, n, hkv, d)) if tokens is None else tokens[b]
            page = torch.tensor([pages[b, r, blk] for r, blk, _ in places[b]], dtype=torch.long)
            slot = torch.tensor([s for _, _, s in places[b]], dtype=torch.long)
            self.index.append((page, slot))
            self.tokens.append((k, v))
            self.values.append(tuple(self._store(which, page, slot, x) for which, x in enumerate((k, v))))

    def _store(self, which, page, slot, x):
        if self.cfg.kv_dtype == BF16:
            self.pool[page, which, :, slot] = x
            return x.double()
        given = (self.k_scale, self.v_scale)[which] if self.scales_kind == "tensor" else None
        if self.scales_kind == "none":
            given = 1.0
        codes, scale = quantised(x, given)
        self.pool.view(torch.uint8)[page, which, :, slot] = codes.view(torch.uint8)
        if self.token_scales is not None:
            self.token_scales[page, which, :, slot] = scale
        return codes.double() * scale.double()[..., None]

    def pages(self):
        return self.pool.reshape(self.num_pages, -1)

    def call(self, device):
        """(pool, table) and the scale options of a call, on the GPU."""
        kw = {}
        if self.scales_kind == "tensor":
            kw.update(k_scale=self.k_scale, v_scale=self.v_scale)
        if self.token_scales is not None:
            kw.update(token_scales=self.token_scales.to(device))
        return self.pages().to(device), self.table.to(device), kw


def starts_of(fresh, first=0):
    out = [first]
    for f in fresh:
        out.append(out[-1] + f)
    return torch.tensor(out, dtype=torch.int32)


def attention(cfg, cache, q, lengths, fresh, first=0, hidden=None):
    """(out, lse, bound of out's error, bound of lse's error) of each of a chunk's rows, float64.

    ``hidden``: per sequence a mask of positions that no row sees.  The bounds:
    P is rounded to BF16 before it meets V (half a step each, against
    sum p |v|), the output once more; scores are sums of D products in 32 bits
    (D roundings of at most 2^-24 of sum |q k|, the scale's and exp2's few), whose
    error moves each p by as much relative to it, above and below the line; sums
    of n terms in 32 bits add n 2^-24.
    """
    group, d = cfg.num_q_heads // cfg.num_kv_heads, cfg.head_dim
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    row = first
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        for i in range(f):
            pos = n - f + i
            count = max(0, min(pos + 1, cache.values[b][0].shape[0]))
            seen = torch.arange(count)
            if hidden is not None:
                seen = seen[~hidden[b][:count]]
            if seen.numel() == 0:
                out[row], lse[row] = 0.0, -math.inf
            else:
                k, v = (x[seen] for x in cache.values[b])
                kr, vr = (x.repeat_interleave(group, dim=1).permute(1, 0, 2) for x in (k, v))
                qr = q[row].double()[:, :, None]
                s = (kr @ qr)[..., 0] * cfg.softmax_scale
                size = (kr.abs() @ qr.abs())[..., 0] * cfg.softmax_scale
                lse[row] = torch.logsumexp(s, dim=1)
                p = torch.exp(s - lse[row][:, None])
                out[row] = (p[:, None] @ vr)[:, 0]
                moved = (d + 8) * 2.0**-24 * size.amax(dim=1) + 2.0**-20 + seen.numel() * 2.0**-24
                spread = (p[:, None] @ vr.abs())[:, 0]
                bound[row] = HALF_STEP * out[row].abs() + (HALF_STEP + 2 * moved[:, None]) * spread * (1 + HALF_STEP)
                lse_bound[row] = moved + 2.0**-22 * lse[row].abs()
            row += 1
    return out, lse, bound, lse_bound
