"""Performance cases of the operators around a paged cache that is served token by token.

Four operators, called one after another once per layer for each chunk of new
tokens (a whole prompt, part of one, or one token of each running sequence):

rotate  norms of Q and K for each head and the position rotation, in one pass
append  new K and V into the pages of their sequences, quantised on the way
        (e4m3 with a scale for each token and head, or for each tensor, or BF16)
attend  causal attention of each sequence's new tokens over its paged cache,
        which holds them already
read    a range of a sequence's cache back as BF16 K and V

A sequence's cache is striped over `pcp` logical ranks as a prefill leaves it
(one rank: an ordinary paged cache).  Q, K and V are N(0, 1) BF16; K and V carry
a factor for each token and head (its logarithm N(0, 0.4^2)), as the rows of real
caches differ in size.

`own` chooses between the framework's kernels and the plain form of the same
calls: elementary torch operations in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import math
import random

import torch

own = False

FP8 = "fp8_e4m3fn"
BF16 = "bfloat16"
SCALE_FLOOR = 2.0 ** -80


def _case(**kw):
    """A case with the common options filled in."""
    case = dict(
        op="attend",       # rotate | append | attend | read
        pcp=1, il=64, block=512, bucket=8192, hq=32, hkv=2, d=256, kv=FP8,
        scales="token",    # e4m3 pools: one scale per token and head | per tensor; "none" for BF16 pools
        table="int32",     # int32 | int64
        # the chunk of new tokens: `batch` sequences of up to `longest` tokens
        # each (the new ones included), drawn from `layout`
        batch=1, longest=8192, new="one",  # one | same | ragged | prompt
        count=1,           # same: the new tokens of each sequence; ragged: about so many
        layout=0,
        lse=False,
        # rotation
        rotary=0, pairs="half", base=10000.0, norm=False, stretch="none", factor=1.0,
        form="chunk",      # chunk: positions from the lengths | positions: given | prefill: striped over the ranks
        first=0,
    )
    case.update(kw)
    return case


def listed():
    return [
        # Q and K of the "full" preset's 4096 current tokens behind a full
        # history, norms and a rotation of a quarter of each head, laid out for
        # the prefill step (striped Q, stacked K and V).
        _case(name="rotate_prefill_64rank", op="rotate", form="prefill", pcp=64, bucket=131072, longest=4096,
              new="prompt", rotary=64, base=1.0e7, norm=True, first=131072),
        # One token of each of 64 running sequences.
        _case(name="rotate_decode_64seq", op="rotate", batch=64, rotary=256, norm=True, layout=1),
        # Packed prompts at explicit positions: interleaved pairs, the
        # frequencies stretched by parts for a longer context, no norms.
        _case(name="rotate_gqa8_positions", op="rotate", form="positions", hq=64, hkv=8, d=128, batch=5, longest=600,
              new="prompt", rotary=128, pairs="interleaved", base=500000.0, stretch="by_parts", factor=8.0, layout=2),
        # One token of each of 64 running sequences into e4m3 pages with a
        # scale for each token and head.
        _case(name="append_decode_64seq", op="append", bucket=2048, batch=64, longest=2048, layout=3),
        # Ragged chunks of nine sequences, some empty.
        _case(name="append_ragged_9seq", op="append", batch=9, longest=4096, new="ragged", count=2000, table="int64",
              layout=11),
        # The whole history of the "full" preset back as BF16, as for a pool
        # of other scales.
        _case(name="read_64rank_fp8", op="read", pcp=64, bucket=131072, longest=131072),
        # An unaligned range of a BF16 cache.
        _case(name="read_16rank_bf16", op="read", pcp=16, longest=7001, first=1003, kv=BF16, scales="none", hq=64, hkv=8,
              d=128, block=256),
        # The smallest calls: four short sequences, one token each, where
        # launches and host time count.
        _case(name="attend_decode_4seq_bf16_d64", pcp=4, il=16, block=128, bucket=2048, hq=8, d=64, kv=BF16,
              scales="none", batch=4, longest=200, layout=5),
        # One token of one conversation over the cache that a prefill of the
        # "full" preset left.
        _case(name="attend_decode_64rank_fp8", pcp=64, bucket=131072 + 4096, longest=131072 + 1001, scales="tensor"),
        # One token of each of 64 sequences of different lengths.
        _case(name="attend_decode_64seq_fp8", batch=64, longest=8192, layout=6),
        # 512 new tokens over a long BF16 cache, GQA with 8 KV heads; the
        # log-sum-exp is wanted by a later merge.
        _case(name="attend_chunk_gqa8_bf16_d128", pcp=16, block=256, bucket=32768, hq=64, hkv=8, d=128, kv=BF16,
              scales="none", longest=32768, new="same", count=512, lse=True),
        # Whole prompts of different lengths, packed.
        _case(name="attend_prompts_fp8", batch=7, longest=4096, new="prompt", table="int64", layout=7),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    """One more case of the listed kinds: any op, striping, head layout, cache type, batch and lengths."""
    op = rng.choice(["rotate", "append", "read", "attend", "attend", "attend", "attend"])
    pcp, il, block = rng.choice([(1, 64, 64), (1, 64, 512), (1, 64, 256), (2, 64, 256), (3, 48, 192), (4, 16, 128),
                                 (5, 32, 64), (16, 64, 512), (64, 64, 512)])
    hq, hkv, d = rng.choice([(32, 2, 256), (32, 2, 256), (16, 4, 256), (8, 2, 64), (64, 8, 128), (28, 4, 128),
                             (24, 8, 64), (6, 6, 128)])
    kv = rng.choice([FP8, FP8, BF16])
    scales = "none" if kv == BF16 else rng.choice(["token", "token", "tensor"])
    stride = pcp * il

    def striped(x):
        return max(1, -(-int(x) // stride)) * stride

    new = rng.choice(["one", "one", "same", "ragged", "prompt"])
    batch = int(_log_uniform(rng, 1, 96))
    longest = int(_log_uniform(rng, 1, 131072 if batch == 1 else 8192))
    count = int(_log_uniform(rng, 1, 512))
    layout = rng.randrange(1 << 30)
    case = _case(op=op, pcp=pcp, il=il, block=block, hq=hq, hkv=hkv, d=d, kv=kv, scales=scales, new=new, batch=batch,
                 longest=longest, count=count, layout=layout, table=rng.choice(["int32", "int64"]),
                 lse=op == "attend" and rng.random() < 0.3)
    if op == "read":
        case.update(new="prompt", batch=1, longest=int(_log_uniform(rng, 1, 131072)))
        case["first"] = rng.randrange(case["longest"]) if rng.random() < 0.5 else 0
    elif op == "rotate":
        case.update(form=rng.choice(["chunk", "positions", "prefill"]), norm=rng.random() < 0.6,
                    rotary=rng.choice([r for r in (16, 32, 64, 128, 256) if r <= d]),
                    pairs=rng.choice(["half", "interleaved"]), base=rng.choice([1.0e4, 5.0e5, 1.0e7]),
                    stretch=rng.choice(["none", "linear", "base", "by_parts"]), factor=rng.choice([2.0, 4.0, 8.0]))
        if case["form"] == "prefill":
            case.update(batch=1, new="prompt", longest=striped(min(case["longest"], 4096)),
                        first=rng.randrange(1 << 20))
        elif case["new"] == "prompt":
            case["longest"] = min(longest, 4096)
    while op != "read" and case["new"] == "prompt" and sum(_lengths(case)[1]) > 8192:
        case["longest"] = case["longest"] // 2 if case["longest"] > 1 else 1
        case["batch"] = max(1, case["batch"] * 3 // 4) if case["longest"] < 64 else case["batch"]
    while op != "read" and case["batch"] * case["count"] > 4096:
        case["count"] = max(1, case["count"] // 2)
    while work(case)["flops"] > 5.0e11 or work(case)["bytes"] > 4.0e8:
        case["count"] = max(1, case["count"] // 2)
        case["longest"] = max(stride if case["form"] == "prefill" else 1, case["longest"] * 3 // 4)
        if case["form"] == "prefill":
            case["longest"] = striped(case["longest"])
        case["first"] = min(case["first"], case["longest"] - 1) if op == "read" else case["first"]
    case["bucket"] = striped(case["longest"])
    return case


# ---- what a case's sizes are ----------------------------------------------------


def _lengths(case):
    """(tokens of each sequence, new tokens of each sequence) of a case's chunk."""
    rng = random.Random(case["layout"])
    batch, longest = case["batch"], case["longest"]
    lengths = [longest] + [rng.randint(max(1, longest // 16), longest) for _ in range(batch - 1)]
    rng.shuffle(lengths)
    if case["new"] == "one":
        fresh = [1] * batch
    elif case["new"] == "same":
        fresh = [case["count"]] * batch
        lengths = [max(n, case["count"]) for n in lengths]
    elif case["new"] == "ragged":
        fresh = [min(n, rng.choice([0, 1, rng.randint(1, 2 * case["count"])])) for n in lengths]
        if not any(fresh):
            fresh[0] = 1
    else:
        fresh = list(lengths)
    return lengths, fresh


def _capacity(case):
    """The bucket of a case's configuration: whole strides that hold its longest sequence."""
    stride = case["pcp"] * case["il"]
    need = max([case["bucket"], *_lengths(case)[0]])
    return -(-need // stride) * stride


def work(case):
    """The bytes and operations of one pass: every input and output once, the products over the keys each row sees."""
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    es = 1 if case["kv"] == FP8 else 2
    scale = 4 if case["scales"] == "token" else 0
    lengths, fresh = _lengths(case)
    n = sum(fresh)
    if case["op"] == "rotate":
        heads = hq + hkv + (hkv if case["form"] == "prefill" else 0)
        # per element: square and sum, the norm's product, two products and a sum
        return {"bytes": 2 * heads * n * d * 2, "flops": 6 * (hq + hkv) * n * d}
    row = hkv * d
    if case["op"] == "append":
        return {"bytes": 2 * n * (row * (2 + es) + hkv * scale), "flops": 4 * n * row}
    if case["op"] == "read":
        n = case["longest"] - case["first"]
        return {"bytes": 2 * n * (row * (2 + es) + hkv * scale), "flops": 2 * n * row}
    seen = sum(f * (length - f) + f * (f + 1) // 2 for length, f in zip(lengths, fresh))
    # a sequence without a new token is not read
    cached = sum(length for length, f in zip(lengths, fresh) if f)
    size = 2 * cached * (row * es + hkv * scale) + 2 * n * hq * d * 2 + (4 * n * hq if case["lse"] else 0)
    return {"bytes": size, "flops": 4 * hq * d * seen}


# ---- inputs ----------------------------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _rows(gen, *shape):
    """BF16 rows of N(0, 1) values, each row with a factor of its own."""
    factor = torch.exp(0.4 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return (torch.randn(*shape, generator=gen, device="cuda") * factor).to(torch.bfloat16)


def _tables(case, gen):
    """([batch, pcp, blocks] pages of the sequences' blocks, -1 where there are no tokens; the pool's pages)."""
    pcp, il, block = case["pcp"], case["il"], case["block"]
    blocks = -(-(_capacity(case) // pcp) // block)
    ranks = torch.arange(pcp).view(1, pcp, 1)
    lengths = torch.tensor(_lengths(case)[0]).view(-1, 1, 1)
    rounds, rest = lengths // (pcp * il), lengths % (pcp * il)
    local = rounds * il + (rest - ranks * il).clamp(0, il)
    used = torch.arange(blocks).view(1, 1, blocks) * block < local
    pages = int(used.sum()) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(gen.initial_seed() + 1))
    table = torch.full(used.shape, -1, dtype=torch.int64)
    table[used] = order[: pages - 3]
    return table.to(device="cuda", dtype=torch.int32 if case["table"] == "int32" else torch.int64), pages


def _places(case, table, positions):
    """(page, slot) of global positions of one sequence, whose table is [pcp, blocks]."""
    pcp, il, block = case["pcp"], case["il"], case["block"]
    chunk = positions // il
    local = (chunk // pcp) * il + positions % il
    return table[chunk % pcp, local // block].long(), local % block


def _quantised(x, scale):
    """(e4m3 codes, float32 scales) of rows x [..., D]: a scale per row, or the given one."""
    x = x.float()
    if scale is None:
        scale = (x.abs().amax(dim=-1) / torch.tensor([448.0], device=x.device)).clamp_min(SCALE_FLOOR)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _bytes(x):
    """Index kernels take the bytes of 8-bit floats."""
    return x.view(torch.uint8) if x.element_size() == 1 else x


def _store(case, pool, scales, which, table, positions, x, tensor_scale):
    """Rows x [n, Hkv, D] of one sequence into its pages."""
    page, slot = _places(case, table, positions)
    slots = pool.view(-1, 2, case["hkv"], case["block"], case["d"])
    if case["kv"] == BF16:
        slots[page, which, :, slot] = x
        return
    given = None
    if case["scales"] == "tensor":
        given = torch.full((1, 1), tensor_scale, device=x.device, dtype=torch.float32)
    codes, scale = _quantised(x, given)
    _bytes(slots)[page, which, :, slot] = _bytes(codes)
    if case["scales"] == "token":
        scales[page, which, :, slot] = scale


def _pool(case, pages):
    pool = torch.zeros((pages, 2 * case["hkv"] * case["block"] * case["d"]), device="cuda",
                       dtype=torch.float8_e4m3fn if case["kv"] == FP8 else torch.bfloat16)
    scales = None
    if case["scales"] == "token":
        scales = torch.zeros((pages, 2, case["hkv"], case["block"]), device="cuda")
    return pool, scales


def _draws(case, seed):
    """Everything that is drawn from the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths, fresh = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    n = sum(fresh)
    got = dict(gen=gen, lengths=lengths, fresh=fresh)
    if case["op"] == "rotate":
        # one projection's output, whose columns are the heads of Q, K and V
        got["qkv"] = _rows(gen, n, hq + 2 * hkv, d)
        if case["norm"]:
            got["q_weight"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(torch.bfloat16)
            got["k_weight"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(torch.bfloat16)
        if case["form"] == "positions":
            start = torch.randint(0, 1 << 20, (len(fresh),), generator=torch.Generator().manual_seed(seed)).tolist()
            got["positions"] = torch.cat([torch.arange(s, s + f) for s, f in zip(start, fresh)]).cuda()
    elif case["op"] == "append":
        got.update(k=_rows(gen, n, hkv, d), v=_rows(gen, n, hkv, d))
    else:
        got["history"] = [(_rows(gen, length, hkv, d), _rows(gen, length, hkv, d)) for length in lengths]
        if case["op"] == "attend":
            got["q"] = _normal(gen, n, hq, d)
    return got


def _tensor_scales(case):
    return (0.1, 0.11) if case["scales"] == "tensor" else (1.0, 1.0)


def _config(case):
    from aws_training_study_amd.pcp_attention import PCPAttentionConfig

    stride = case["pcp"] * case["il"]
    current = case["longest"] if case["op"] == "rotate" and case["form"] == "prefill" else stride
    bucket = _capacity(case)
    return PCPAttentionConfig(
        pcp_size=case["pcp"], current_len=current, max_history_len=bucket, actual_history_len=bucket,
        block_size=case["block"], interleave_size=case["il"], num_q_heads=case["hq"], num_kv_heads=case["hkv"],
        head_dim=case["d"], backend="hip", kv_dtype=case["kv"]).validate()


def _rotary(case):
    from aws_training_study_amd.pcp_attention import RotaryEmbedding

    stretch = {} if case["stretch"] == "none" else dict(scaling=case["stretch"], factor=case["factor"])
    if case["stretch"] == "by_parts":
        stretch.update(original_len=8192, amplitude=_amplitude(case))
    return RotaryEmbedding(rotary_dim=case["rotary"], base=case["base"], pairs=case["pairs"], **stretch)


def prepare(case, seed):
    drawn = _draws(case, seed)
    lengths, fresh = drawn["lengths"], drawn["fresh"]
    starts = [0]
    for f in fresh:
        starts.append(starts[-1] + f)
    state = dict(
        case=case, lens=lengths, fresh=fresh, starts=starts,
        lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
        # sequences with the same number of new tokens need no starts
        chunk_starts=None if len(set(fresh)) == 1 else torch.tensor(starts, dtype=torch.int32, device="cuda"))
    for name in ("positions", "q_weight", "k_weight", "k", "v", "q"):
        state[name] = drawn.get(name)
    if case["op"] == "rotate":
        hq, hkv = case["hq"], case["hkv"]
        qkv = drawn["qkv"]
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
        if own:
            from aws_training_study_amd.pcp_attention import QueryKeyRotation

            state["kernel"] = QueryKeyRotation(_config(case), _rotary(case), norm_eps=1e-6)
        return state
    table, pages = _tables(case, drawn["gen"])
    pool, scales = _pool(case, pages)
    k_scale, v_scale = _tensor_scales(case)
    for b, (k, v) in enumerate(drawn.get("history", ())):
        positions = torch.arange(lengths[b], device="cuda")
        _store(case, pool, scales, 0, table[b], positions, k, k_scale)
        _store(case, pool, scales, 1, table[b], positions, v, v_scale)
    state.update(table=table, pool=pool, scales=scales, k_scale=k_scale, v_scale=v_scale)
    if own:
        from aws_training_study_amd.pcp_attention import CacheReader, ChunkAttentionKernel, ChunkCacheWriter

        kinds = {"append": ChunkCacheWriter, "attend": ChunkAttentionKernel, "read": CacheReader}
        state["kernel"] = kinds[case["op"]](_config(case))
    return state


# ---- one pass ----------------------------------------------------------------------


def _amplitude(case):
    return 1.0 + 0.1 * math.log(case["factor"]) if case["stretch"] == "by_parts" else 1.0


def _frequencies(case):
    """Radians per position of every rotated pair, in 64 bits."""
    dim, base, factor = case["rotary"], case["base"], case["factor"]
    pair = torch.arange(dim // 2, dtype=torch.float64)
    if case["stretch"] == "base":
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-2.0 * pair / dim)
    if case["stretch"] == "linear":
        freq = freq / factor
    elif case["stretch"] == "by_parts":
        # pairs that turn more than 32 times over 8192 positions stay, those
        # that turn less than once are stretched, a ramp between
        keep = ((8192 * freq / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)
    return freq


def _plain_positions(state):
    case = state["case"]
    if case["form"] == "positions":
        return state["positions"]
    if case["form"] == "prefill":
        return case["first"] + torch.arange(case["longest"], device="cuda")
    at = [torch.arange(n - f, n, device="cuda") for n, f in zip(state["lens"], state["fresh"])]
    return torch.cat(at)


def _plain_rotate(x, weight, cos, sin, case):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-6) * weight.float()
    dim = case["rotary"]
    turned, rest = x[..., :dim], x[..., dim:]
    if case["pairs"] == "half":
        a, b = turned[..., : dim // 2], turned[..., dim // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    return torch.cat((turned, rest), dim=-1).to(torch.bfloat16)


def _stripe(x, case):
    """[n, H, D] in token order as [pcp, H, n / pcp, D], each rank's chunks."""
    n, heads, d = x.shape
    pcp, il = case["pcp"], case["il"]
    return x.view(n // (pcp * il), pcp, il, heads, d).permute(1, 3, 0, 2, 4).reshape(pcp, heads, n // pcp, d)


def _run_rotate(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    weights = {"q_weight": state["q_weight"], "k_weight": state["k_weight"]}
    if own:
        if case["form"] == "prefill":
            return state["kernel"].prefill(q, k, v, first_pos=case["first"], **weights)
        if case["form"] == "positions":
            return state["kernel"](q, k, positions=state["positions"], **weights)
        return state["kernel"](q, k, lengths=state["lengths"], chunk_starts=state["chunk_starts"], **weights)
    # angles of far positions in 64 bits, their cosines and sines in 32
    angle = _plain_positions(state).double()[:, None] * _frequencies(case).cuda()
    amplitude = _amplitude(case)
    cos, sin = ((f(angle) * amplitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    q = _plain_rotate(q, weights["q_weight"], cos, sin, case)
    k = _plain_rotate(k, weights["k_weight"], cos, sin, case)
    if case["form"] == "prefill":
        return _stripe(q, case), torch.stack((k.transpose(0, 1), v.transpose(0, 1)))
    return q, k


def _run_append(state):
    case, pool, scales = state["case"], state["pool"], state["scales"]
    if own:
        state["kernel"](state["k"], state["v"], pool, state["table"], state["lengths"],
                        chunk_starts=state["chunk_starts"], k_scale=state["k_scale"], v_scale=state["v_scale"],
                        token_scales=scales)
    else:
        for b, (n, f) in enumerate(zip(state["lens"], state["fresh"])):
            if not f:
                continue
            positions = torch.arange(n - f, n, device="cuda")
            rows = slice(state["starts"][b], state["starts"][b + 1])
            _store(case, pool, scales, 0, state["table"][b], positions, state["k"][rows], state["k_scale"])
            _store(case, pool, scales, 1, state["table"][b], positions, state["v"][rows], state["v_scale"])
    return {"pool": pool} if scales is None else {"pool": pool, "scales": scales}


def _plain_cache(state, b, positions):
    """K and V [n, Hkv, D] float32 of one sequence's positions, as its pages hold them."""
    case = state["case"]
    page, slot = _places(case, state["table"][b], positions)
    slots = state["pool"].view(-1, 2, case["hkv"], case["block"], case["d"])
    got = []
    for which, scale in ((0, state["k_scale"]), (1, state["v_scale"])):
        x = _bytes(slots)[page, which, :, slot].view(slots.dtype).float()
        if state["scales"] is not None:
            x = x * state["scales"][page, which, :, slot][..., None]
        got.append(x * scale)
    return got


def _run_read(state):
    case = state["case"]
    first, count = case["first"], case["longest"] - case["first"]
    if own:
        return state["kernel"](state["pool"], state["table"][0], first_pos=first, num_tokens=count,
                               k_scale=state["k_scale"], v_scale=state["v_scale"], token_scales=state["scales"])
    k, v = _plain_cache(state, 0, torch.arange(first, first + count, device="cuda"))
    return k.to(torch.bfloat16).transpose(0, 1).contiguous(), v.to(torch.bfloat16).transpose(0, 1).contiguous()


def _run_attend(state):
    case = state["case"]
    q = state["q"]
    if own:
        return state["kernel"](q, state["pool"], state["table"], state["lengths"], chunk_starts=state["chunk_starts"],
                               k_scale=state["k_scale"], v_scale=state["v_scale"], token_scales=state["scales"],
                               return_lse=case["lse"])
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    group = hq // hkv
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], device="cuda")
    for b, (n, f) in enumerate(zip(state["lens"], state["fresh"])):
        if not f:
            continue
        k, v = _plain_cache(state, b, torch.arange(n, device="cuda"))
        most = max(1, (1 << 28) // (n * group))  # rows of scores at a time
        for i in range(0, f, most):
            j = min(f, i + most)
            rows = slice(state["starts"][b] + i, state["starts"][b] + j)
            sees = torch.arange(n - f + i, n - f + j, device="cuda")
            hidden = (torch.arange(n, device="cuda")[None, :] > sees[:, None]).repeat_interleave(group, dim=0)
            for g in range(hkv):
                heads = slice(g * group, (g + 1) * group)
                s = q[rows, heads].float().reshape(-1, d) @ k[:, g].t() * (1.0 / math.sqrt(d))
                s.masked_fill_(hidden, -math.inf)
                top = s.amax(dim=1, keepdim=True)
                p = torch.exp(s - top)
                total = p.sum(dim=1, keepdim=True)
                out[rows, heads] = ((p @ v[:, g]) / total).view(j - i, group, d).to(torch.bfloat16)
                lse[rows, heads] = (top + torch.log(total)).view(j - i, group)
    return (out, lse) if case["lse"] else out


def run(state):
    return {"rotate": _run_rotate, "append": _run_append, "read": _run_read, "attend": _run_attend}[
        state["case"]["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------------


def _e4m3(x):
    """The nearest e4m3 value of finite float64 values below 464, ties to the even code."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -9))).clamp_min(-6)
    # log2 may round up to the next whole number just below it
    exponent = torch.where(torch.exp2(exponent) > x.abs().clamp_min(2.0 ** -6), exponent - 1, exponent)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _stored(x, case, which):
    """(what the cache's codes stand for, the scales) of BF16 rows, in 64 bits."""
    x = x.double()
    if case["kv"] == BF16:
        return x, None
    if case["scales"] == "tensor":
        # a cache of 8 bits with a given scale holds 32-bit quotients
        scale = torch.tensor(_tensor_scales(case)[which], device=x.device, dtype=torch.float32).double()
        return _e4m3((x / scale).float().double()) * scale, None
    scale = (x.abs().amax(dim=-1) / 448.0).clamp_min(SCALE_FLOOR)
    held = scale.float().double()  # the scale that is kept, which the codes are relative to
    return _e4m3((x / held[..., None]).float().double()) * held[..., None], scale


def _exact_rotate(case, drawn):
    hq, hkv = case["hq"], case["hkv"]
    lengths, fresh = drawn["lengths"], drawn["fresh"]
    if case["form"] == "positions":
        at = drawn["positions"].double()
    elif case["form"] == "prefill":
        at = torch.arange(case["first"], case["first"] + case["longest"], device="cuda").double()
    else:
        at = torch.tensor([n - f + i for n, f in zip(lengths, fresh) for i in range(f)], device="cuda").double()
    x = drawn["qkv"][:, : hq + hkv].double()
    if case["norm"]:
        weight = torch.cat((drawn["q_weight"].double().expand(hq, -1), drawn["k_weight"].double().expand(hkv, -1)))
        x = x / torch.sqrt((x ** 2).sum(dim=2, keepdim=True) / case["d"] + 1e-6) * weight
    dim = case["rotary"]
    index = torch.arange(dim // 2, device="cuda")
    first, second = (index, index + dim // 2) if case["pairs"] == "half" else (2 * index, 2 * index + 1)
    turn = torch.polar(torch.full((), _amplitude(case), device="cuda", dtype=torch.float64),
                       at[:, None] * _frequencies(case).cuda())[:, None]
    z = torch.complex(x[:, :, first], x[:, :, second]) * turn
    x = x.clone()
    x[:, :, first], x[:, :, second] = z.real, z.imag
    q, k = x[:, :hq], x[:, hq:]
    if case["form"] != "prefill":
        return q, k
    n, pcp, il = case["longest"], case["pcp"], case["il"]
    token = torch.arange(n, device="cuda")
    rank, local = (token // il) % pcp, token // (il * pcp) * il + token % il
    stacked = torch.empty(pcp, hq, n // pcp, case["d"], device="cuda", dtype=torch.float64)
    stacked[rank, :, local] = q
    v = drawn["qkv"][:, hq + hkv:].double()
    return stacked, torch.stack((k.transpose(0, 1), v.transpose(0, 1)))


def _exact_attend(case, drawn):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q = drawn["q"].double().view(-1, hkv, hq // hkv, d)
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:3], device="cuda", dtype=torch.float64)
    row = 0
    for (k, v), n, f in zip(drawn["history"], drawn["lengths"], drawn["fresh"]):
        if not f:
            continue
        k, v = _stored(k, case, 0)[0], _stored(v, case, 1)[0]
        most = max(1, (1 << 27) // (n * (hq // hkv)))
        for i in range(0, f, most):
            c = min(most, f - i)
            last = n - f + i + c  # later keys are seen by none of these rows
            later = torch.ones(c, last, device="cuda", dtype=torch.bool).triu(diagonal=last - c + 1)
            for g in range(hkv):
                s = torch.matmul(q[row + i:row + i + c, g].transpose(0, 1).contiguous(), k[:last, g].t().contiguous())
                s = (s / math.sqrt(d)).masked_fill(later, -math.inf)
                total = torch.logsumexp(s, dim=-1)
                lse[row + i:row + i + c, g] = total.transpose(0, 1)
                p = s.sub_(total[..., None]).exp_()
                out[row + i:row + i + c, g] = torch.matmul(p, v[:last, g].contiguous()).transpose(0, 1)
        row += f
    out = out.view(-1, hq, d)
    return (out, lse.view(-1, hq)) if case["lse"] else out


def exact(case, seed):
    drawn = _draws(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(case, drawn)
    if case["op"] == "attend":
        return _exact_attend(case, drawn)
    if case["op"] == "read":
        (k, v), first = drawn["history"][0], case["first"]
        return tuple(_stored(x[first:], case, which)[0].transpose(0, 1) for which, x in enumerate((k, v)))
    # append: the pages' values are the codes', relative to the scales beside them
    table, pages = _tables(case, drawn["gen"])
    shape = (pages, 2, case["hkv"], case["block"])
    pool = torch.zeros(*shape, case["d"], device="cuda", dtype=torch.float64)
    scales = torch.zeros(shape, device="cuda", dtype=torch.float64)
    row = 0
    for b, (n, f) in enumerate(zip(drawn["lengths"], drawn["fresh"])):
        for which, x in enumerate((drawn["k"][row:row + f], drawn["v"][row:row + f])):
            if not f:
                continue
            page, slot = _places(case, table[b], torch.arange(n - f, n, device="cuda"))
            value, scale = _stored(x, case, which)
            if case["scales"] == "token":
                value = value / scale.float().double()[..., None]
                scales[page, which, :, slot] = scale
            elif case["scales"] == "tensor":
                value = value / torch.tensor(_tensor_scales(case)[which], dtype=torch.float32).double().item()
            pool[page, which, :, slot] = value
        row += f
    pool = pool.view(pages, -1)
    return {"pool": pool} if case["scales"] != "token" else {"pool": pool, "scales": scales}
