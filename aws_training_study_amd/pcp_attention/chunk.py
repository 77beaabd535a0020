"""Sequences served chunk by chunk over the paged cache: the steps after a prefill.

The reference's cache holds one prompt's history and ends there
(run_poc.py:221-266).  Here several sequences, each with a block table of its
own over one page pool, take new tokens - one each, or whole prompts: K and V
go into their pages (``ChunkCacheWriter``), the new tokens attend to their
sequence's cache (``ChunkAttentionKernel``), and a cache can be read back
(``CacheReader``).  ``ChunkStep`` chains rotation, write and attention.

A chunk is the new tokens of ``batch`` sequences, packed into ``n`` rows.
``lengths`` (int32 ``[batch]``) are the tokens each cache holds, the new ones
included; sequence b's rows are ``chunk_starts[b] .. chunk_starts[b + 1] - 1``
(int32 ``[batch + 1]``, not decreasing), or ``n / batch`` each without
``chunk_starts``, and row i of them is position ``lengths[b] - n_b + i``.  Both
are GPU tensors read by the kernels, so that a captured graph follows them.
Rows that belong to no sequence (padding behind the last one) are left alone.

Block tables are ``[batch, pcp, max_local_blocks]`` (``[pcp,
max_local_blocks]`` for one sequence), each sequence striped over the config's
logical ranks as ``KVCacheWriter`` stripes it (layout.py:10-16), so a prefill's
cache is served as it is; with ``pcp_size`` 1 it is an ordinary paged cache.
"""

from __future__ import annotations

import ctypes
from dataclasses import replace
from typing import Optional

from .config import PCPAttentionConfig
from .kernel import _KV_DTYPE_CODES, _torch_kv_dtype
from .rotary import (
    QueryKeyRotation,
    RotaryEmbedding,
    _check_lengths,
    _check_output,
    _own_places,
    _pointer,
    _row_view,
    _rows,
)


def empty_token_scales(config: PCPAttentionConfig, device, num_pages: Optional[int] = None):
    """Zeroed scales of an e4m3 pool with one for each token and head: float32
    ``[num_pages, 2, Hkv, block_size]``, K's then V's of each page."""
    import torch

    if config.kv_dtype != "fp8_e4m3fn":
        raise ValueError("token scales go with an fp8_e4m3fn cache")
    pages = config.num_pages if num_pages is None else int(num_pages)
    return torch.zeros((pages, 2, config.num_kv_heads, config.block_size), dtype=torch.float32, device=device)


class _CacheOperator:
    """What the operators over a paged cache share: the configuration, its launch parameters and checks."""

    def __init__(self, config: PCPAttentionConfig):
        from .. import _native

        self.config = replace(config, backend="hip").validate()
        self._native = _native
        self._lib = _native.load_library()
        cfg = self.config
        self._static = dict(
            abi_version=_native.ABI_VERSION, pcp_size=cfg.pcp_size, num_q_heads=cfg.num_q_heads,
            num_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, local_q_len=cfg.local_q_len,
            block_size=cfg.block_size, max_local_blocks=cfg.max_local_blocks, q_dtype=_native.DTYPE_BF16,
            kv_dtype=_KV_DTYPE_CODES[cfg.kv_dtype], out_dtype=_native.DTYPE_BF16, softmax_scale=cfg.softmax_scale)
        status = self._lib.pcpa_check_params(ctypes.byref(self._params(cfg.num_pages, 1.0, 1.0)))
        if status != _native.PCPA_OK:
            raise ValueError(f"configuration rejected by the HIP kernel: {_native.status_string(status)}")
        self._fast = None  # the native call, made by the first one

    def _native_call(self, kind: str, fn):
        self._fast = self._native.fast_calls().make(
            kind, bytes(self._params(self.config.num_pages, 1.0, 1.0)), self.config.kv_dtype == "fp8_e4m3fn",
            self.config.interleave_size, self._native.function_address(fn))
        return self._fast

    def _params(self, num_pages: int, k_scale: float, v_scale: float, table64: bool = False):
        return self._native.PcpaParams(num_pages=num_pages, k_scale=float(k_scale), v_scale=float(v_scale),
                                       flags=self._native.FLAG_TABLE_INT64 if table64 else 0, **self._static)

    def _cache_params(self, kv_pages, block_table, token_scales, k_scale, v_scale, batch: int, device):
        """The launch parameters of a call on this cache, its tensors checked."""
        import torch

        cfg = self.config
        if (kv_pages.ndim != 2 or kv_pages.shape[1] != cfg.page_elements or kv_pages.shape[0] == 0
                or kv_pages.dtype != _torch_kv_dtype(cfg.kv_dtype) or not kv_pages.is_contiguous()
                or kv_pages.device != device):
            raise ValueError(f"kv_pages must be a contiguous {cfg.kv_dtype} [num_pages, {cfg.page_elements}] pool on "
                             f"{device}, got {kv_pages.dtype} {tuple(kv_pages.shape)} on {kv_pages.device}")
        shape = (batch, cfg.pcp_size, cfg.max_local_blocks)
        if (tuple(block_table.shape) not in ((shape, shape[1:]) if batch == 1 else (shape,))
                or block_table.dtype not in (torch.int32, torch.int64) or block_table.device != device
                or not block_table.is_contiguous()):
            raise ValueError(f"block_table must be contiguous int32 or int64 {shape} on {device}, got "
                             f"{block_table.dtype} {tuple(block_table.shape)} on {block_table.device}")
        if token_scales is not None:
            if cfg.kv_dtype != "fp8_e4m3fn":
                raise ValueError("token_scales go with an fp8_e4m3fn cache")
            scales = (kv_pages.shape[0], 2, cfg.num_kv_heads, cfg.block_size)
            if (tuple(token_scales.shape) != scales or token_scales.dtype != torch.float32
                    or token_scales.device != device or not token_scales.is_contiguous()):
                raise ValueError(f"token_scales must be contiguous float32 {scales} on {device}, got "
                                 f"{token_scales.dtype} {tuple(token_scales.shape)} on {token_scales.device}")
            if float(k_scale) != 1.0 or float(v_scale) != 1.0:
                raise ValueError("pass either token_scales or k_scale and v_scale")
        return self._params(kv_pages.shape[0], k_scale, v_scale, block_table.dtype == torch.int64)

    def _chunk(self, num_tokens: int, batch: int, lengths, chunk_starts):
        return self._native.PcpaChunk(self.config.interleave_size, batch, num_tokens, 0, lengths.data_ptr(),
                                      _pointer(chunk_starts))


def _sequences(block_table) -> int:
    return block_table.shape[0] if block_table.ndim == 3 else 1


class ChunkCacheWriter(_CacheOperator):
    """Writes a chunk's K and V into the pages of its sequences.

    ``writer(k, v, kv_pages, block_table, lengths, *, chunk_starts=None,
    k_scale=1.0, v_scale=1.0, token_scales=None)``: ``k``/``v`` BF16 ``[n, Hkv,
    D]`` GPU rows in token order (any strides that are multiples of 8 values).

    An e4m3 pool holds ``x / scale`` rounded to e4m3: with ``token_scales``
    (``empty_token_scales``) each row x of a token and head has the scale
    ``max(max|x| / 448, 2^-80)`` over its finite values, which is written beside
    the pages (values that are not finite become NaN codes); without, the given
    ``k_scale``/``v_scale`` hold for all, as in ``KVCacheWriter``.  A BF16 pool
    holds x.  Rows whose position is negative or beyond the cache, or whose
    table entry is outside ``[0, num_pages)``, are not written; of two rows for
    one place (a page that two sequences name for new tokens) either may stay.
    Asynchronous on the current stream.
    """

    def __call__(self, k, v, kv_pages, block_table, lengths, *, chunk_starts=None, k_scale: float = 1.0,
                 v_scale: float = 1.0, token_scales=None) -> None:
        call = self._fast or self._native_call("chunk_write", self._lib.pcpa_chunk_write)
        status = call(k, v, kv_pages, block_table, lengths, chunk_starts, k_scale, v_scale, token_scales)
        if status is not None:
            self._native.check(status)
            return
        # not the common form
        import torch

        cfg = self.config
        _rows("k", k, cfg.num_kv_heads, cfg.head_dim, None)
        device, n = k.device, k.shape[0]
        _rows("v", v, cfg.num_kv_heads, cfg.head_dim, n, device)
        batch = _check_lengths(lengths, chunk_starts, _sequences(block_table), n, device)
        params = self._cache_params(kv_pages, block_table, token_scales, k_scale, v_scale, batch, device)
        if n == 0:
            return
        chunk = self._chunk(n, batch, lengths, chunk_starts)
        with torch.cuda.device(device):
            status = self._lib.pcpa_chunk_write(
                ctypes.byref(params), ctypes.byref(chunk), _row_view(self._native, k), _row_view(self._native, v),
                block_table.data_ptr(), kv_pages.data_ptr(), _pointer(token_scales),
                torch.cuda.current_stream(device).cuda_stream)
        self._native.check(status)


class CacheReader(_CacheOperator):
    """Reads a range of one sequence's cache back as BF16 K and V.

    ``reader(kv_pages, block_table, *, first_pos=0, num_tokens, k_scale=1.0,
    v_scale=1.0, token_scales=None) -> (k, v)``: positions ``first_pos ..
    first_pos + num_tokens - 1``, ``[Hkv, num_tokens, D]`` each, as
    ``KVCacheWriter`` and ``build_page_pool`` take them (a cache of token scales
    becomes one of per-tensor scales that way).  Codes times their scale, rounded
    once; positions beyond the cache, or whose table entry is outside ``[0,
    num_pages)``, are zeros.  Asynchronous on the current stream.
    """

    def __call__(self, kv_pages, block_table, *, first_pos: int = 0, num_tokens: int, k_scale: float = 1.0,
                 v_scale: float = 1.0, token_scales=None):
        call = self._fast or self._native_call("cache_read", self._lib.pcpa_cache_read)
        result = call(kv_pages, block_table, first_pos, num_tokens, k_scale, v_scale, token_scales)
        if type(result) is int:  # the status of a launch that failed
            self._native.check(result)
        if result is not None:
            return result
        # not the common form
        import torch

        cfg = self.config
        first_pos, num_tokens = int(first_pos), int(num_tokens)
        if not kv_pages.is_cuda:
            raise ValueError("kv_pages must be a GPU tensor")
        if num_tokens < 0 or first_pos < 0 or num_tokens >= 2**31 or first_pos >= 2**62:
            raise ValueError("first_pos and num_tokens must be non-negative, num_tokens below 2^31 and first_pos "
                             "below 2^62")
        device = kv_pages.device
        if _sequences(block_table) != 1:
            raise ValueError(f"block_table must be one sequence's, got {tuple(block_table.shape)}")
        params = self._cache_params(kv_pages, block_table, token_scales, k_scale, v_scale, 1, device)
        k, v = (torch.empty((cfg.num_kv_heads, num_tokens, cfg.head_dim), dtype=torch.bfloat16, device=device)
                for _ in range(2))
        if num_tokens == 0:
            return k, v
        with torch.cuda.device(device):
            status = self._lib.pcpa_cache_read(
                ctypes.byref(params), cfg.interleave_size, first_pos, num_tokens, block_table.data_ptr(),
                kv_pages.data_ptr(), _pointer(token_scales), k.data_ptr(), v.data_ptr(),
                torch.cuda.current_stream(device).cuda_stream)
        self._native.check(status)
        return k, v


class ChunkAttentionKernel(_CacheOperator):
    """Causal attention of a chunk's new tokens over their sequences' caches.

    ``kernel(q, kv_pages, block_table, lengths, *, chunk_starts=None,
    k_scale=1.0, v_scale=1.0, token_scales=None, out=None, return_lse=False,
    workspace=None) -> out``

    * ``q``: contiguous BF16 ``[n, Hq, D]``; the row at position p of a sequence
      sees the keys at positions ``0 .. p`` of its cache, which already holds the
      chunk's own (``ChunkCacheWriter``).
    * ``out``: as ``q``, which it may be; rows of no sequence are left as they
      are.  A row that sees no key (more new tokens than the cache holds, no page)
      is zeros, as is one whose scores are all ``-inf``.
    * ``return_lse``: also the log-sum-exp of each row's scores, float32 ``[n,
      Hq]``, ``-inf`` for a row that sees no key.
    * ``workspace``: uint8 GPU tensor of ``workspace_bytes(n, batch)`` bytes for
      the partial results of long walks, else one that the object keeps per
      (device, stream, thread).

    Both products run on BF16 operands whatever the cache holds: e4m3 codes are
    widened exactly, the scales applied in float32, the probabilities as two BF16
    values or, where there are many rows (over 32 a sequence and KV head on average
    and over about 4000 in all), rounded to one.  Asynchronous on the current stream.
    """

    def __init__(self, config: PCPAttentionConfig):
        super().__init__(config)
        self._workspaces = {}
        self._sizes = {}

    def workspace_bytes(self, num_tokens: int, batch: int, ragged: bool = True) -> int:
        """Bytes of the workspace of a call with this many rows and sequences
        (``ragged``: with ``chunk_starts``)."""
        key = (int(num_tokens), int(batch), bool(ragged))
        size = self._sizes.get(key)
        if size is None:
            # (the size depends on the shapes alone; a non-null address stands for starts)
            chunk = self._native.PcpaChunk(self.config.interleave_size, key[1], key[0], 0, None, 16 if key[2] else None)
            size = self._lib.pcpa_chunk_workspace_bytes(
                ctypes.byref(self._params(self.config.num_pages, 1.0, 1.0)), ctypes.byref(chunk))
            if size < 0:
                self._native.check(int(size))
            if len(self._sizes) >= 256:
                self._sizes.clear()
            size = self._sizes[key] = int(size)
        return size

    def _workspace(self, size: int, device, stream: int):
        """The workspace kept for this thread's calls on (``device``, ``stream``), which
        run in order (another thread's launches may come between a call's two); a
        call that is being captured gets one of its graph's memory, as graphs
        captured on one stream may be replayed on several."""
        import threading

        import torch

        if torch.cuda.is_current_stream_capturing():
            return torch.empty(size, dtype=torch.uint8, device=device)
        key = (device, stream, threading.get_ident())
        ws = self._workspaces.get(key)
        if ws is None or ws.numel() < size:
            if ws is None and len(self._workspaces) >= 16:
                self._workspaces.clear()
            ws = self._workspaces[key] = torch.empty(size, dtype=torch.uint8, device=device)
            if self._fast is not None:
                self._fast.forget()  # workspaces dropped here are dropped there too
        return ws

    def _attention_call(self):
        import weakref

        import torch

        native, me = self._native, weakref.ref(self)  # (the call is ours: no cycle that keeps workspaces)
        self._fast = native.fast_calls().make_attention(
            bytes(self._params(self.config.num_pages, 1.0, 1.0)), self.config.kv_dtype == "fp8_e4m3fn",
            self.config.interleave_size, native.function_address(self._lib.pcpa_chunk_attention),
            native.function_address(self._lib.pcpa_chunk_workspace_bytes),
            lambda size, index, stream: me()._workspace(size, torch.device("cuda", index), stream))
        return self._fast

    def __call__(self, q, kv_pages, block_table, lengths, *, chunk_starts=None, k_scale: float = 1.0,
                 v_scale: float = 1.0, token_scales=None, out=None, return_lse: bool = False, workspace=None):
        call = self._fast or self._attention_call()
        result = call(q, kv_pages, block_table, lengths, chunk_starts, k_scale, v_scale, token_scales, out, return_lse,
                      workspace)
        if type(result) is int:  # the status of a launch that failed
            self._native.check(result)
        if result is not None:
            return result
        # not the common form
        import torch

        cfg = self.config
        _rows("q", q, cfg.num_q_heads, cfg.head_dim, None)
        device, n = q.device, q.shape[0]
        if not q.is_contiguous():
            raise ValueError(f"q must be contiguous, got strides {tuple(q.stride())}")
        batch = _check_lengths(lengths, chunk_starts, _sequences(block_table), n, device)
        params = self._cache_params(kv_pages, block_table, token_scales, k_scale, v_scale, batch, device)
        if out is None:
            out = torch.empty_like(q)
        else:
            _rows("out", out, cfg.num_q_heads, cfg.head_dim, n, device)
            if not out.is_contiguous():
                raise ValueError(f"out must be contiguous, got strides {tuple(out.stride())}")
            _check_output("out", out, q)
        lse = torch.empty((n, cfg.num_q_heads), dtype=torch.float32, device=device) if return_lse else None
        if n > 0:
            size = self.workspace_bytes(n, batch, chunk_starts is not None)
            if workspace is not None:
                if workspace.dtype != torch.uint8 or workspace.device != device or not workspace.is_contiguous():
                    raise ValueError(f"workspace must be a contiguous uint8 tensor on {device}")
            with torch.cuda.device(device):
                stream = torch.cuda.current_stream(device).cuda_stream
                if workspace is None and size > 0:
                    workspace = self._workspace(size, device, stream)
                chunk = self._chunk(n, batch, lengths, chunk_starts)
                status = self._lib.pcpa_chunk_attention(
                    ctypes.byref(params), ctypes.byref(chunk), q.data_ptr(), kv_pages.data_ptr(),
                    _pointer(token_scales), block_table.data_ptr(), out.data_ptr(), _pointer(lse), _pointer(workspace),
                    0 if workspace is None else workspace.numel(), stream)
            self._native.check(status)
        return (out, lse) if return_lse else out

    def graphed(self, q, kv_pages, block_table, lengths, *, chunk_starts=None, warmup: int = 1, **kwargs):
        """This call captured into a HIP graph (``launch.GraphedLaunch``) with an
        output and a workspace of its own; ``replay()`` follows the current contents
        of the same tensors, ``lengths`` and ``chunk_starts`` among them."""
        import torch

        from .launch import GraphedLaunch

        if kwargs.get("out") is None:
            kwargs["out"] = torch.empty_like(q)
        if kwargs.get("workspace") is None:
            kwargs["workspace"] = self.graph_workspace(q, block_table, chunk_starts)
        return GraphedLaunch(lambda: self(q, kv_pages, block_table, lengths, chunk_starts=chunk_starts, **kwargs),
                             warmup=warmup)

    def graph_workspace(self, q, block_table, chunk_starts):
        """A new workspace for a call of these shapes, ``None`` if it needs none."""
        import torch

        size = self.workspace_bytes(q.shape[0], _sequences(block_table), chunk_starts is not None)
        return torch.empty(size, dtype=torch.uint8, device=q.device) if size > 0 else None


class ChunkStep:
    """One layer's step of a chunk: rotation and cache write, then attention.

    ``step(q, k, v, kv_pages, block_table, lengths, *, chunk_starts=None,
    q_weight=None, k_weight=None, k_scale=1.0, v_scale=1.0, token_scales=None,
    out=None, return_lse=False, workspace=None) -> out``: ``q`` ``[n, Hq, D]`` and
    ``k``/``v`` ``[n, Hkv, D]`` as they come out of the projection.  The rotated K
    and V go straight into the pages (one launch, the same results as
    ``QueryKeyRotation`` followed by ``ChunkCacheWriter``), then the rotated Q
    attends (``ChunkAttentionKernel``).
    """

    def __init__(self, config: PCPAttentionConfig, rotary: RotaryEmbedding, *, norm_eps: float = 1e-6):
        self.rotation = QueryKeyRotation(config, rotary, norm_eps=norm_eps)
        self.attention = ChunkAttentionKernel(config)
        self.config = self.attention.config

    def prepare(self, q, k, v, kv_pages, block_table, lengths, *, chunk_starts=None, q_weight=None, k_weight=None,
                k_scale: float = 1.0, v_scale: float = 1.0, token_scales=None, q_out=None):
        """The first launch alone: K and V in their pages, the rotated Q returned."""
        cfg, op, rotation = self.config, self.attention, self.rotation
        turns = rotation._turns.get(getattr(q, "device", None))
        if turns is not None:
            call = rotation._fast.get("chunk_prepare") or rotation._native_call("chunk_prepare",
                                                                                op._lib.pcpa_chunk_prepare)
            result = call(q, k, v, kv_pages, block_table, lengths, chunk_starts, q_weight, k_weight, k_scale, v_scale,
                          token_scales, q_out, turns)
            if type(result) is int:  # the status of a launch that failed
                op._native.check(result)
            if result is not None:
                return result
        # not the common form
        import torch

        native = op._native
        _rows("q", q, cfg.num_q_heads, cfg.head_dim, None)
        device, n = q.device, q.shape[0]
        _rows("k", k, cfg.num_kv_heads, cfg.head_dim, n, device)
        _rows("v", v, cfg.num_kv_heads, cfg.head_dim, n, device)
        batch = _check_lengths(lengths, chunk_starts, _sequences(block_table), n, device)
        params = op._cache_params(kv_pages, block_table, token_scales, k_scale, v_scale, batch, device)
        if q_out is None:
            q_out = torch.empty((n, cfg.num_q_heads, cfg.head_dim), dtype=torch.bfloat16, device=device)
        else:
            _rows("q_out", q_out, cfg.num_q_heads, cfg.head_dim, n, device)
            _own_places("q_out", q_out)
            _check_output("q_out", q_out, q, k, v)
        rotary = self.rotation._rotary_args(device, q_weight, k_weight)
        if n == 0:
            return q_out
        chunk = op._chunk(n, batch, lengths, chunk_starts)
        with torch.cuda.device(device):
            status = op._lib.pcpa_chunk_prepare(
                ctypes.byref(params), ctypes.byref(chunk), ctypes.byref(rotary), _row_view(native, q),
                _row_view(native, k), _row_view(native, v), _row_view(native, q_out), block_table.data_ptr(),
                kv_pages.data_ptr(), _pointer(token_scales), torch.cuda.current_stream(device).cuda_stream)
        native.check(status)
        return q_out

    def __call__(self, q, k, v, kv_pages, block_table, lengths, *, chunk_starts=None, q_weight=None, k_weight=None,
                 k_scale: float = 1.0, v_scale: float = 1.0, token_scales=None, out=None, return_lse: bool = False,
                 workspace=None):
        cache = dict(chunk_starts=chunk_starts, k_scale=k_scale, v_scale=v_scale, token_scales=token_scales)
        turned = self.prepare(q, k, v, kv_pages, block_table, lengths, q_weight=q_weight, k_weight=k_weight, **cache)
        return self.attention(turned, kv_pages, block_table, lengths, out=out, return_lse=return_lse,
                              workspace=workspace, **cache)

    def graphed(self, q, k, v, kv_pages, block_table, lengths, *, chunk_starts=None, warmup: int = 1, **kwargs):
        """Both launches captured into one HIP graph (``launch.GraphedLaunch``), with
        an output and a workspace of the graph's own."""
        import torch

        from .launch import GraphedLaunch

        if kwargs.get("out") is None:
            kwargs["out"] = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if kwargs.get("workspace") is None:
            kwargs["workspace"] = self.attention.graph_workspace(q, block_table, chunk_starts)
        return GraphedLaunch(lambda: self(q, k, v, kv_pages, block_table, lengths, chunk_starts=chunk_starts,
                                          **kwargs), warmup=warmup)
