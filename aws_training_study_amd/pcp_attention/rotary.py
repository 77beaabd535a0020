"""Norms of Q and K for each head and the rotation by position: the step before the cache.

The reference takes Q and K as they come (run_poc.py:81-104 draws them); a
model's Q and K come out of a projection in token order, are normed over each
head and rotated by their position first.  ``QueryKeyRotation`` does both in
one pass on the GPU, and its ``prefill`` form lays Q out striped over the ranks
(layout.py:34-51) and stacks K and V, as ``PrefillAttention`` takes them.
``RotaryEmbedding`` holds the frequencies.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, replace
from typing import Optional

from .config import PCPAttentionConfig
from .kernel import _KV_DTYPE_CODES

PAIR_LAYOUTS = ("half", "interleaved")
ROTARY_SCALINGS = ("none", "linear", "base", "by_parts")


@dataclass(frozen=True)
class RotaryEmbedding:
    """Which values of a head turn with the position, and how fast.

    The first ``rotary_dim`` values of a head (a multiple of 16) form pairs
    ``i = 0 .. R / 2 - 1`` (R = ``rotary_dim``): values ``(i, i + R / 2)`` in the
    ``"half"`` layout, ``(2 i, 2 i + 1)`` in the ``"interleaved"`` one.  Pair i
    turns by ``f_i = base^(-2 i / R)`` radians per position; the other values
    stay.  For contexts longer than the model was trained on (``scaling``):

    ``"linear"``    ``f_i / factor``: positions are interpolated.
    ``"base"``      ``base * factor^(R / (R - 2))`` instead of ``base``: the
                    slowest pair turns ``factor`` times slower, the fastest as
                    before.
    ``"by_parts"``  pairs that turn at least ``fast_turns`` times over
                    ``original_len`` positions keep ``f_i``, those that turn at
                    most ``slow_turns`` times take ``f_i / factor``, a linear
                    ramp between.

    ``amplitude`` multiplies the rotated values.
    """

    rotary_dim: int
    base: float = 10000.0
    pairs: str = "half"
    scaling: str = "none"
    factor: float = 1.0
    original_len: int = 0
    slow_turns: float = 1.0
    fast_turns: float = 32.0
    amplitude: float = 1.0

    def validate(self, head_dim: int) -> "RotaryEmbedding":
        if self.pairs not in PAIR_LAYOUTS:
            raise ValueError(f"pairs must be one of {PAIR_LAYOUTS}, got {self.pairs!r}")
        if self.scaling not in ROTARY_SCALINGS:
            raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}, got {self.scaling!r}")
        if not 0 < self.rotary_dim <= head_dim or self.rotary_dim % 16:
            raise ValueError(f"rotary_dim must be a multiple of 16 in [16, {head_dim}], got {self.rotary_dim}")
        for name in ("base", "factor"):
            value = getattr(self, name)
            if not (math.isfinite(value) and value > 0):
                raise ValueError(f"{name} must be finite and positive, got {value}")
        if not math.isfinite(self.amplitude):
            raise ValueError(f"amplitude must be finite, got {self.amplitude}")
        if self.scaling == "by_parts":
            if self.original_len <= 0:
                raise ValueError(f"original_len must be positive for scaling 'by_parts', got {self.original_len}")
            if not 0 <= self.slow_turns < self.fast_turns < math.inf:
                raise ValueError("slow_turns must be non-negative and below fast_turns, got "
                                 f"{self.slow_turns} and {self.fast_turns}")
        return self

    def frequencies(self):
        """Radians per position of every pair, float64 ``[rotary_dim / 2]`` on the CPU."""
        import torch

        dim, base = self.rotary_dim, self.base
        if self.scaling == "base":
            base = base * self.factor ** (dim / (dim - 2))
        freq = base ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
        if self.scaling == "linear":
            freq = freq / self.factor
        elif self.scaling == "by_parts":
            turns = self.original_len * freq / (2 * math.pi)
            keep = ((turns - self.slow_turns) / (self.fast_turns - self.slow_turns)).clamp(0, 1)
            freq = freq * (keep + (1 - keep) / self.factor)
        return freq


# Revolutions per position of every pair, for each embedding and device: kept for
# good, as kernels on any stream and graphs of the caller's own may read them after
# the object that made them is gone.
_TURNS = {}


def _rows(name: str, t, heads: int, head_dim: int, n: Optional[int], device=None) -> None:
    """``ValueError`` unless ``t`` is ``[n, heads, head_dim]`` BF16 GPU rows the kernels can address."""
    import torch

    if (t.ndim != 3 or t.shape[1] != heads or t.shape[2] != head_dim or (n is not None and t.shape[0] != n)
            or t.dtype != torch.bfloat16 or not t.is_cuda or (device is not None and t.device != device)):
        raise ValueError(f"{name} must be a bfloat16 GPU tensor [{'n' if n is None else n}, {heads}, {head_dim}]"
                         f"{'' if device is None else f' on {device}'}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.numel() and (t.stride(2) != 1 or (t.shape[0] > 1 and t.stride(0) % 8) or (heads > 1 and t.stride(1) % 8)
                      or t.data_ptr() % 16):
        raise ValueError(f"{name}'s heads must be contiguous and start at multiples of 16 bytes, got strides "
                         f"{tuple(t.stride())}")


def _row_view(native, t):
    # (a stride that is never taken may be anything)
    return native.PcpaRows(t.data_ptr(), t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0)


def _own_places(name: str, t) -> None:
    """``ValueError`` if two rows of an output share memory (an expanded or overlapping view)."""
    if t.numel() == 0:
        return
    # sorted by stride, each dimension steps over the whole extent of the ones below
    extent = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s > 1), key=lambda x: x[1]):
        if stride < extent:
            raise ValueError(f"{name}'s rows overlap in memory (strides {tuple(t.stride())})")
        extent = stride * (size - 1) + extent


def _share_memory(a, b) -> bool:
    """Whether rows of ``a`` and ``b`` ``[n, heads, D]`` have memory in common; views of one token stride
    (parts of one projection's output) are told apart by their places in a token."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    size = a.element_size()
    (at_a, one_a), (at_b, one_b) = ((t.data_ptr() // size, (t.shape[1] - 1) * t.stride(1) + t.shape[2]) for t in (a, b))
    n = a.shape[0]
    if at_a >= at_b + (n - 1) * b.stride(0) + one_b or at_b >= at_a + (n - 1) * a.stride(0) + one_a:
        return False
    step = a.stride(0)
    if n > 1 and step == b.stride(0) and step > 0:
        apart = (at_b - at_a) % step
        return apart < one_a or apart + one_b > step
    return True


def _check_output(name: str, out, own, *others) -> None:
    """``ValueError`` unless ``out`` is its own input ``own`` or shares no memory with any."""
    same = out.data_ptr() == own.data_ptr() and all(
        s == t for n, s, t in zip(own.shape, out.stride(), own.stride()) if n > 1)
    if (not same and _share_memory(out, own)) or any(_share_memory(out, t) for t in others):
        raise ValueError(f"{name} must be its own input or share no memory with any")


def _check_lengths(lengths, chunk_starts, batch: Optional[int], num_tokens: int, device) -> int:
    """The chunk's number of sequences, its lengths and starts checked."""
    import torch

    if (lengths.ndim != 1 or lengths.dtype != torch.int32 or lengths.device != device or not lengths.is_contiguous()
            or lengths.shape[0] == 0 or (batch is not None and lengths.shape[0] != batch)):
        raise ValueError(f"lengths must be contiguous int32 [{'batch' if batch is None else batch}] on {device}, got "
                         f"{lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
    batch = lengths.shape[0]
    if chunk_starts is None:
        if num_tokens % batch:
            raise ValueError(f"{num_tokens} rows do not divide evenly over {batch} sequences: pass chunk_starts")
    elif (tuple(chunk_starts.shape) != (batch + 1,) or chunk_starts.dtype != torch.int32
          or chunk_starts.device != device or not chunk_starts.is_contiguous()):
        raise ValueError(f"chunk_starts must be contiguous int32 [{batch + 1}] on {device}, got "
                         f"{chunk_starts.dtype} {tuple(chunk_starts.shape)} on {chunk_starts.device}")
    return batch


def _pointer(t):
    return None if t is None else t.data_ptr()


class QueryKeyRotation:
    """Norms and rotation of Q and K in one pass.

    ``rotation(q, k, *, positions=None, lengths=None, chunk_starts=None,
    q_weight=None, k_weight=None, q_out=None, k_out=None) -> (q_out, k_out)``

    * ``q`` ``[n, Hq, D]``, ``k`` ``[n, Hkv, D]``: BF16 GPU rows in token order,
      of any token and head strides that are multiples of 8 values (views of one
      projection's output).
    * positions, one of: ``positions`` (int32 or int64 ``[n]``), or the chunk's
      own (``lengths``, and ``chunk_starts`` for sequences of different numbers
      of rows: ``ChunkAttentionKernel``), where rows of no sequence are left.
    * ``q_weight``/``k_weight`` ``[D]`` (both BF16 or both float32, either may be
      absent): rows are divided by the root of their mean square plus
      ``norm_eps`` and multiplied by the weight before they turn.
    * ``q_out``/``k_out``: as ``q``/``k``, which they may be (in place); else they
      share no memory with inputs or each other.

    ``prefill(q, k, v, *, first_pos, q_weight=None, k_weight=None) -> (q_stacked,
    kv_current)``: the ``current_len`` tokens at positions ``first_pos ..`` laid
    out for ``PrefillAttention``: Q ``[pcp, Hq, local_q, D]`` and K and V ``[2,
    Hkv, current_len, D]`` (whose halves ``KVCacheWriter`` takes).

    Angles are formed in 64 bits and reduced to a turn (off by less than 2^-22 of
    one for positions below 2^31), the rest is computed in float32 and rounded
    once.  Asynchronous on the current torch stream; an embedding's first call on a
    device copies its frequencies there, which no capture can hold.
    """

    def __init__(self, config: PCPAttentionConfig, rotary: RotaryEmbedding, *, norm_eps: float = 1e-6):
        from .. import _native

        self.config = replace(config, backend="hip").validate()
        self.rotary = rotary.validate(self.config.head_dim)
        self.norm_eps = float(norm_eps)
        if not (math.isfinite(self.norm_eps) and self.norm_eps >= 2.0**-126):
            raise ValueError(f"norm_eps must be finite and at least 2^-126, got {norm_eps}")
        self._native = _native
        self._lib = _native.load_library()
        cfg = self.config
        self._params = _native.PcpaParams(
            abi_version=_native.ABI_VERSION, pcp_size=cfg.pcp_size, num_q_heads=cfg.num_q_heads,
            num_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, local_q_len=cfg.local_q_len,
            block_size=cfg.block_size, max_local_blocks=cfg.max_local_blocks, num_pages=cfg.num_pages,
            q_dtype=_native.DTYPE_BF16, kv_dtype=_KV_DTYPE_CODES[cfg.kv_dtype], out_dtype=_native.DTYPE_BF16,
            softmax_scale=cfg.softmax_scale, k_scale=1.0, v_scale=1.0, flags=0)
        self._turns = {}  # per device: revolutions per position of every pair
        self._fast = {}   # the native calls, made by the first ones

    def _native_call(self, kind: str, fn):
        native, rotary = self._native, self.rotary
        static = native.PcpaRotary(rotary.rotary_dim, int(rotary.pairs == "interleaved"), native.DTYPE_BF16,
                                   rotary.amplitude, self.norm_eps, None, None, None)
        call = self._fast[kind] = native.fast_calls().make_rotation(
            kind, bytes(self._params), self.config.kv_dtype == "fp8_e4m3fn", self.config.interleave_size,
            native.function_address(fn), bytes(static))
        return call

    def turns(self, device):
        """Revolutions per position of every pair, float64 on ``device`` (made once per embedding and device)."""
        import torch

        got = self._turns.get(device)
        if got is None:
            got = _TURNS.get((self.rotary, device))
            if got is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("an embedding's first call on a device copies its frequencies there: make one "
                                       "before a capture")
                got = _TURNS.setdefault((self.rotary, device), (self.rotary.frequencies() / (2 * math.pi)).to(device))
            self._turns[device] = got
        return got

    def _rotary_args(self, device, q_weight, k_weight):
        import torch

        dtype = torch.bfloat16
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is None:
                continue
            if (tuple(w.shape) != (self.config.head_dim,) or w.dtype not in (torch.bfloat16, torch.float32)
                    or w.device != device or not w.is_contiguous()):
                raise ValueError(f"{name} must be contiguous bfloat16 or float32 [{self.config.head_dim}] on {device}, "
                                 f"got {w.dtype} {tuple(w.shape)} on {w.device}")
            if w.data_ptr() % (4 * w.element_size()):
                raise ValueError(f"{name} must start at a multiple of {4 * w.element_size()} bytes")
            dtype = w.dtype
        if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
            raise ValueError(f"q_weight and k_weight must share one dtype, got {q_weight.dtype} and {k_weight.dtype}")
        native = self._native
        return native.PcpaRotary(
            self.rotary.rotary_dim, int(self.rotary.pairs == "interleaved"),
            native.DTYPE_FP32 if dtype == torch.float32 else native.DTYPE_BF16, self.rotary.amplitude, self.norm_eps,
            self.turns(device).data_ptr(), _pointer(q_weight), _pointer(k_weight))

    def __call__(self, q, k, *, positions=None, lengths=None, chunk_starts=None, q_weight=None, k_weight=None,
                 q_out=None, k_out=None):
        turns = self._turns.get(getattr(q, "device", None))
        if turns is not None:
            call = self._fast.get("rotate") or self._native_call("rotate", self._lib.pcpa_rotate)
            result = call(q, k, positions, lengths, chunk_starts, q_weight, k_weight, q_out, k_out, turns)
            if type(result) is int:  # the status of a launch that failed
                self._native.check(result)
            if result is not None:
                return result
        # not the common form
        import torch

        cfg, native = self.config, self._native
        _rows("q", q, cfg.num_q_heads, cfg.head_dim, None)
        device, n = q.device, q.shape[0]
        _rows("k", k, cfg.num_kv_heads, cfg.head_dim, n, device)
        if (positions is None) == (lengths is None):
            raise ValueError("pass either positions or lengths")
        batch, bits = 1, 0
        if positions is None:
            batch = _check_lengths(lengths, chunk_starts, None, n, device)
        else:
            if chunk_starts is not None:
                raise ValueError("chunk_starts goes with lengths")
            if (tuple(positions.shape) != (n,) or positions.dtype not in (torch.int32, torch.int64)
                    or positions.device != device or not positions.is_contiguous()):
                raise ValueError(f"positions must be contiguous int32 or int64 [{n}] on {device}, got "
                                 f"{positions.dtype} {tuple(positions.shape)} on {positions.device}")
            bits = 64 if positions.dtype == torch.int64 else 32
        if q_out is None:
            q_out = torch.empty((n, cfg.num_q_heads, cfg.head_dim), dtype=torch.bfloat16, device=device)
        else:
            _rows("q_out", q_out, cfg.num_q_heads, cfg.head_dim, n, device)
            _own_places("q_out", q_out)
        if k_out is None:
            k_out = torch.empty((n, cfg.num_kv_heads, cfg.head_dim), dtype=torch.bfloat16, device=device)
        else:
            _rows("k_out", k_out, cfg.num_kv_heads, cfg.head_dim, n, device)
            _own_places("k_out", k_out)
        _check_output("q_out", q_out, q, k, k_out)
        _check_output("k_out", k_out, k, q)
        rotary = self._rotary_args(device, q_weight, k_weight)
        if n == 0:
            return q_out, k_out
        chunk = native.PcpaChunk(cfg.interleave_size, batch, n, 0, _pointer(lengths), _pointer(chunk_starts))
        with torch.cuda.device(device):
            status = self._lib.pcpa_rotate(
                ctypes.byref(self._params), ctypes.byref(chunk), ctypes.byref(rotary), _pointer(positions), bits, 0,
                _row_view(native, q), _row_view(native, k), None, _row_view(native, q_out), _row_view(native, k_out),
                None, 0, torch.cuda.current_stream(device).cuda_stream)
        native.check(status)
        return q_out, k_out

    def prefill(self, q, k, v, *, first_pos: int, q_weight=None, k_weight=None):
        turns = self._turns.get(getattr(q, "device", None))
        if turns is not None:
            call = self._fast.get("rotate_prefill") or self._native_call("rotate_prefill", self._lib.pcpa_rotate)
            result = call(q, k, v, first_pos, q_weight, k_weight, turns)
            if type(result) is int:  # the status of a launch that failed
                self._native.check(result)
            if result is not None:
                return result
        # not the common form
        import torch

        cfg, native = self.config, self._native
        n = cfg.current_len
        _rows("q", q, cfg.num_q_heads, cfg.head_dim, n)
        device = q.device
        _rows("k", k, cfg.num_kv_heads, cfg.head_dim, n, device)
        _rows("v", v, cfg.num_kv_heads, cfg.head_dim, n, device)
        if not 0 <= int(first_pos) < 2**62:
            raise ValueError(f"first_pos must be non-negative and below 2^62, got {first_pos}")
        q_stacked = torch.empty((cfg.pcp_size, cfg.num_q_heads, cfg.local_q_len, cfg.head_dim), dtype=torch.bfloat16,
                                device=device)
        kv_current = torch.empty((2, cfg.num_kv_heads, n, cfg.head_dim), dtype=torch.bfloat16, device=device)
        k_out, v_out = kv_current.transpose(1, 2)
        rotary = self._rotary_args(device, q_weight, k_weight)
        chunk = native.PcpaChunk(cfg.interleave_size, 1, n, 0, None, None)
        with torch.cuda.device(device):
            status = self._lib.pcpa_rotate(
                ctypes.byref(self._params), ctypes.byref(chunk), ctypes.byref(rotary), None, -1, int(first_pos),
                _row_view(native, q), _row_view(native, k), _row_view(native, v),
                native.PcpaRows(q_stacked.data_ptr(), 0, 0), _row_view(native, k_out), _row_view(native, v_out), 1,
                torch.cuda.current_stream(device).cuda_stream)
        native.check(status)
        return q_stacked, kv_current
