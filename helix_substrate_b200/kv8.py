"""A key/value cache held in 8 bits, and the operators that fill and read it: rotary embedding +
append (one token a sequence, or packed prompts), single-query attention, rows back as bf16.
Thin bf16 wrappers over the C ABI; no counterpart in the reference, whose decode loop keeps the
framework's 16-bit cache (helix_substrate/basin_runtime.py:358-445)."""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import HxqKv8

BLOCK = 64      # positions that share one scale


_raw_stream = torch._C._cuda_getCurrentRawStream
_entries: dict = {}


def _call(dev: torch.device, name: str, *args) -> None:
    """One C call on the current stream of ``dev`` (appended as its last argument), ``dev`` being current."""
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = getattr(_lib.lib(), name)
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        st = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            st = f(*args, _raw_stream(index))
    if st != _lib.HXQ_OK:
        _lib.check(st, name)


def _rows(t: torch.Tensor, name: str, dev: torch.device, width: int) -> None:
    if not (t.dtype is torch.bfloat16 and t.device == dev and t.shape[1:] == (width,) and t.stride()[1] == 1):
        raise TypeError(f"{name}: expected a bf16 [rows, {width}] tensor on {dev}, contiguous along its rows, got "
                        f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _ints(t: torch.Tensor, name: str, dev: torch.device, dtype: torch.dtype, n: int) -> None:
    if not (t.dtype is dtype and t.device == dev and t.shape == (n,) and t.is_contiguous()):
        raise TypeError(f"{name}: expected a contiguous {dtype} tensor of {n} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _positions(t: torch.Tensor, name: str, dev: torch.device, n: int) -> int:
    """Checks int64 positions, one per sequence or one for all; returns their stride."""
    shape = t.shape
    if not (t.dtype is torch.int64 and t.device == dev and (shape == (n,) or shape == (1,)) and t.is_contiguous()):
        raise TypeError(f"{name}: expected a contiguous int64 tensor of 1 or {n} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return int(n > 1 and shape[0] == n)


class Kv8Cache:
    """Keys and values of ``slots`` sequences in 8 bits: codes int8 [slots, kv_heads, max_len, D], one fp32
    scale per block of 64 positions and head, and a bf16 tail [slots, kv_heads, 64, D] with the rows of each
    sequence's last, unfinished block (row = position mod 64).  ``x = scale * code``, the scale being
    max|x| / 127 of its block rounded up to bf16 (2^-126 at least), the code rounded to nearest even; a block
    with an infinity or a NaN has the scale NaN.  A row is quantised once, when its block is complete."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 k_tail: torch.Tensor, v_tail: torch.Tensor):
        if k.ndim != 4:
            raise ValueError(f"k: expected [slots, kv_heads, max_len, D], got {tuple(k.shape)}")
        slots, nkv, max_len, D = k.shape
        want = {"k": (k, torch.int8, (slots, nkv, max_len, D)), "v": (v, torch.int8, (slots, nkv, max_len, D)),
                "k_scale": (k_scale, torch.float32, (slots, nkv, max_len // BLOCK)),
                "v_scale": (v_scale, torch.float32, (slots, nkv, max_len // BLOCK)),
                "k_tail": (k_tail, torch.bfloat16, (slots, nkv, BLOCK, D)),
                "v_tail": (v_tail, torch.bfloat16, (slots, nkv, BLOCK, D))}
        for name, (t, dtype, shape) in want.items():
            if t.dtype is not dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != k.device:
                raise TypeError(f"{name}: expected a contiguous {dtype} tensor {shape} on {k.device}, got {t.dtype} "
                                f"{tuple(t.shape)} on {t.device}")
        if slots < 1 or nkv < 1 or max_len < BLOCK or max_len % BLOCK or D % 16 or not 16 <= D <= 128:
            raise ValueError(f"an 8-bit cache has at least one slot and KV head, max_len a multiple of {BLOCK} and D a multiple "
                             f"of 16 up to 128, got {tuple(k.shape)}")
        if not k.is_cuda:
            raise TypeError("k: expected a CUDA tensor (there is no CPU path)")
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail = k, v, k_scale, v_scale, k_tail, v_tail
        self.device, self.slots, self.kv_heads, self.max_len, self.D = k.device, slots, nkv, max_len, D
        self.desc = HxqKv8(*(t.data_ptr() for t in (k, v, k_scale, v_scale, k_tail, v_tail)), slots, nkv, D, max_len)
        self._ref = C.byref(self.desc)

    @classmethod
    def empty(cls, slots: int, kv_heads: int, max_len: int, D: int, device) -> "Kv8Cache":
        """A cache for sequences of up to ``max_len`` positions (rounded up to whole blocks)."""
        n = (max_len + BLOCK - 1) // BLOCK * BLOCK
        codes = lambda: torch.zeros(slots, kv_heads, n, D, device=device, dtype=torch.int8)             # noqa: E731
        scale = lambda: torch.zeros(slots, kv_heads, n // BLOCK, device=device, dtype=torch.float32)    # noqa: E731
        tail = lambda: torch.zeros(slots, kv_heads, BLOCK, D, device=device, dtype=torch.bfloat16)      # noqa: E731
        return cls(codes(), codes(), scale(), scale(), tail(), tail())

    def __getitem__(self, slots: slice) -> "Kv8Cache":
        """The same cache, some of its slots: ``cache[2:3]`` to append to or read one sequence."""
        if not isinstance(slots, slice) or slots.step not in (None, 1):
            raise TypeError("a Kv8Cache is indexed with a slice of its slots")
        return Kv8Cache(*(t[slots] for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail)))

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail))


def _tables(cos: torch.Tensor, sin: torch.Tensor, cache: Kv8Cache) -> None:
    for name, t in (("cos", cos), ("sin", sin)):
        if not (t.dtype is torch.float32 and t.device == cache.device and t.shape[1:] == (cache.D,) and t.shape[0] >= cache.max_len
                and t.is_contiguous()):
            raise TypeError(f"{name}: expected a contiguous fp32 [{cache.max_len} or more, {cache.D}] table on {cache.device}, got "
                            f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _groups(nq: int, cache: Kv8Cache) -> None:
    if nq < 1 or nq % cache.kv_heads:
        raise ValueError(f"{nq} query heads over {cache.kv_heads} KV heads")


def rope_append_kv8(qkv: torch.Tensor, pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, q_out: torch.Tensor,
                    cache: Kv8Cache, nq: int) -> torch.Tensor:
    """qkv [B, (nq + 2 kv_heads) D] of one new token per slot -> rotated q in q_out [B, nq D]; rotated k and v
    appended at position ``pos`` (int64 on the device, one per sequence or one for all).  A sequence whose position
    is negative or past the cache is left as it is, its q_out too."""
    _groups(nq, cache)
    dev, B = cache.device, qkv.shape[0]
    _rows(qkv, "qkv", dev, (nq + 2 * cache.kv_heads) * cache.D)
    _rows(q_out, "q_out", dev, nq * cache.D)
    _tables(cos, sin, cache)
    stride = _positions(pos, "pos", dev, B)
    if q_out.shape[0] != B or not 1 <= B <= cache.slots:
        raise ValueError(f"{B} tokens, {q_out.shape[0]} rows of q_out, {cache.slots} slots")
    _call(dev, "hxq_rope_append_kv8", cache._ref, qkv.data_ptr(), qkv.stride(0), pos.data_ptr(), stride, cos.data_ptr(), sin.data_ptr(),
          q_out.data_ptr(), q_out.stride(0), B, nq)
    return q_out


def rope_append_prompt_kv8(qkv: torch.Tensor, cu: torch.Tensor, max_q: int, pos: torch.Tensor, cos: torch.Tensor,
                           sin: torch.Tensor, q_out: torch.Tensor, k_out: Optional[torch.Tensor], cache: Kv8Cache,
                           nq: int) -> torch.Tensor:
    """The same for packed prompts: rows ``cu[s]`` .. ``cu[s + 1] - 1`` of qkv [T, (nq + 2 kv_heads) D] are the next
    tokens of slot s, from position ``pos[s]`` on (what the slot holds already).  ``cu`` int32 [S + 1] on the device,
    ascending; no sequence longer than ``max_q`` (rows past that are not looked at).  Rotated q in q_out [T, nq D],
    rotated k in k_out [T, kv_heads, D] (or None)."""
    _groups(nq, cache)
    dev, T, S = cache.device, qkv.shape[0], cu.shape[0] - 1 if cu.ndim == 1 else -1
    _rows(qkv, "qkv", dev, (nq + 2 * cache.kv_heads) * cache.D)
    _rows(q_out, "q_out", dev, nq * cache.D)
    _tables(cos, sin, cache)
    _ints(cu, "cu", dev, torch.int32, S + 1)
    if not 1 <= S <= cache.slots or q_out.shape[0] != T or max_q < 0:
        raise ValueError(f"{S} sequences of up to {max_q} tokens, {T} rows of qkv, {q_out.shape[0]} of q_out, {cache.slots} slots")
    stride = _positions(pos, "pos", dev, S)
    ld_k, max_q = 0, min(max_q, T)
    if k_out is not None:
        if not (k_out.dtype is torch.bfloat16 and k_out.device == dev and tuple(k_out.shape) == (T, cache.kv_heads, cache.D)
                and k_out.stride(2) == 1 and (cache.kv_heads == 1 or k_out.stride(1) == cache.D)
                and (T <= 1 or k_out.stride(0) >= cache.kv_heads * cache.D)):
            raise TypeError(f"k_out: expected a bf16 [{T}, {cache.kv_heads}, {cache.D}] tensor on {dev}, contiguous along heads and D, its "
                            f"rows apart")
        ld_k = k_out.stride(0) if T > 1 else cache.kv_heads * cache.D        # (a single row's stride says nothing)
    if T == 0:
        return q_out
    _call(dev, "hxq_rope_append_prompt_kv8", cache._ref, qkv.data_ptr(), qkv.stride(0), T, cu.data_ptr(), S, max_q, pos.data_ptr(), stride,
          cos.data_ptr(), sin.data_ptr(), q_out.data_ptr(), q_out.stride(0), None if k_out is None else k_out.data_ptr(), ld_k, nq)
    return q_out


_ws_bytes: dict = {}


def attn_decode_kv8(q: torch.Tensor, cache: Kv8Cache, pos: torch.Tensor, out: torch.Tensor, nq: int, scale: float) -> torch.Tensor:
    """Attention of one query token per slot over positions 0..pos of the cache (pos int64 on the device, one per
    sequence or one for all; a negative one, or one past the cache, gives zeros).  At most eight query heads per KV
    head.  A query row is held in 16 bits: off by 2^-16 of its largest element, whatever the size of the others.  The scratch comes from the caching allocator for the call alone, so captured graphs do not share it."""
    _groups(nq, cache)
    dev, B = cache.device, q.shape[0]
    _rows(q, "q", dev, nq * cache.D)
    _rows(out, "out", dev, nq * cache.D)
    stride = _positions(pos, "pos", dev, B)
    if out.shape[0] != B or not 1 <= B <= cache.slots:
        raise ValueError(f"{B} queries, {out.shape[0]} rows of out, {cache.slots} slots")
    key = (B, nq, cache.kv_heads, cache.D, cache.max_len)
    nb = _ws_bytes.get(key)
    if nb is None:
        nb = _ws_bytes[key] = _lib.lib().hxq_attn_decode_kv8_workspace_bytes(*key)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    _call(dev, "hxq_attn_decode_kv8", cache._ref, q.data_ptr(), q.stride(0), pos.data_ptr(), stride, out.data_ptr(), out.stride(0),
          None if ws is None else ws.data_ptr(), nb, B, nq, scale)
    return out


def kv8_rows(cache: Kv8Cache, length: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor):
    """Rows 0 .. length - 1 of every slot as bf16, scale * code rounded once, into k_out and v_out [S, kv_heads,
    rows, D] (any strides over the first three); at most ``rows`` of them, the rest of the outputs is left as it is.
    ``length`` int64 on the device, one per sequence or one for all: how many positions each slot holds."""
    dev, shape, strides = cache.device, k_out.shape, k_out.stride()
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if not (t.dtype is torch.bfloat16 and t.device == dev and t.shape == shape and t.stride() == strides and len(shape) == 4
                and shape[1] == cache.kv_heads and shape[3] == cache.D and strides[3] == 1):
            raise TypeError(f"{name}: expected a bf16 [slots, {cache.kv_heads}, rows, {cache.D}] tensor on {dev}, contiguous along D, both "
                            f"outputs alike, got {t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}")
    S = shape[0]
    if not 1 <= S <= cache.slots:
        raise ValueError(f"outputs of {S} sequences, {cache.slots} slots")
    stride = _positions(length, "length", dev, S)
    if shape[2] == 0:
        return k_out, v_out
    _call(dev, "hxq_kv8_rows", cache._ref, length.data_ptr(), stride, S, shape[2], k_out.data_ptr(), v_out.data_ptr(), strides[0], strides[1],
          strides[2])
    return k_out, v_out
