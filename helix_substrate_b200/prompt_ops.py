"""Attention of whole prompts: causal, grouped heads, packed sequences of different lengths, keys and values
packed like the queries or in a cache's slabs.  A thin bf16 wrapper over the C ABI, one launch; no counterpart in
the reference, whose HF models use the framework's attention (helix_substrate/basin_runtime.py:281-330)."""

from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import _lib
from .kv8 import _call, _ints
from .packed import _status_word, check_status        # noqa: F401  (check_status: whether a wait inside attn_prompt gave up)


_ATTN = struct.Struct("@4P10q3P8if4x")       # HxqAttn as bytes, in half the time that its constructor takes
assert _ATTN.size == C.sizeof(_lib.HxqAttn)


def _heads(t: torch.Tensor, name: str, dev: torch.device, shape: tuple) -> None:
    if not (t.dtype is torch.bfloat16 and t.device == dev and t.is_cuda and t.shape == shape and t.stride()[-1] == 1):
        raise TypeError(f"{name}: expected a CUDA bf16 tensor {tuple('*' if w is None else w for w in shape)} on {dev}, contiguous along "
                        f"its last dimension, got {t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}")


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, max_q: int,
                scale: float, *, cu_k: Optional[torch.Tensor] = None, k_len: Optional[torch.Tensor] = None,
                causal: bool = True) -> torch.Tensor:
    """Sequence s has the queries ``q[cu_q[s]: cu_q[s + 1]]`` of q [T, nq, D] (int32 offsets on the device, none longer
    than ``max_q``: queries past it are not computed and their rows of ``out`` left as they are).  Its keys and values are the same rows of k, v [T, nkv, D]; or rows ``cu_k[s]`` .. of k, v [Tk, nkv,
    D]; or rows 0 .. ``k_len[s] - 1`` (int64) of slab s of k, v [S, nkv, rows, D].  Causal attention is aligned at the end:
    with more keys than queries the queries are the last ones.  A query that sees no key gets zeros, rows of ``out``
    [T, nq, D] of no sequence are left as they are, and what a query does not see may hold anything.  q, k, v and out may be
    views (strides of whole 16 bytes).  ``check_status(device)`` tells whether a bounded wait inside the kernel gave up.  The first
    call on a device is not to be a captured one."""
    dev = q.device
    slabs = k_len is not None
    if slabs and cu_k is not None:
        raise ValueError("keys lie packed (cu_k) or in slabs (k_len), not both")
    q_shape, k_shape = q.shape, k.shape
    _heads(q, "q", dev, q_shape if len(q_shape) == 3 else (None, None, None))
    T, nq, D = q_shape
    S = cu_q.shape[0] - 1 if cu_q.ndim == 1 else -1
    if S < 1 or max_q < 0:
        raise ValueError(f"cu_q of shape {tuple(cu_q.shape)}, max_q {max_q}")
    _ints(cu_q, "cu_q", dev, torch.int32, S + 1)
    if slabs:
        nkv, rows = k_shape[1:3] if len(k_shape) == 4 else (None, None)
        _heads(k, "k", dev, (S, nkv, rows, D))
    else:
        rows, nkv = k_shape[:2] if len(k_shape) == 3 else (None, None)
        _heads(k, "k", dev, (rows, nkv, D))
    _heads(v, "v", dev, k_shape)
    _heads(out, "out", dev, q_shape)
    if nkv < 1 or nq % nkv:
        raise ValueError(f"{nq} query heads over {nkv} KV heads")
    if slabs:
        _ints(k_len, "k_len", dev, torch.int64, S)
    elif cu_k is not None:
        _ints(cu_k, "cu_k", dev, torch.int32, S + 1)
    elif rows != T:
        raise ValueError(f"{T} rows of q and {rows} of k: cu_k says where each sequence's keys lie")
    else:
        cu_k = cu_q
    if T == 0 or max_q == 0:
        return out
    if rows == 0:
        raise ValueError("k and v have no rows")
    ks, vs, qs, os = k.stride(), v.stride(), q.stride(), out.stride()
    if not slabs:
        ks, vs = (0, ks[1], ks[0]), (0, vs[1], vs[0])
    p = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qs[0], qs[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os[0], os[1],
                   cu_q.data_ptr(), 0 if slabs else cu_k.data_ptr(), k_len.data_ptr() if slabs else 0, T, rows, S, min(max_q, T), nq, nkv, D,
                   1 if causal else 0, scale)
    nb = _lib.lib().hxq_attn_prompt_workspace_bytes(p)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None       # for this call alone: captured graphs do not share it
    _call(dev, "hxq_attn_prompt", p, None if ws is None else ws.data_ptr(), nb, _status_word(dev).data_ptr())
    return out
