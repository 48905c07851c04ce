"""Attention of whole prompts without a device: the struct, the workspace's size, refusals of the C entry and of the wrapper."""

import ctypes as C

import numpy as np
import pytest
import torch


def _args(**kw):
    from helix_substrate_b200._lib import HxqAttn
    p = _args.buf.ctypes.data
    p += -p % 16
    a = dict(q=p, k=p, v=p, out=p, q_tok=512, q_head=128, k_seq=0, k_head=128, k_row=256, v_seq=0, v_head=128, v_row=256, o_tok=512, o_head=128,
             cu_q=p, cu_k=p, k_len=None, Tq=40, Tk=40, S=2, max_q=20, nq=4, nkv=2, D=128, causal=1, scale=0.1)
    for n, x in kw.items():
        a[n] = p + x[0] if isinstance(x, tuple) else x
    return C.byref(HxqAttn(*(a[n] for n, _ in HxqAttn._fields_)))


_args.buf = np.zeros(256, dtype=np.uint8)


def test_struct_matches_the_header():
    from helix_substrate_b200._lib import HxqAttn
    assert C.sizeof(HxqAttn) == 176 and HxqAttn.cu_q.offset == 112 and HxqAttn.Tq.offset == 136 and HxqAttn.scale.offset == 168


def test_c_entry_refuses_without_a_device():
    from helix_substrate_b200 import _lib as E
    L = E.lib()

    def call(ws=None, nb=0, **kw):
        return L.hxq_attn_prompt(_args(**kw), ws, nb, None, None)

    assert L.hxq_attn_prompt(None, None, 0, None, None) == E.HXQ_E_ARG and L.hxq_attn_prompt_workspace_bytes(None) == 0
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_q=None), dict(cu_k=None), dict(k_len=(0,)), dict(Tq=-1), dict(Tk=-1),
                dict(S=0), dict(max_q=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert call(**bad) == E.HXQ_E_ARG, bad
    for bad in (dict(nq=0), dict(nkv=0), dict(nq=3), dict(nq=130), dict(D=0), dict(D=12), dict(D=136), dict(Tk=0), dict(Tk=(1 << 30) + 1), dict(Tq=(1 << 30) + 1)):
        assert call(**bad) == E.HXQ_E_SHAPE, bad
    for bad in (dict(q=(8,)), dict(k=(2,)), dict(v=(8,)), dict(out=(8,)), dict(q_tok=516), dict(q_head=-8), dict(k_row=4), dict(v_head=1 << 38),
                dict(o_tok=4), dict(k_seq=2, cu_k=None, k_len=(0,))):
        assert call(**bad) == E.HXQ_E_ALIGN, bad
    assert call(Tq=0) == E.HXQ_OK and call(max_q=0) == E.HXQ_OK         # nothing to do


def test_workspace():
    """Few queries before many keys share the keys out; whole items need no workspace."""
    from helix_substrate_b200 import _lib as E
    L = E.lib()
    size = lambda **kw: L.hxq_attn_prompt_workspace_bytes(_args(**kw))
    slab = dict(cu_k=None, k_len=(0,), S=1, max_q=20, Tq=20)
    assert size() == 0 and size(**dict(slab, Tk=1000)) == 0 and size(**dict(slab, Tk=100000, S=80)) == 0
    assert size(Tq=100000, Tk=100000, max_q=100000) == 0
    assert size(Tq=100000, Tk=100000, max_q=20) == 0
    many = size(**dict(slab, Tk=1 << 20))
    assert many > 0 and many == size(**dict(slab, Tk=1 << 29)) and 0 < size(**dict(slab, Tk=2000)) < many
    assert size(**dict(slab, Tk=1 << 20, D=64)) < many and size(**dict(slab, Tk=1 << 20, nq=3)) == 0
    p = _args.buf.ctypes.data
    for ws, nb in ((None, many), (p + -p % 8, many - 1), (p + -p % 8 + 4, many)):
        assert L.hxq_attn_prompt(_args(**dict(slab, Tk=1 << 20)), ws, nb, None, None) == E.HXQ_E_WORKSPACE


def test_wrapper_refuses():
    from helix_substrate_b200.prompt_ops import attn_prompt
    q, k = torch.zeros(4, 4, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu, n = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([4])
    with pytest.raises(TypeError, match="CUDA"):
        attn_prompt(q, k, k, q, cu, 4, 0.1)
    with pytest.raises(ValueError, match="not both"):
        attn_prompt(q, k, k, q, cu, 4, 0.1, cu_k=cu, k_len=n)


def test_first_use_under_capture_is_refused(monkeypatch):
    """The device's status word is made and cleared outside a capture: as a node of a graph the clearing would run at every replay."""
    from helix_substrate_b200 import packed
    monkeypatch.setattr(packed, "_status_words", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        packed._status_word(torch.device("cpu"))
    assert not packed._status_words
    word = packed._status_words[None] = torch.tensor([-7], dtype=torch.int32)
    assert packed._status_word(torch.device("cpu")) is word


def test_status_is_read_per_device(monkeypatch):
    from helix_substrate_b200 import packed, prompt_ops
    monkeypatch.setattr(packed, "_status_words", {3: torch.tensor([-7], dtype=torch.int32)})
    assert prompt_ops.check_status(torch.device("cuda", 3)) == -7
    assert prompt_ops.check_status("cuda:2") == 0 and 2 not in packed._status_words        # nothing has run there
