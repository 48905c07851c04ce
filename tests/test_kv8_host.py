"""The 8-bit cache without a device: sizes, refusals of the wrappers and of the C entry points, and the
claim that 32-bit division decides every code as exact arithmetic does."""

import ctypes as C
from fractions import Fraction

import numpy as np
import pytest
import torch

from kv8_ref import quantise


def test_struct_matches_the_header():
    from helix_substrate_b200._lib import HxqKv8
    assert C.sizeof(HxqKv8) == 6 * 8 + 4 * 4 and HxqKv8.slots.offset == 48 and HxqKv8.max_len.offset == 60


def test_c_entry_points_refuse_without_a_device():
    from helix_substrate_b200 import _lib
    L = _lib.lib()
    buf = np.zeros(64, dtype=np.uint8)
    p = buf.ctypes.data
    p += -p % 16
    ok = dict(slots=2, nkv=2, D=64, max_len=128)

    def cache(**kw):
        return C.byref(_lib.HxqKv8(p, p, p, p, p, p, *(dict(ok, **kw)[n] for n in ("slots", "nkv", "D", "max_len"))))

    def step(c, B=2, nq=4, ld=512, ldq=256, stride=1, qkv=p):
        return L.hxq_rope_append_kv8(c, qkv, ld, p, stride, p, p, p, ldq, B, nq, None)

    def prompt(c, cu=p, T=2, S=2, max_q=2, ldk=128, k_out=p, ld=512):
        return L.hxq_rope_append_prompt_kv8(c, p, ld, T, cu, S, max_q, p, 1, p, p, p, 256, k_out, ldk, 4, None)

    def decode(c, B=2, nq=4, ws=None, nb=0, stride=1, q=p):
        return L.hxq_attn_decode_kv8(c, q, nq * 64, p, stride, p, nq * 64, ws, nb, B, nq, 0.1, None)

    def rows(c, S=2, n=10, ld=(1 << 14, 1 << 12, 64), out=p):
        return L.hxq_kv8_rows(c, p, 1, S, n, out, out, *ld, None)

    E = _lib
    for f in (step, prompt, decode, rows):
        assert f(None) == E.HXQ_E_ARG
        assert f(C.byref(E.HxqKv8(p, None, p, p, p, p, 2, 2, 64, 128))) == E.HXQ_E_ARG
        assert f(C.byref(E.HxqKv8(p + 8, p, p, p, p, p, 2, 2, 64, 128))) == E.HXQ_E_ALIGN
        for bad in (dict(D=24), dict(D=0), dict(D=144), dict(max_len=100), dict(max_len=0), dict(nkv=0), dict(slots=0)):
            assert f(cache(**bad)) == E.HXQ_E_SHAPE, bad
    assert step(cache(), B=0) == E.HXQ_E_ARG and step(cache(), qkv=None) == E.HXQ_E_ARG
    assert step(cache(), B=3) == E.HXQ_E_SHAPE and step(cache(), nq=3) == E.HXQ_E_SHAPE and step(cache(), ld=511) == E.HXQ_E_SHAPE
    assert step(cache(), ldq=255) == E.HXQ_E_SHAPE and step(cache(), stride=2) == E.HXQ_E_SHAPE
    assert step(cache(), qkv=p + 2) == E.HXQ_E_ALIGN and step(cache(), ld=514) == E.HXQ_E_ALIGN
    assert prompt(cache(), cu=None) == E.HXQ_E_ARG and prompt(cache(), S=3) == E.HXQ_E_SHAPE and prompt(cache(), ldk=120) == E.HXQ_E_SHAPE
    assert prompt(cache(), T=-1) == E.HXQ_E_ARG and prompt(cache(), max_q=-1) == E.HXQ_E_ARG and prompt(cache(), k_out=p + 4) == E.HXQ_E_ALIGN
    assert prompt(cache(), T=0) == E.HXQ_OK and prompt(cache(), max_q=0) == E.HXQ_OK         # nothing to do
    assert decode(cache(max_len=1 << 20)) == E.HXQ_E_WORKSPACE
    nb = L.hxq_attn_decode_kv8_workspace_bytes(2, 4, 2, 64, 1 << 20)
    assert nb > 0 and decode(cache(max_len=1 << 20), ws=p, nb=nb - 1) == E.HXQ_E_WORKSPACE
    assert decode(cache(), nq=18) == E.HXQ_E_SHAPE and decode(cache(), B=3) == E.HXQ_E_SHAPE and decode(cache(), q=p + 8) == E.HXQ_E_ALIGN
    assert rows(cache(), S=3) == E.HXQ_E_SHAPE and rows(cache(), ld=(1 << 14, 1 << 12, 60)) == E.HXQ_E_SHAPE
    assert rows(cache(), ld=(1 << 14, 1 << 12, 68)) == E.HXQ_E_ALIGN and rows(cache(), n=0) == E.HXQ_OK and rows(cache(), out=None) == E.HXQ_E_ARG
    assert L.hxq_attn_decode_kv8_workspace_bytes(0, 4, 2, 64, 128) == 0


def test_wrappers_refuse_cpu_tensors_and_odd_caches():
    from helix_substrate_b200.kv8 import Kv8Cache
    with pytest.raises(TypeError, match="CUDA"):
        Kv8Cache.empty(1, 2, 100, 64, "cpu")
    t = [torch.zeros(1, 2, 64, 64, dtype=torch.int8)] * 2 + [torch.zeros(1, 2, 1)] * 2 + [torch.zeros(1, 2, 64, 64, dtype=torch.bfloat16)] * 2
    for i, wrong in ((0, t[0].float()), (1, t[0][:, :1]), (2, t[2].double()), (4, t[4].half()), (5, t[4].transpose(1, 2))):
        with pytest.raises(TypeError):
            Kv8Cache(*(wrong if j == i else x for j, x in enumerate(t)))
    with pytest.raises(ValueError):
        Kv8Cache(torch.zeros(1, 64, 64, dtype=torch.int8), *t[1:])


def test_32_bit_division_decides_codes_exactly():
    """x and the scale have 8 significant bits each: fp32 max|x| / 127, rounded up to bf16, and x / scale, rounded to even, give the
    codes of exact arithmetic, for every mantissa of max|x| and of x and a range of exponents between them."""
    m = torch.arange(128, 256, dtype=torch.float32)
    for e in (-126, -10, 0, 1, 60):
        amax = m * 2.0 ** e
        r = amax / 127.0
        s = ((r.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32).clamp_min(2.0 ** -126)
        for a, x in zip(amax.tolist(), s.tolist()):
            exact = Fraction(a) / 127
            assert Fraction(x) >= exact and (x == 2.0 ** -126 or Fraction(x) - exact < Fraction(x) / 128)
            for d in range(0, 9):
                y = torch.arange(128, 256, dtype=torch.float32) * 2.0 ** (e - d)
                y = y[y <= a]
                got = torch.round(y / x)
                q, want = Fraction(x), []
                for v in y.tolist():
                    want.append(round(Fraction(v) / q))        # (a Fraction rounds ties to even)
                assert got.tolist() == want and max(want, default=0) <= 127


def test_reference_quantiser_bounds():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 128, 32, generator=g).bfloat16()
    codes, s = quantise(x)
    back = codes.double() * s.repeat_interleave(64, 1)[..., None]
    assert codes.abs().max() == 127 or codes.abs().max() == 126
    assert float(((back - x.double()).abs() / s.repeat_interleave(64, 1)[..., None]).max()) <= 0.5


@pytest.mark.parametrize("T", [1, 3])
def test_prompt_append_takes_no_rows_that_lie_over_one_another(T, monkeypatch):
    """k_out's rows are written by their stride: one expanded over the tokens, or with rows that overlap, is refused before the C entry
    is called (whose stride could not stand for it); a single row may have any stride."""
    from types import SimpleNamespace
    from helix_substrate_b200 import kv8
    calls = []
    monkeypatch.setattr(kv8, "_call", lambda dev, name, *args: calls.append(args))
    nq, nkv, D = 4, 2, 64
    cache = SimpleNamespace(device=torch.device("cpu"), kv_heads=nkv, D=D, max_len=128, slots=2, _ref=None)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)       # noqa: E731

    def append(k_out):
        kv8.rope_append_prompt_kv8(bf(T, (nq + 2 * nkv) * D), torch.tensor([0, T], dtype=torch.int32), T, torch.tensor([0]), torch.zeros(128, D),
                                   torch.zeros(128, D), bf(T, nq * D), k_out, cache, nq)
        return calls.pop()[-2]          # the stride that the C entry gets

    assert append(bf(T, nkv, D)) == nkv * D and append(bf(T, nkv + 1, D)[:, :nkv]) >= nkv * D
    for k_out in (bf(1, nkv, D).expand(T, nkv, D), bf(T * D + nkv * D).as_strided((T, nkv, D), (D, D, 1))):
        if T == 1:
            assert append(k_out) >= nkv * D
        else:
            with pytest.raises(TypeError, match="k_out"):
                append(k_out)
            assert not calls


@pytest.mark.parametrize("e", [-126, -124, -118, -100, -10, 0, 1, 60, 120, 127])
def test_reciprocal_and_snapping_give_the_exact_codes(e):
    """The append's arithmetic, step by step in fp32: x fl(1 / s) added to 12288 in one rounding and taken off again (multiples of 1/1024),
    the code from the low byte of that + 1.5 * 2^23.  Under every mantissa of max|x|, for every mantissa of x in ten octaves, both signs.
    x / s is a tie or 1/510 and more off one, so its fp64 quotient, off by 2^-46 at most, rounds as exact arithmetic does."""
    f32 = np.float32
    m = np.arange(128, 256) * 2.0 ** (e - 7)
    m = m[m < 3.39e38].astype(f32)
    s = ((m / f32(127)).view(np.uint32) + np.uint32(0xffff) & np.uint32(0xffff0000)).view(f32)
    s = np.maximum(s, f32(2.0 ** -126))[:, None]
    x = np.concatenate([np.arange(128, 256) * 2.0 ** (e - 7 - d) for d in range(10)])
    x = torch.from_numpy(np.concatenate([x, -x, [0.0]])).bfloat16().double().numpy()          # (some below 2^-133: none)
    x = np.where(np.abs(x) <= m[:, None].astype(np.float64), x, 0.0)
    want = np.rint(x / s.astype(np.float64))
    inv = f32(1) / s
    # (the product has 32 bits, 12288 is 2^13.6 and x inv at least 2^-12 where it can matter: fp64 holds the sum, one rounding follows)
    q = (x * inv.astype(np.float64) + 12288.0).astype(f32) - f32(12288)
    assert np.array_equal(np.abs(q - np.floor(q)) == 0.5, np.abs(x / s.astype(np.float64) - np.floor(x / s.astype(np.float64))) == 0.5), "ties are ties"
    code = ((q + f32(12582912)).view(np.uint32) & np.uint32(0xff)).astype(np.uint8).view(np.int8)
    assert np.array_equal(code, want) and np.abs(want).max() <= 127
