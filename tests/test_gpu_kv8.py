"""The 8-bit key/value cache: what an append writes, what attention and kv8_rows read, against plain
64-bit arithmetic; streams, captured graphs, idle slots and rows that must not be touched."""

import pytest
import torch

from conftest import rel_l2
from kv8_ref import BLOCK, RefCache, attention, rotate, tables

pytestmark = pytest.mark.gpu

# bf16 rounding is off by at most 2^-9 of a value (half of eps 2^-7 ... eps / 2 = 2^-8 bounds the relative error); the rms over
# random mantissas is below 2^-9.  An fp16 probability adds 2^-11 at most, rms below 2^-12.  rel-L2 of an output: 2^-8 at most.
TOL = 2.0 ** -8


def _dev():
    return torch.device("cuda:0")


def _filled(slots, nkv, max_len, D, lens, seed, loud=1.0):
    """A cache whose slot s holds lens[s] random rows, appended through the C ABI, and its reference."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_prompt_kv8
    dev = _dev()
    g = torch.Generator().manual_seed(seed)
    cache, ref = Kv8Cache.empty(slots, nkv, max_len, D, dev), RefCache(slots, nkv, D)
    T = sum(lens)
    qkv = (torch.randn(T, 3 * nkv * D, generator=g) * loud).bfloat16()
    cos, sin = tables(cache.max_len, D, "cpu")
    cu, at = [0], 0
    for s, n in enumerate(lens):
        x = qkv[at: at + n].view(n, 3 * nkv, D)
        ref.append(s, rotate(x[:, nkv: 2 * nkv], cos[:n, None], sin[:n, None]), x[:, 2 * nkv:])
        at += n
        cu.append(at)
    if T:
        rope_append_prompt_kv8(qkv.to(dev), torch.tensor(cu, dtype=torch.int32, device=dev), max(lens), torch.zeros(slots, dtype=torch.int64, device=dev),
                               cos.to(dev), sin.to(dev), torch.empty(T, nkv * D, device=dev, dtype=torch.bfloat16), None, cache, nkv)
    return cache, ref


def _check_cache(cache, ref):
    """Codes, scales and tails are exactly what 64-bit arithmetic makes of the rows."""
    for name in ("k", "v"):
        codes, scale, tail = (getattr(cache, name + x).cpu() for x in ("", "_scale", "_tail"))
        for s in range(cache.slots):
            n = ref.length(s)
            whole = n // BLOCK * BLOCK
            want = ref.values(name, s)
            got = codes[s, :, :whole].double() * scale[s, :, : whole // BLOCK].double().repeat_interleave(BLOCK, 1)[..., None]
            assert torch.equal(got, want[:, :whole]), (name, s, "finished blocks")
            assert torch.equal(tail[s, :, : n - whole].double(), want[:, whole:]), (name, s, "tail")


@pytest.mark.parametrize("nq,nkv,D", [(28, 4, 128), (4, 2, 64), (3, 1, 16), (8, 8, 80), (6, 2, 96)])
def test_append_prompts_in_pieces(nq, nkv, D):
    """Pieces that start and end inside blocks, a slot that gets nothing, rows behind the last sequence: the cache is exactly the
    rows', however they were cut; q and k are the 64-bit rotation rounded once; other rows keep what they held."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_prompt_kv8
    dev, max_len = _dev(), 640
    g = torch.Generator().manual_seed(nq * 1000 + D)
    cache, ref = Kv8Cache.empty(4, nkv, max_len, D, dev), RefCache(4, nkv, D)
    cos, sin = tables(max_len, D, "cpu")
    width = (nq + 2 * nkv) * D
    for lens in ([1, 0, 64, 63], [62, 0, 1, 1], [200, 0, 64, 129], [3, 0, 0, 127], [64, 0, 65, 1]):
        S, T = len(lens), sum(lens)
        big = torch.randn(T + 3, width + 8, generator=g).bfloat16()
        qkv = big[:, :width]
        pos = [ref.length(s) for s in range(S)]
        cu = [sum(lens[:s]) for s in range(S + 1)]
        q_out = torch.full((T + 3, nq * D), 7.0, device=dev, dtype=torch.bfloat16)
        k_out = torch.full((T + 3, nkv, D), 7.0, device=dev, dtype=torch.bfloat16)
        rope_append_prompt_kv8(big.to(dev)[:, :width], torch.tensor(cu, dtype=torch.int32, device=dev), max(lens),
                               torch.tensor(pos, device=dev), cos.to(dev), sin.to(dev), q_out, k_out, cache, nq)
        x = qkv.reshape(T + 3, nq + 2 * nkv, D)
        at = torch.tensor([p + i for p, n in zip(pos, lens) for i in range(n)])
        turned = rotate(x[:T, : nq + nkv], cos[at][:, None], sin[at][:, None])
        assert torch.equal(q_out[:T].cpu(), turned[:, :nq].reshape(T, -1))
        assert torch.equal(k_out[:T].cpu(), turned[:, nq:])
        assert bool((q_out[T:] == 7).all()) and bool((k_out[T:] == 7).all()), "rows of no sequence"
        for s in range(S):
            ref.append(s, turned[cu[s]: cu[s + 1], nq:], x[cu[s]: cu[s + 1], nq + nkv:])
        _check_cache(cache, ref)


@pytest.mark.parametrize("S", [75, 32, 33, 1100])
def test_append_of_many_packed_prompts(S):
    """More sequences than a warp has lanes, most of them short or empty, one long: every block finds its CTA."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_prompt_kv8
    dev, nq, nkv, D, max_len = _dev(), 5, 1, 112, 1024
    g = torch.Generator().manual_seed(8)
    cache, ref = Kv8Cache.empty(S, nkv, max_len, D, dev), RefCache(S, nkv, D)
    cos, sin = tables(max_len, D, "cpu")
    for turn in range(2):
        lens = [int(x) for x in torch.randint(0, 30, (S,), generator=g)]
        lens[3], lens[20], lens[S - 1] = 500, 0, 64
        pos = [ref.length(s) for s in range(S)]
        cu = [sum(lens[:s]) for s in range(S + 1)]
        qkv = torch.randn(cu[-1], (nq + 2 * nkv) * D, generator=g).bfloat16()
        q_out = torch.empty(cu[-1], nq * D, device=dev, dtype=torch.bfloat16)
        rope_append_prompt_kv8(qkv.to(dev), torch.tensor(cu, dtype=torch.int32, device=dev), 500, torch.tensor(pos, device=dev), cos.to(dev), sin.to(dev),
                               q_out, None, cache, nq)
        x = qkv.view(-1, nq + 2 * nkv, D)
        at = torch.tensor([p + i for p, n in zip(pos, lens) for i in range(n)])
        turned = rotate(x[:, : nq + nkv], cos[at][:, None], sin[at][:, None])
        assert torch.equal(q_out.cpu(), turned[:, :nq].flatten(1))
        for s in range(S):
            ref.append(s, turned[cu[s]: cu[s + 1], nq:], x[cu[s]: cu[s + 1], nq + nkv:])
        _check_cache(cache, ref)


def test_rotation_next_to_borders():
    """Angles and values for which fp32 sums lie on or next to a border of bf16, cancel to nothing, or overflow: as 64-bit arithmetic
    rounds them; infinities and NaNs stay what they are."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_prompt_kv8
    dev, D, n = _dev(), 128, 640
    g = torch.Generator().manual_seed(12)
    x = torch.randn(n, 3, D, generator=g).bfloat16()
    x[:64] = torch.randint(-300, 300, (64, 3, D), generator=g).bfloat16()
    x[64:128] *= 1e30
    x[128:192] *= 1e-38
    x[200, 0, 5], x[201, 0, 70], x[202, 0, 9] = float("inf"), float("-inf"), float("nan")
    x[203, 0, 3], x[203, 0, 67] = 3.3e38, -3.3e38
    x[192:256, 1:] = 1.0
    cos, sin = torch.randn(n, D, generator=g), torch.randn(n, D, generator=g)
    cos[:32], sin[:32] = 1.0, 2.0 ** -9          # sums half-way between two bf16 numbers
    cos[32:64], sin[32:64] = 0.5, 0.5            # and sums that cancel
    cos[300:400] = sin[300:400] + 1e-7 * torch.randn(100, D, generator=g)
    x[300:400, :, 64:] = x[300:400, :, :64]
    cache = Kv8Cache.empty(1, 1, n, D, dev)
    q_out = torch.empty(n, D, device=dev, dtype=torch.bfloat16)
    rope_append_prompt_kv8(x.flatten(1).to(dev), torch.tensor([0, n], dtype=torch.int32, device=dev), n, torch.zeros(1, dtype=torch.int64, device=dev),
                           cos.to(dev), sin.to(dev), q_out, None, cache, 1)
    want, got = rotate(x[:, 0], cos, sin), q_out.cpu()
    assert torch.equal(want.isnan(), got.isnan())
    assert torch.equal(want.nan_to_num(0.0, 1.0, -1.0), got.nan_to_num(0.0, 1.0, -1.0))


@pytest.mark.parametrize("one_pos", [False, True])
def test_append_steps(one_pos):
    """130 tokens one at a time (two finished blocks), all slots alike or each at its own position."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_kv8
    dev, B, nq, nkv, D, max_len = _dev(), 3, 14, 2, 64, 256
    g = torch.Generator().manual_seed(5)
    cache, ref = Kv8Cache.empty(B, nkv, max_len, D, dev), RefCache(B, nkv, D)
    cos, sin = tables(max_len, D, "cpu")
    start = [0, 0, 0] if one_pos else [0, 30, 64]
    for s, n in enumerate(start):       # (rows the slot held already)
        if n:
            from helix_substrate_b200.kv8 import rope_append_prompt_kv8
            x = torch.randn(n, (nq + 2 * nkv) * D, generator=g).bfloat16()
            rope_append_prompt_kv8(x.to(dev), torch.tensor([0, n], dtype=torch.int32, device=dev), n, torch.zeros(1, dtype=torch.int64, device=dev),
                                   cos.to(dev), sin.to(dev), torch.empty(n, nq * D, device=dev, dtype=torch.bfloat16), None, cache[s: s + 1], nq)
            y = x.view(n, -1, D)
            ref.append(s, rotate(y[:, nq: nq + nkv], cos[:n, None], sin[:n, None]), y[:, nq + nkv:])
    cd, sd = cos.to(dev), sin.to(dev)
    q_out = torch.empty(B, nq * D, device=dev, dtype=torch.bfloat16)
    for i in range(130):
        at = torch.tensor([n + i for n in start])
        x = torch.randn(B, (nq + 2 * nkv) * D, generator=g).bfloat16()
        rope_append_kv8(x.to(dev), (at[:1] if one_pos else at).to(dev), cd, sd, q_out, cache, nq)
        y = x.view(B, -1, D)
        turned = rotate(y[:, : nq + nkv], cos[at][:, None], sin[at][:, None])
        assert torch.equal(q_out.cpu(), turned[:, :nq].reshape(B, -1)), i
        for s in range(B):
            ref.append(s, turned[s: s + 1, nq:], y[s: s + 1, nq + nkv:])
        if i % 13 == 0 or i in (33, 62, 63, 64, 126, 127, 128, 129):
            _check_cache(cache, ref)


def test_append_leaves_idle_and_full_slots_alone():
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_kv8, rope_append_prompt_kv8
    dev, nq, nkv, D, max_len = _dev(), 4, 2, 64, 128
    cache = Kv8Cache.empty(3, nkv, max_len, D, dev)
    names = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")
    before = {n: getattr(cache, n).clone() for n in names}
    cos, sin = tables(max_len, D, dev)
    x = torch.randn(3, (nq + 2 * nkv) * D, device=dev).bfloat16()
    q = torch.full((3, nq * D), 3.0, device=dev, dtype=torch.bfloat16)
    rope_append_kv8(x, torch.tensor([-1, max_len, 1 << 40], device=dev), cos, sin, q, cache, nq)
    assert bool((q == 3).all()) and all(torch.equal(before[n], getattr(cache, n)) for n in names)
    # a prompt that runs past the end of its slot: what has a place is kept, the other slots stay
    x = torch.randn(70, (nq + 2 * nkv) * D, device=dev).bfloat16()
    q = torch.full((70, nq * D), 3.0, device=dev, dtype=torch.bfloat16)
    rope_append_prompt_kv8(x, torch.tensor([0, 0, 70, 70], dtype=torch.int32, device=dev), 70, torch.tensor([0, 100, -5], device=dev), cos, sin, q, None, cache, nq)
    assert bool((q[28:] == 3).all()) and not bool((q[:28] == 3).all(1).any())
    for n in names:
        assert torch.equal(before[n][0], getattr(cache, n)[0]) and torch.equal(before[n][2], getattr(cache, n)[2])
    # a max_q below the longest prompt: the rows past it are not looked at
    q.fill_(3.0)
    rope_append_prompt_kv8(x, torch.tensor([0, 70], dtype=torch.int32, device=dev), 10, torch.tensor([0], device=dev), cos, sin, q, None, cache[2:3], nq)
    assert bool((q[10:] == 3).all()) and torch.equal(cache.k_tail[2, :, 10:], before["k_tail"][2, :, 10:]) and not bool(cache.k[2].any())


@pytest.mark.parametrize("fill", ["zeros", "tiny", "huge", "inf", "nan"])
def test_blocks_of_extreme_values(fill):
    """A block of zeros, of bf16's smallest and largest values: exact codes; one with an infinity or a NaN reads back as NaN, and
    its neighbours do not."""
    from helix_substrate_b200.kv8 import Kv8Cache, kv8_rows, rope_append_prompt_kv8
    dev, nkv, D = _dev(), 2, 64
    g = torch.Generator().manual_seed(1)
    cache, ref = Kv8Cache.empty(1, nkv, 192, D, dev), RefCache(1, nkv, D)
    x = torch.randn(192, 3 * nkv, D, generator=g).bfloat16()
    mid = x[64:128]
    if fill == "zeros":
        mid.zero_()
    elif fill == "tiny":
        mid.copy_((mid.sign() * torch.randint(1, 4, mid.shape, generator=g) * 2.0 ** -133).bfloat16())
    elif fill == "huge":
        mid.copy_((mid.sign() * 3.3e38).bfloat16())
        mid[:, nkv: 2 * nkv] *= 0.5        # (a rotated pair of the largest values would overflow)
    else:
        mid[5, 2 * nkv, 7] = float(fill)
    cos, sin = tables(192, D, "cpu")
    rope_append_prompt_kv8(x.flatten(1).to(dev), torch.tensor([0, 192], dtype=torch.int32, device=dev), 192, torch.zeros(1, dtype=torch.int64, device=dev),
                           cos.to(dev), sin.to(dev), torch.empty(192, nkv * D, device=dev, dtype=torch.bfloat16), None, cache, nkv)
    k_out, v_out = (torch.zeros(1, nkv, 192, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    kv8_rows(cache, torch.tensor([192], device=dev), k_out, v_out)
    if fill in ("inf", "nan"):
        assert bool(v_out[0, 0, 64:128].isnan().all()) and int(v_out.isnan().sum()) == 64 * D and not bool(k_out.isnan().any())
        assert not bool(cache.v[0, 0, 64:128].any())
        x[64:128, 2 * nkv] = 0          # the rest as ever
        cache.v_scale[0, 0, 1] = 2.0 ** -126
    ref.append(0, rotate(x[:, nkv: 2 * nkv], cos[:192, None], sin[:192, None]), x[:, 2 * nkv:])
    _check_cache(cache, ref)


@pytest.mark.parametrize("nkv,D,max_len,lens", [(4, 128, 512, [1, 0, 64, 130, 448, 500]), (2, 64, 256, [63, 256]), (3, 80, 128, [128, 65, 0])])
def test_rows(nkv, D, max_len, lens):
    from helix_substrate_b200.kv8 import kv8_rows
    dev = _dev()
    cache, ref = _filled(len(lens), nkv, max_len, D, lens, seed=D)
    for rows in {max(lens), max(1, max(lens) - 70), max_len}:
        buf = torch.full((2, len(lens), nkv + 1, rows + 5, D), 9.0, device=dev, dtype=torch.bfloat16)
        k_out, v_out = buf[0, :, :nkv, :rows], buf[1, :, :nkv, :rows]
        kv8_rows(cache, torch.tensor(lens, device=dev), k_out, v_out)
        for s, n in enumerate(lens):
            n = min(n, rows)
            for name, o in (("k", k_out), ("v", v_out)):
                want = ref.values(name, s)[:, :n]
                assert torch.equal(o[s, :, :n].cpu(), want.float().bfloat16()), (name, s)
                assert bool((o[s, :, n:] == 9).all())
        assert bool((buf[:, :, nkv] == 9).all()) and bool((buf[:, :, :, rows:] == 9).all())


@pytest.mark.parametrize("nq,nkv,D", [(28, 4, 128), (40, 8, 128), (4, 2, 64), (8, 1, 128), (8, 8, 64), (3, 1, 16), (6, 2, 96), (5, 1, 80), (14, 2, 48)])
@pytest.mark.parametrize("max_len,lens", [(2304, [2048, 0, 1, 63, 64, 65, 129, 2300]), (128, [100]), (64, [64, 7]), (8192, [8192])])
def test_attn_decode_kv8(nq, nkv, D, max_len, lens):
    from helix_substrate_b200.kv8 import attn_decode_kv8
    dev, B = _dev(), len(lens)
    cache, ref = _filled(B, nkv, max_len, D, lens, seed=nq + max_len)
    for n in ("k_tail", "v_tail"):      # the rows past each sequence's last hold anything
        t = getattr(cache, n)
        for s, ln in enumerate(lens):
            t[s, :, ln % BLOCK:] = float("nan")
    for n, x in (("k_scale", float("nan")), ("v_scale", float("inf"))):
        for s, ln in enumerate(lens):
            getattr(cache, n)[s, :, ln // BLOCK:] = x
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(B, nq * D + 8, generator=g).bfloat16()
    q = wide[:, : nq * D]
    wide_out = torch.full((B, nq * D + 8), 5.0, device=dev, dtype=torch.bfloat16)
    out = wide_out[:, : nq * D]
    pos = torch.tensor([n - 1 for n in lens], device=dev)
    attn_decode_kv8(wide.to(dev)[:, : nq * D], cache, pos, out, nq, D ** -0.5)
    got = out.cpu().double().view(B, nq, D)
    for s, n in enumerate(lens):
        if n == 0:
            assert not bool(got[s].any()), "an empty slot gives zeros"
            continue
        want = attention(q[s].view(nq, 1, D), ref.values("k", s), ref.values("v", s), D ** -0.5)[:, 0]
        assert rel_l2(got[s], want) < TOL, (s, n, rel_l2(got[s], want))
        big = (got[s] - want).abs() / want.abs().clamp_min(float(want.pow(2).mean().sqrt()))
        assert float(big.max()) < 2.0 ** -7, (s, n)
    assert bool((wide_out[:, nq * D:] == 5).all())
    again = torch.empty_like(wide_out)[:, : nq * D]
    attn_decode_kv8(wide.to(dev)[:, : nq * D], cache, pos, again, nq, D ** -0.5)
    assert torch.equal(again, out), "the same call gives the same bits"


@pytest.mark.parametrize("case", ["loud queries", "quiet queries", "peaked", "one position for all", "nan query", "nan block"])
def test_attn_decode_kv8_values(case):
    """Queries far from 1 in size, scores far apart (a softmax that is nearly one row), NaNs where they belong."""
    from helix_substrate_b200.kv8 import attn_decode_kv8
    dev, B, nq, nkv, D, lens = _dev(), 2, 14, 2, 64, [333, 333]
    cache, ref = _filled(B, nkv, 512, D, lens, seed=3)
    q = torch.randn(B, nq, D, generator=torch.Generator().manual_seed(2))
    scale = D ** -0.5
    if case == "loud queries":
        q, scale = q * 1e30, scale * 1e-30
    elif case == "quiet queries":
        q, scale = q * 1e-30, scale * 1e30
    elif case == "peaked":
        q = q * 60
    q = q.bfloat16()
    if case == "nan query":
        q[0, 3, 5] = float("nan")
    if case == "nan block":
        cache.v_scale[1, 0, 2] = float("nan")
    pos = torch.tensor([332] if case == "one position for all" else [332, 332], device=dev)
    out = torch.empty(B, nq * D, device=dev, dtype=torch.bfloat16)
    attn_decode_kv8(q.flatten(1).to(dev), cache, pos, out, nq, scale)
    got = out.cpu().double().view(B, nq, D)
    for s in range(B):
        want = attention(q[s].view(nq, 1, D), ref.values("k", s), ref.values("v", s), scale)[:, 0]
        if case == "nan block" and s == 1:
            want[:7] = float("nan")
        nan = want.isnan()
        assert torch.equal(nan, got[s].isnan())
        assert rel_l2(got[s][~nan], want[~nan]) < TOL, case


@pytest.mark.parametrize("nq,nkv,D", [(4, 2, 64), (7, 1, 128), (2, 1, 112)])
@pytest.mark.parametrize("B", [14, 33, 70, 130, 300, 700])
def test_attn_decode_kv8_many_sequences(nq, nkv, D, B):
    """More sequences than a warp has lanes, lengths from nothing to many blocks, idle slots in between and at both ends: every
    CTA finds its share; all at one position too."""
    from helix_substrate_b200.kv8 import attn_decode_kv8
    dev, max_len = _dev(), 1280
    g = torch.Generator().manual_seed(B)
    lens = [0, 0] + [int(x) for x in torch.randint(0, 1281, (B - 4,), generator=g) // torch.randint(1, 20, (B - 4,), generator=g)] + [1280, 0]
    cache, ref = _filled(B, nkv, max_len, D, lens, seed=B)
    q = torch.randn(B, nq * D, generator=g).bfloat16()
    out = torch.full((B, nq * D), 5.0, device=dev, dtype=torch.bfloat16)
    attn_decode_kv8(q.to(dev), cache, torch.tensor([n - 1 for n in lens], device=dev), out, nq, 0.2)
    for s, n in enumerate(lens):
        want = attention(q[s].view(nq, 1, D), ref.values("k", s), ref.values("v", s), 0.2)[:, 0].reshape(-1) if n else torch.zeros(nq * D).double()
        assert (not bool(out[s].any()) if n == 0 else rel_l2(out[s].cpu().double(), want) < TOL), (s, n)
    held = [s for s, n in enumerate(lens) if n > 66]
    attn_decode_kv8(q.to(dev), cache, torch.tensor([63], device=dev), out, nq, 0.2)      # the first block of everybody
    for s in held[:5] + held[-5:]:
        want = attention(q[s].view(nq, 1, D), ref.values("k", s)[:, :64], ref.values("v", s)[:, :64], 0.2)[:, 0].reshape(-1)
        assert rel_l2(out[s].cpu().double(), want) < TOL, s


def test_a_long_cache_past_32_bit_offsets():
    """Slots whose codes lie beyond 2^31 bytes: appended to, read, attended to."""
    from helix_substrate_b200.kv8 import Kv8Cache, attn_decode_kv8, kv8_rows, rope_append_kv8
    dev, nq, nkv, D, max_len = _dev(), 16, 8, 128, 1 << 20
    cache = Kv8Cache.empty(3, nkv, max_len, D, dev)           # 1 GB of codes a slot, each of keys and values
    cos, sin = tables(64, D, dev)
    g = torch.Generator(device=dev).manual_seed(0)
    tall = torch.zeros(max_len, D, device=dev)
    tall[:, : D // 2], tall[:, D // 2:] = 1.0, 1.0            # angles of zero: cos 1, sin 0
    zero = torch.zeros_like(tall)
    p0 = max_len - 64
    rows = torch.randn(64, (nq + 2 * nkv) * D, device=dev, generator=g).bfloat16()
    q_out = torch.empty(1, nq * D, device=dev, dtype=torch.bfloat16)
    last = cache[2:3]
    for i in range(64):
        rope_append_kv8(rows[i: i + 1], torch.tensor([p0 + i], device=dev), tall, zero, q_out, last, nq)
    ref = RefCache(1, nkv, D)
    y = rows.cpu().view(64, -1, D)
    ref.append(0, y[:, nq: nq + nkv], y[:, nq + nkv:])
    got = last.k[0, :, p0:].cpu().double() * last.k_scale[0, :, -1].cpu().double()[:, None, None]
    assert torch.equal(got, ref.values("k", 0))
    # every earlier block of that slot: codes of zero but a score pushed down by nothing - attention averages them in
    out = torch.empty(3, nq * D, device=dev, dtype=torch.bfloat16)
    q = torch.zeros(3, nq * D, device=dev, dtype=torch.bfloat16)
    attn_decode_kv8(q, cache, torch.tensor([-1, 70, max_len - 1], device=dev), out, nq, D ** -0.5)
    want = (ref.values("v", 0).sum(1) / max_len).repeat_interleave(nq // nkv, 0).reshape(-1)
    assert not bool(out[:2].any()) and rel_l2(out[2].cpu().double(), want) < TOL
    del cos, sin
    k_out, v_out = (torch.empty(1, nkv, max_len, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    kv8_rows(last, torch.tensor([max_len], device=dev), k_out, v_out)
    assert torch.equal(v_out[0, :, p0:].cpu(), ref.values("v", 0).float().bfloat16()) and not bool(v_out[0, :, :p0].any())


def test_captured_steps_and_streams():
    """A captured append + attention replayed at moving positions equals the eager calls; two graphs replayed at once on two streams
    do not disturb one another; a call on a stream of its own is ordered by that stream."""
    from helix_substrate_b200.kv8 import Kv8Cache, attn_decode_kv8, rope_append_kv8
    dev, B, nq, nkv, D, max_len = _dev(), 2, 28, 4, 128, 4096
    cos, sin = tables(max_len, D, dev)
    x = torch.randn(2, 80, B, (nq + 2 * nkv) * D, device=dev, generator=torch.Generator(device=dev).manual_seed(0)).bfloat16()

    def state():
        return dict(cache=Kv8Cache.empty(B, nkv, max_len, D, dev), pos=torch.zeros(B, dtype=torch.int64, device=dev), x=torch.zeros_like(x[0, 0]),
                    q=torch.empty(B, nq * D, device=dev, dtype=torch.bfloat16), out=torch.empty(B, nq * D, device=dev, dtype=torch.bfloat16))

    def body(s):
        rope_append_kv8(s["x"], s["pos"], cos, sin, s["q"], s["cache"], nq)
        attn_decode_kv8(s["q"], s["cache"], s["pos"], s["out"], nq, D ** -0.5)

    want = []
    for w in range(2):
        s, outs = state(), []
        for i in range(80):
            s["x"].copy_(x[w, i]); s["pos"].fill_(i)
            body(s)
            outs.append(s["out"].clone())
        want.append(outs)
    states, graphs, streams = [state(), state()], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    side = torch.cuda.Stream()
    for s in states:
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            body(s)
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                body(s)
        graphs.append(graph)
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(80):
        for w in range(2):
            with torch.cuda.stream(streams[w]):
                states[w]["x"].copy_(x[w, i]); states[w]["pos"].fill_(i)
                graphs[w].replay()
                got[w].append(states[w]["out"].clone())
    torch.cuda.synchronize()
    for w in range(2):
        for i in range(80):
            assert torch.equal(got[w][i], want[w][i]), (w, i)


def test_kv8_refuses_on_the_gpu():
    from helix_substrate_b200 import _lib
    from helix_substrate_b200.kv8 import Kv8Cache, attn_decode_kv8, kv8_rows, rope_append_kv8, rope_append_prompt_kv8
    dev, nq, nkv, D = _dev(), 4, 2, 64
    cache = Kv8Cache.empty(2, nkv, 128, D, dev)
    cos, sin = tables(128, D, dev)
    bf = lambda *s: torch.zeros(*s, device=dev, dtype=torch.bfloat16)       # noqa: E731
    i64 = lambda *v: torch.tensor(v, device=dev)                           # noqa: E731
    qkv, q, out = bf(2, 8 * D), bf(2, nq * D), bf(2, nq * D)
    bad = [
        (TypeError, lambda: rope_append_kv8(qkv.float(), i64(0, 0), cos, sin, q, cache, nq)),
        (TypeError, lambda: rope_append_kv8(qkv[:, :-1], i64(0, 0), cos, sin, q, cache, nq)),
        (TypeError, lambda: rope_append_kv8(qkv, i64(0, 0).int(), cos, sin, q, cache, nq)),
        (TypeError, lambda: rope_append_kv8(qkv, i64(0, 0, 0), cos, sin, q, cache, nq)),
        (TypeError, lambda: rope_append_kv8(qkv, i64(0, 0), cos[:100], sin, q, cache, nq)),
        (TypeError, lambda: rope_append_kv8(qkv, i64(0, 0), cos.double(), sin, q, cache, nq)),
        (ValueError, lambda: rope_append_kv8(qkv, i64(0, 0), cos, sin, q, cache, 3)),
        (ValueError, lambda: rope_append_kv8(bf(3, 8 * D), i64(0), cos, sin, bf(3, nq * D), cache, nq)),
        (TypeError, lambda: rope_append_prompt_kv8(qkv, i64(0, 2), 2, i64(0), cos, sin, q, None, cache, nq)),
        (ValueError, lambda: rope_append_prompt_kv8(qkv, i64(0, 1, 1, 2).int(), 2, i64(0), cos, sin, q, None, cache, nq)),
        (TypeError, lambda: rope_append_prompt_kv8(qkv, i64(0, 2).int(), 2, i64(0), cos, sin, q, bf(2, nkv, 32), cache, nq)),
        (TypeError, lambda: attn_decode_kv8(q.half(), cache, i64(0, 0), out, nq, 0.1)),
        (ValueError, lambda: attn_decode_kv8(q, cache, i64(0, 0), bf(1, nq * D), nq, 0.1)),
        (TypeError, lambda: attn_decode_kv8(q, cache, torch.zeros(2, dtype=torch.int64), out, nq, 0.1)),
        (_lib.HxqError, lambda: attn_decode_kv8(bf(2, 18 * D), cache, i64(0, 0), bf(2, 18 * D), 18, 0.1)),       # nine query heads a KV head
        (_lib.HxqError, lambda: attn_decode_kv8(bf(2, nq * D + 1)[:, 1:], cache, i64(0, 0), out, nq, 0.1)),      # not 16-byte aligned
        (TypeError, lambda: kv8_rows(cache, i64(1), bf(2, nkv, 64, D), bf(2, nkv, 32, D))),
        (ValueError, lambda: kv8_rows(cache, i64(1), bf(3, nkv, 64, D), bf(3, nkv, 64, D))),
        (TypeError, lambda: cache[0]),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    assert rope_append_prompt_kv8(bf(0, 8 * D), i64(0, 0).int(), 5, i64(0), cos, sin, bf(0, nq * D), None, cache, nq).shape[0] == 0


@pytest.mark.parametrize("B,max_len", [(500, 256), (40, 2048), (2, 32768)])
def test_captured_attention_with_what_reads_it(B, max_len):
    """Joined over borders between shares, over a few and over many results; idle slots among them; each call followed by a reader
    that comes in early.  Replays leave the bits of calls one by one."""
    from helix_substrate_b200.decode_ops import swiglu
    from helix_substrate_b200.kv8 import Kv8Cache, attn_decode_kv8
    dev, nq, nkv, D, N = _dev(), 4, 2, 64, 8
    g = torch.Generator(device=dev).manual_seed(B)
    cache = Kv8Cache.empty(B, nkv, max_len, D, dev)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(-127, 128, t.shape, device=dev, generator=g, dtype=torch.int8))
    for t in (cache.k_scale, cache.v_scale):
        t.uniform_(0.005, 0.02, generator=g)
    for t in (cache.k_tail, cache.v_tail):
        t.normal_(generator=g)
    pos = torch.randint(-max_len // 16, max_len, (B,), device=dev, generator=g)
    qs = [torch.randn(B, nq * D, device=dev, generator=g).bfloat16() for _ in range(N)]
    gate = torch.full((B, nq * D), 20.0, device=dev, dtype=torch.bfloat16)
    outs, reads = [torch.empty_like(q) for q in qs], [torch.empty_like(q) for q in qs]

    def call(i, wait):
        attn_decode_kv8(qs[i], cache, pos, outs[i], nq, 0.1)
        if wait:
            torch.cuda.synchronize()
        swiglu(gate, outs[i], reads[i])

    for i in range(N):
        call(i, True)
    assert not bool(outs[0][pos < 0].any()) and bool(outs[0][pos >= 0].any(1).all())
    want = [t.clone() for t in outs + reads]
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
    st.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(st), torch.cuda.graph(graph, stream=st):
        for i in range(N):
            call(i, False)
    for _ in range(5):
        for t in outs + reads:
            t.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs + reads, want))


@pytest.mark.parametrize("S", [32, 33, 40, 1100])
@pytest.mark.parametrize("lead", [64, 200])
def test_append_behind_rows_of_no_sequence(S, lead):
    """Packed prompts whose first one does not start at row 0, fresh slots and slots that hold finished blocks: these, the slots on
    either side and the rows of no sequence stay as they are."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_prompt_kv8
    dev, nq, nkv, D, max_len = _dev(), 3, 1, 64, 256
    g = torch.Generator().manual_seed(S + lead)
    outer, ref = Kv8Cache.empty(S + 4, nkv, max_len, D, dev), RefCache(S, nkv, D)
    cache = outer[2: S + 2]
    cos, sin = tables(max_len, D, "cpu")
    for turn in range(3):
        lens = [int(x) for x in torch.randint(0, 80, (S,), generator=g)]
        lens[0], lens[S - 1] = (10, 64) if turn else (70, 5)
        pos = [ref.length(s) for s in range(S)]
        cu = [lead + sum(lens[:s]) for s in range(S + 1)]
        qkv = torch.randn(cu[-1], (nq + 2 * nkv) * D, generator=g).bfloat16()
        qkv[:lead] = float("nan")
        q_out = torch.full((cu[-1], nq * D), 7.0, device=dev, dtype=torch.bfloat16)
        k_out = torch.full((cu[-1], nkv, D), 7.0, device=dev, dtype=torch.bfloat16)
        rope_append_prompt_kv8(qkv.to(dev), torch.tensor(cu, dtype=torch.int32, device=dev), max(lens), torch.tensor(pos, device=dev), cos.to(dev), sin.to(dev),
                               q_out, k_out, cache, nq)
        x = qkv[lead:].view(-1, nq + 2 * nkv, D)
        at = torch.tensor([p + i for p, n in zip(pos, lens) for i in range(n)])
        turned = rotate(x[:, : nq + nkv], cos[at][:, None], sin[at][:, None])
        assert torch.equal(q_out[lead:].cpu(), turned[:, :nq].flatten(1)) and torch.equal(k_out[lead:].cpu(), turned[:, nq:])
        assert bool((q_out[:lead] == 7).all()) and bool((k_out[:lead] == 7).all())
        for s in range(S):
            a, b = cu[s] - lead, cu[s + 1] - lead
            ref.append(s, turned[a:b, nq:], x[a:b, nq + nkv:])
        _check_cache(cache, ref)
        for name in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail"):
            t = getattr(outer, name)
            assert not bool(t[:2].any()) and not bool(t[S + 2:].any()), name


@pytest.mark.parametrize("max_len,n", [(128, 36), (512, 300), (512, 257), (1 << 15, 20000), (1 << 15, 30)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_bad_values_in_the_tail(max_len, n, bad):
    """An infinity or a NaN in a row of V of the unfinished block is that dimension's result, for the heads that read it; in a row of K
    it makes its scores infinite or none.  Clusters and shares, a tail alone and behind blocks."""
    from helix_substrate_b200.kv8 import attn_decode_kv8
    dev, nq, nkv, D = _dev(), 14, 2, 64
    cache, ref = _filled(1, nkv, max_len, D, [n], seed=n)
    g = torch.Generator().manual_seed(n)
    q = torch.rand(1, nq, D, generator=g).bfloat16() + 0.25          # (of one sign: what an infinite key's score is)
    out = torch.empty(1, nq * D, device=dev, dtype=torch.bfloat16)
    pos = torch.tensor([n - 1], device=dev)

    def check(what):
        attn_decode_kv8(q.flatten(1).to(dev), cache, pos, out, nq, 0.1)
        got = out.cpu().double().view(nq, D)
        k, v = (ref.values(x, 0).repeat_interleave(nq // nkv, 0) for x in ("k", "v"))
        s = torch.einsum("hd,hjd->hj", q[0].double(), k) * 0.1
        want = torch.einsum("hj,hjd->hd", s.softmax(-1), v)          # (a key of -inf with a value of inf: 0 * inf, none)
        assert torch.equal(want.isnan(), got.isnan()), what
        assert torch.equal(want.isinf(), got.isinf()) and torch.equal(want[want.isinf()], got[got.isinf()]), what
        fine = want.isfinite()
        assert not bool(fine.any()) or rel_l2(got[fine], want[fine]) < TOL, what

    first, last = n // BLOCK * BLOCK, n - 1
    for name in ("v", "k"):
        tail, rows = getattr(cache, name + "_tail"), ref.rows[name][0]
        for row, h, d in ((first, 0, 3), (last, 1, 62)):
            keep = rows[h, row, d].clone()
            rows[h, row, d] = bad
            tail[0, h, row % BLOCK, d] = bad
            check((name, row))
            if row == last:
                break
            rows[h, row, d] = keep
            tail[0, h, row % BLOCK, d] = keep
        rows[1, last, 62], tail[0, 1, last % BLOCK, 62] = 0.5, 0.5


@pytest.mark.parametrize("e", [-126, -124, -100, -10, 0, 1, 60, 120])
def test_codes_of_every_mantissa(e):
    """Blocks under every mantissa of the largest element (scales clamped to 2^-126 among them), each holding every mantissa in nine
    octaves below it, both signs, ties in plenty: exactly the codes of exact arithmetic."""
    from helix_substrate_b200.kv8 import Kv8Cache, rope_append_prompt_kv8
    from kv8_ref import quantise
    dev, D = _dev(), 128
    m = torch.arange(128, 256, dtype=torch.float64)
    x = torch.cat([m * 2.0 ** (e - 7 - d) for d in range(9)])                          # [9 * 128]
    rows = torch.zeros(128, BLOCK * D, dtype=torch.float64)
    for i, a in enumerate(m.tolist()):
        y = x.where(x <= a * 2.0 ** (e - 7), -x / 2)
        rows[i, : 2 * y.numel()] = torch.cat([y, -y])
        rows[i, 2 * y.numel()] = a * 2.0 ** (e - 7)
    rows = rows.view(128 * BLOCK, D).bfloat16()
    n = rows.shape[0]
    qkv = torch.zeros(n, 3, D, dtype=torch.bfloat16)
    qkv[:, 2] = rows
    cache, cos = Kv8Cache.empty(1, 1, n, D, dev), torch.zeros(n, D, device=dev)
    rope_append_prompt_kv8(qkv.flatten(1).to(dev), torch.tensor([0, n], dtype=torch.int32, device=dev), n, torch.zeros(1, dtype=torch.int64, device=dev),
                           cos, cos, torch.empty(n, D, device=dev, dtype=torch.bfloat16), None, cache, 1)
    codes, s = quantise(rows[None])
    assert torch.equal(cache.v_scale[0, 0].cpu().double(), s[0])
    assert torch.equal(cache.v[0, 0].cpu(), codes[0])
    assert bool(codes.any())


@pytest.mark.parametrize("n", [1 << 10, 1 << 17, 1 << 20])
@pytest.mark.parametrize("spread", [0.01, 1.0])
def test_values_that_cancel(n, spread):
    """Pairs of positions with the same key and values of opposite sign: the result is what the arithmetic leaves.  Codes enter as
    1152 + code, and 1152 times the sum of the weights is taken off: three sums (the weights', two products') that hold numbers of up to
    1279 times it, each cut to 24 bits, 3 * 2^-23 * 1279 < 2^-11 of a code's step, whatever the length; fp32 sums over the blocks and the
    output's rounding add 2^-8 of that at most."""
    from helix_substrate_b200.kv8 import Kv8Cache, attn_decode_kv8
    dev, nq, D = _dev(), 8, 128
    cache = Kv8Cache.empty(1, 1, n, D, dev)
    g = torch.Generator(device=dev).manual_seed(n)
    v, k = (torch.randint(-127, 128, (n // 2, D), device=dev, generator=g, dtype=torch.int8) for _ in range(2))
    cache.v[0, 0, 0::2], cache.v[0, 0, 1::2] = v, -v
    cache.k[0, 0, 0::2], cache.k[0, 0, 1::2] = k, k
    cache.v_scale.fill_(1.0)
    cache.k_scale.fill_(1.0)
    q, out = torch.randn(1, nq * D, device=dev, generator=g).bfloat16(), torch.empty(1, nq * D, device=dev, dtype=torch.bfloat16)
    attn_decode_kv8(q, cache, torch.tensor([n - 1], device=dev), out, nq, spread / 73 / D ** 0.5)         # (scores of that size)
    assert float(out.double().abs().max()) <= 2.0 ** -11 * (1 + 2.0 ** -8)
