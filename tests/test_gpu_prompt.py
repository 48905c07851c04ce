"""Attention of whole prompts against plain 64-bit arithmetic: packed sequences, slabs of a cache, lengths around
the tiles, grouped heads that do not divide them, rows that see nothing, NaNs where nobody looks."""

import pytest
import torch

from conftest import rel_l2
from kv8_ref import attention

pytestmark = pytest.mark.gpu

# Each weight is rounded to bf16 (2^-9 of it at most half an ulp: eps / 2 = 2^-8 as a bound), the output once more: the two
# together stay below 2^-7; rms over random mantissas, sqrt(2) * 2^-9.2.  Bound of rel-L2: 2^-8.
TOL = 2.0 ** -8


def _dev():
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _no_wait_gave_up():
    """Every wait in the kernels is bounded; none may have run out."""
    yield
    from helix_substrate_b200.packed import _status_word
    assert int(_status_word(_dev())) == 0


def _want(q, k, v, scale, causal):
    lq, lk = q.shape[0], k.shape[0]
    seen = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(lk - lq)
    return attention(q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), scale, seen).transpose(0, 1)


def _compare(got, want, what):
    nan = want.isnan()
    assert torch.equal(nan, got.isnan()), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf].to(got.dtype)), what
    fine = ~(nan | inf)
    got, want = got.double()[fine], want[fine]
    if not want.numel() or not bool(want.any()):
        assert not bool(got.any()), what
        return
    assert rel_l2(got.cpu(), want.cpu()) < TOL, (what, rel_l2(got.cpu(), want.cpu()))
    big = (got - want).abs() / want.abs().clamp_min(float(want.pow(2).mean().sqrt()))
    assert float(big.max()) < 2.0 ** -5, (what, float(big.max()))


@pytest.mark.parametrize("nq,nkv,D", [(28, 4, 128), (4, 2, 64), (40, 8, 128), (3, 3, 128), (8, 1, 64), (5, 1, 80), (6, 2, 16), (64, 1, 128), (9, 3, 72), (2, 1, 8)])
@pytest.mark.parametrize("lens", [[1], [37, 0, 1, 256, 129], [700, 3], [127, 128, 300]])
def test_packed(nq, nkv, D, lens):
    """Views of one projection's output, sequences of every kind, two rows that belong to none."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T = _dev(), sum(lens)
    g = torch.Generator(device=dev).manual_seed(T + nq)
    qkv = torch.randn(T + 2, nq + 2 * nkv, D, device=dev, generator=g).bfloat16()
    qkv[T:] = float("nan")
    q, k, v = qkv.split([nq, nkv, nkv], 1)
    cu = [sum(lens[:s]) for s in range(len(lens) + 1)]
    for causal in (True, False):
        out = torch.full((T + 2, nq, D), 7.0, device=dev, dtype=torch.bfloat16)
        attn_prompt(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device=dev), max(lens), D ** -0.5, causal=causal)
        for a, b in zip(cu, cu[1:]):
            if b > a:
                _compare(out[a:b], _want(q[a:b], k[a:b], v[a:b], D ** -0.5, causal), (causal, a, b))
        assert bool((out[T:] == 7).all())
        again = torch.full_like(out, 7.0)
        attn_prompt(q, k, v, again, torch.tensor(cu, dtype=torch.int32, device=dev), max(lens) + 500, D ** -0.5, causal=causal)
        assert torch.equal(out, again), "the same bits, whatever max_q"


@pytest.mark.parametrize("nq,nkv,D", [(28, 4, 128), (4, 2, 64), (3, 1, 40)])
@pytest.mark.parametrize("lens,keys", [([5, 64, 1, 130], [1000, 64, 513, 131]), ([300, 10], [299, 4]), ([20], [0]), ([256, 3], [2048, 1])])
def test_slabs_and_more_or_fewer_keys_than_queries(nq, nkv, D, lens, keys):
    """Keys in a cache's slabs, rows past each length NaN; fewer keys than queries leave the first queries nothing to see."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T, S, rows = _dev(), sum(lens), len(lens), max(keys) + 70
    g = torch.Generator(device=dev).manual_seed(T + D)
    q = torch.randn(T, nq + 1, D, device=dev, generator=g).bfloat16()[:, :nq]
    kc = torch.randn(S, nkv, rows, D, device=dev, generator=g).bfloat16()
    vc = torch.randn(S, nkv + 2, rows, D, device=dev, generator=g).bfloat16()[:, 1: nkv + 1]
    for s, n in enumerate(keys):
        kc[s, :, n:] = float("nan")
        vc[s, :, n:] = float("inf")
    cu = [sum(lens[:s]) for s in range(S + 1)]
    cu_d, len_d = torch.tensor(cu, dtype=torch.int32, device=dev), torch.tensor(keys, device=dev)
    for causal in (True, False):
        out = torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16)
        attn_prompt(q, kc, vc, out, cu_d, max(lens), 0.3, k_len=len_d, causal=causal)
        for s, (a, b) in enumerate(zip(cu, cu[1:])):
            n = keys[s]
            _compare(out[a:b], _want(q[a:b], kc[s, :, :n].transpose(0, 1), vc[s, :, :n].transpose(0, 1), 0.3, causal), (causal, s))
        # the same keys, packed
        if sum(keys):
            kp = torch.cat([kc[s, :, :n].transpose(0, 1) for s, n in enumerate(keys)]).contiguous()
            vp = torch.cat([vc[s, :, :n].transpose(0, 1) for s, n in enumerate(keys)]).contiguous()
            cu_k = torch.tensor([sum(keys[:s]) for s in range(S + 1)], dtype=torch.int32, device=dev)
            packed = torch.empty_like(out)
            attn_prompt(q, kp, vp, packed, cu_d, max(lens), 0.3, cu_k=cu_k, causal=causal)
            assert torch.equal(out, packed)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [0, 5, 127, 128, 200, 299])
def test_infinities_and_nans_reach_only_the_rows_that_see_them(D, at):
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, T = _dev(), 14, 2, 300
    g = torch.Generator(device=dev).manual_seed(at)
    q, k, v = (torch.randn(T, n, D, device=dev, generator=g).bfloat16() for n in (nq, nkv, nkv))
    v[at, 0, 3], v[at, 0, 4], v[at, 1, 0] = float("inf"), float("nan"), float("-inf")
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    out = torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16)
    attn_prompt(q, k, v, out, cu, T, D ** -0.5)
    _compare(out, _want(q, k, v, D ** -0.5, True), at)
    v.nan_to_num_(0.0, 0.0, 0.0)
    k[at, 1, 2] = float("nan")
    attn_prompt(q, k, v, out, cu, T, D ** -0.5)
    want = _want(q, k, v, D ** -0.5, True)
    want[at:, 7:] = float("nan")
    _compare(out, want, ("key", at))


@pytest.mark.parametrize("case", ["growing", "peaked", "huge scores", "equal", "lowest"])
def test_running_softmax(case):
    """Scores that grow along the sequence (the reference point moves at every tile), one key that takes all, scores of 1e5, equal
    keys, and rows whose scores are the type's lowest."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, T, D = _dev(), 6, 2, 1000, 64
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v = (torch.randn(T, n, D, device=dev, generator=g) for n in (nq, nkv, nkv))
    scale = D ** -0.5
    if case == "growing":
        q, k = q.abs(), k.abs() * torch.linspace(0.1, 12, T, device=dev)[:, None, None]
    elif case == "peaked":
        k[333] = 20 * k[333].sign()
        q = 4 * k[333, :1].sign() + 0.1 * q
    elif case == "huge scores":
        q, k = q * 200, k * 200
    elif case == "equal":
        k = torch.ones_like(k)
    else:
        q, k, scale = torch.full_like(q, 1e18), torch.full_like(k, -3e18), 1.0
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    out = torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16)
    attn_prompt(q, k, v, out, torch.tensor([0, T], dtype=torch.int32, device=dev), T, scale)
    _compare(out, _want(q, k, v, scale, True), case)


def test_offsets_past_32_bits_and_a_stream_of_its_own():
    """Slabs whose second one lies past 2^31 elements; a call on another stream than the one the inputs were made on."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D, rows = _dev(), 4, 2, 128, 1 << 22
    kc = torch.empty(3, nkv, rows, D, device=dev, dtype=torch.bfloat16)
    vc = torch.empty_like(kc)
    g = torch.Generator(device=dev).manual_seed(4)
    n = 200
    for c in (kc, vc):
        c[:, :, :n] = torch.randn(3, nkv, n, D, device=dev, generator=g).bfloat16()
    q = torch.randn(3 * 40, nq, D, device=dev, generator=g).bfloat16()
    cu = torch.tensor([0, 40, 80, 120], dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attn_prompt(q, kc, vc, out, cu, 40, D ** -0.5, k_len=torch.tensor([n, n, n], device=dev))
    torch.cuda.current_stream().wait_stream(side)
    for s in range(3):
        _compare(out[40 * s: 40 * s + 40], _want(q[40 * s: 40 * s + 40], kc[s, :, :n].transpose(0, 1), vc[s, :, :n].transpose(0, 1), D ** -0.5, True), s)


def test_captured_and_replayed():
    """Lengths are read on the device: a captured call follows them."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D, T = _dev(), 28, 4, 128, 400
    g = torch.Generator(device=dev).manual_seed(6)
    q, k, v = (torch.randn(T, n, D, device=dev, generator=g).bfloat16() for n in (nq, nkv, nkv))
    cu = torch.tensor([0, 100, T], dtype=torch.int32, device=dev)
    out = torch.zeros(T, nq, D, device=dev, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        attn_prompt(q, k, v, out, cu, T, D ** -0.5)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            attn_prompt(q, k, v, out, cu, T, D ** -0.5)
    for mid in (100, 0, 333):
        cu[1] = mid
        graph.replay()
        want = torch.zeros_like(out)
        attn_prompt(q, k, v, want, cu, T, D ** -0.5)
        assert torch.equal(out, want)


def test_prompt_refuses():
    from helix_substrate_b200 import _lib
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T, nq, nkv, D = _dev(), 10, 4, 2, 64
    bf = lambda *s: torch.zeros(*s, device=dev, dtype=torch.bfloat16)       # noqa: E731
    q, k, v, out = bf(T, nq, D), bf(T, nkv, D), bf(T, nkv, D), bf(T, nq, D)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    n1 = torch.tensor([5], device=dev)
    bad = [
        (TypeError, lambda: attn_prompt(q.half(), k, v, out, cu, T, 0.1)),
        (TypeError, lambda: attn_prompt(q.cpu(), k, v, out, cu, T, 0.1)),
        (TypeError, lambda: attn_prompt(q, k.transpose(0, 2), v, out, cu, T, 0.1)),
        (TypeError, lambda: attn_prompt(q, k, v[:, :1], out, cu, T, 0.1)),
        (TypeError, lambda: attn_prompt(q, k, v, out[:5], cu, T, 0.1)),
        (TypeError, lambda: attn_prompt(q, k, v, out, cu.long(), T, 0.1)),
        (TypeError, lambda: attn_prompt(q, k, v, out, cu, T, 0.1, k_len=n1)),
        (ValueError, lambda: attn_prompt(q, k, v, out, cu, T, 0.1, cu_k=cu, k_len=n1)),
        (ValueError, lambda: attn_prompt(q, k[:5], v[:5], out, cu, T, 0.1)),
        (ValueError, lambda: attn_prompt(q[:, :3], k, v, out[:, :3], cu, T, 0.1)),
        (ValueError, lambda: attn_prompt(q, k, v, out, cu[:1], T, 0.1)),
        (ValueError, lambda: attn_prompt(q, k, v, out, cu, -1, 0.1)),
        (_lib.HxqError, lambda: attn_prompt(q, k, v, out, cu, T, 0.0)),
        (_lib.HxqError, lambda: attn_prompt(q, k, v, out, cu, T, float("nan"))),
        (_lib.HxqError, lambda: attn_prompt(bf(T, nq, 136), bf(T, nkv, 136), bf(T, nkv, 136), bf(T, nq, 136), cu, T, 0.1)),
        (_lib.HxqError, lambda: attn_prompt(bf(T, nq, D + 4)[..., :D], k, v, out, cu, T, 0.1)),
        (_lib.HxqError, lambda: attn_prompt(bf(T, 65, D), bf(T, 1, D), bf(T, 1, D), bf(T, 65, D), cu, T, 0.1)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    assert attn_prompt(q[:0], k[:0], v[:0], out[:0], torch.zeros(2, dtype=torch.int32, device=dev), 0, 0.1).shape[0] == 0


@pytest.mark.parametrize("nq,nkv,D", [(28, 4, 128), (4, 2, 64), (9, 3, 72), (64, 1, 128)])
@pytest.mark.parametrize("lens,keys", [([1], [5000]), ([16], [513]), ([7], [512]), ([130], [1025]), ([3, 40], [4097, 90]), ([2, 1, 1], [1600, 0, 7]), ([700], [1300])])
def test_few_queries_before_many_keys(nq, nkv, D, lens, keys):
    """Where the keys are shared out among thread blocks; a longer slab, or a larger max_q, changes no bit."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T, S, rows = _dev(), sum(lens), len(lens), max(keys) + 9
    g = torch.Generator(device=dev).manual_seed(T + D)
    q = torch.randn(T, nq, D, device=dev, generator=g).bfloat16()
    kc = torch.randn(S, nkv, rows, D, device=dev, generator=g).bfloat16()
    vc = torch.randn(S, nkv, rows, D, device=dev, generator=g).bfloat16()
    for s, n in enumerate(keys):
        kc[s, :, n:], vc[s, :, n:] = float("nan"), float("inf")
    longer = [torch.cat([c, torch.full((S, nkv, 20000, D), float("nan"), device=dev, dtype=torch.bfloat16)], 2) for c in (kc, vc)]
    cu = [sum(lens[:s]) for s in range(S + 1)]
    cu_d, len_d = torch.tensor(cu, dtype=torch.int32, device=dev), torch.tensor(keys, device=dev)
    for causal in (True, False):
        out, again = (torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
        attn_prompt(q, kc, vc, out, cu_d, max(lens), 0.2, k_len=len_d, causal=causal)
        attn_prompt(q, *longer, again, cu_d, max(lens) + 300, 0.2, k_len=len_d, causal=causal)
        assert torch.equal(out, again)
        for s, (a, b) in enumerate(zip(cu, cu[1:])):
            n = keys[s]
            _compare(out[a:b], _want(q[a:b], kc[s, :, :n].transpose(0, 1), vc[s, :, :n].transpose(0, 1), 0.2, causal), (causal, s))


@pytest.mark.parametrize("at", [0, 700, 2990, 2999])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_values_in_a_share_of_the_keys(at, bad):
    """Ten queries behind 2990 keys, the keys in shares: a bad value of V reaches its dimension, one of K the whole row."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D, T, n = _dev(), 14, 2, 128, 10, 3000
    g = torch.Generator(device=dev).manual_seed(at)
    q = torch.randn(T, nq, D, device=dev, generator=g).bfloat16()
    kc, vc = (torch.randn(1, nkv, n, D, device=dev, generator=g).bfloat16() for _ in range(2))
    vc[0, 1, at, 5] = bad
    cu, k_len = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.tensor([n], device=dev)
    out = torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16)
    attn_prompt(q, kc, vc, out, cu, T, D ** -0.5, k_len=k_len)
    _compare(out, _want(q, kc[0].transpose(0, 1), vc[0].transpose(0, 1), D ** -0.5, True), at)
    vc.nan_to_num_(0.0, 0.0, 0.0)
    kc[0, 0, at, 2] = float("nan")
    attn_prompt(q, kc, vc, out, cu, T, D ** -0.5, k_len=k_len)
    _compare(out, _want(q, kc[0].transpose(0, 1), vc[0].transpose(0, 1), D ** -0.5, True), at)


@pytest.mark.parametrize("nq,nkv,D,lens", [(28, 4, 128, [900, 37, 1, 300]), (4, 2, 64, [2000])])
def test_the_same_bits_every_time(nq, nkv, D, lens):
    """Rows whose maxima keep growing, so that outputs are rescaled up to the last step: sixty calls at different moments."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T = _dev(), sum(lens)
    g = torch.Generator(device=dev).manual_seed(T)
    q, k, v = (torch.randn(T, n, D, device=dev, generator=g).bfloat16() for n in (nq, nkv, nkv))
    q = q.abs()
    k *= torch.linspace(0.0, 40.0, T, device=dev)[:, None, None].bfloat16()
    k.abs_()
    cu = torch.tensor([sum(lens[:s]) for s in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    outs = [torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16) for _ in range(60)]
    for o in outs:
        attn_prompt(q, k, v, o, cu, max(lens), D ** -0.5)
    assert all(torch.equal(outs[0], o) for o in outs)
    a, b = int(cu[0]), int(cu[1])
    _compare(outs[0][a:b], _want(q[a:b], k[a:b], v[a:b], D ** -0.5, True), "the first")


@pytest.mark.parametrize("nq,nkv,D", [(128, 4, 128), (128, 4, 64), (112, 16, 72)])
def test_many_tiles(nq, nkv, D):
    """So many rows that thread blocks take two tiles each; a sequence by itself, one tile each, gives the same bits."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, lens = _dev(), [800, 37, 0, 1, 256, 129, 300]
    T = sum(lens)
    g = torch.Generator(device=dev).manual_seed(D)
    q = torch.randn(T, nq, D, device=dev, generator=g).bfloat16()
    k, v = (torch.randn(T, nkv, D, device=dev, generator=g).bfloat16() for _ in range(2))
    v[1000, 1, 3] = float("inf")
    cu = [sum(lens[:s]) for s in range(len(lens) + 1)]
    for causal in (True, False):
        out = torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16)
        attn_prompt(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device=dev), max(lens), D ** -0.5, causal=causal)
        for a, b in zip(cu, cu[1:]):
            if b == a:
                continue
            _compare(out[a:b], _want(q[a:b], k[a:b], v[a:b], D ** -0.5, causal), (causal, a, b))
            alone = torch.empty(b - a, nq, D, device=dev, dtype=torch.bfloat16)
            attn_prompt(q[a:b], k[a:b], v[a:b], alone, torch.tensor([0, b - a], dtype=torch.int32, device=dev), b - a, D ** -0.5, causal=causal)
            assert torch.equal(alone.view(torch.int16), out[a:b].view(torch.int16)), (causal, a, b)


@pytest.mark.parametrize("n", [31, 33, 128, 129, 1000, 3000])
def test_many_sequences(n):
    """Around the numbers that a warp's lanes hold, most of them short, one long, some empty."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D = _dev(), 6, 2, 64
    lens = [(7 * s) % 23 for s in range(n)]
    lens[n * 4 // 7] = 500
    T = sum(lens)
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v = (torch.randn(T, n, D, device=dev, generator=g).bfloat16() for n in (nq, nkv, nkv))
    cu = [sum(lens[:s]) for s in range(len(lens) + 1)]
    out = torch.full((T, nq, D), 7.0, device=dev, dtype=torch.bfloat16)
    attn_prompt(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device=dev), max(lens), 0.125)
    want = torch.cat([_want(q[a:b], k[a:b], v[a:b], 0.125, True) for a, b in zip(cu, cu[1:]) if b > a])
    _compare(out, want, "all")


def test_one_slab_seen_by_all():
    """Five sequences over the same 300 rows (a slab expanded, no copy), one query head's keys for both KV heads, outputs over the queries."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, S, n, D = _dev(), 5, 300, 64
    g = torch.Generator(device=dev).manual_seed(8)
    q = torch.randn(S * 7, 8, D, device=dev, generator=g).bfloat16()
    k, v = (torch.randn(1, 1, n, D, device=dev, generator=g).bfloat16().expand(S, 2, n, D) for _ in range(2))
    cu, k_len = torch.arange(S + 1, device=dev, dtype=torch.int32) * 7, torch.full((S,), n, device=dev)
    want = torch.cat([_want(q[7 * s: 7 * s + 7], k[s].transpose(0, 1), v[s].transpose(0, 1), 0.1, True) for s in range(S)])
    attn_prompt(q, k, v, q, cu, 7, 0.1, k_len=k_len)
    _compare(q, want, "in place")


def test_two_streams_at_once():
    """Whole items and shared ones on two streams, again and again: the bits of a call alone."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T = _dev(), 2000
    g = torch.Generator(device=dev).manual_seed(9)
    q, k, v = (torch.randn(T, n, 128, device=dev, generator=g).bfloat16() for n in (14, 2, 2))
    kc = torch.randn(1, 2, 9000, 128, device=dev, generator=g).bfloat16()
    cu, few, k_len = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.tensor([0, 16], dtype=torch.int32, device=dev), torch.tensor([9000], device=dev)

    def both():
        a, b = torch.empty_like(q), torch.empty_like(q[:16])
        attn_prompt(q, k, v, a, cu, T, 0.1)
        attn_prompt(q[:16], kc, kc, b, few, 16, 0.1, k_len=k_len)
        return a, b

    want = both()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for st in streams:
            with torch.cuda.stream(st):
                got.append(both())
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for pair in got for x, y in zip(pair, want))


@pytest.mark.parametrize("lens,keys", [([40], [40]), ([6], [3006])])
def test_scores_of_minus_infinity(lens, keys):
    """A key whose scores are -inf has no weight; a row that sees such keys alone is NaN, as 0 / 0 is; keys whole and in shares."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D, T, n = _dev(), 4, 2, 64, lens[0], keys[0]
    g = torch.Generator(device=dev).manual_seed(n)
    q = torch.rand(T, nq, D, device=dev, generator=g).bfloat16() + 0.5
    kc, vc = (torch.randn(1, nkv, n, D, device=dev, generator=g).bfloat16() for _ in range(2))
    kc[0, 0, : n - T + 1, 5] = float("-inf")          # all that the first query sees, in one head
    kc[0, 1, n - 3, 5] = float("-inf")
    cu, k_len = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.tensor([n], device=dev)
    out = torch.empty(T, nq, D, device=dev, dtype=torch.bfloat16)
    attn_prompt(q, kc, vc, out, cu, T, 0.1, k_len=k_len)
    s = torch.einsum("thd,hkd->htk", q.double(), kc[0].double().repeat_interleave(nq // nkv, 0)) * 0.1
    s = s.masked_fill(~torch.ones(T, n, device=dev).tril(n - T).bool(), float("-inf"))
    want = torch.einsum("htk,hkd->thd", s.softmax(-1), vc[0].double().repeat_interleave(nq // nkv, 0))
    assert bool(want[0, :2].isnan().all()) and int(want.isnan().sum()) == 2 * D
    _compare(out, want, "-inf")


def test_captured_with_what_reads_it():
    """Calls that share their keys out, each followed by a reader that comes in early: replays leave the bits of calls one by one."""
    from helix_substrate_b200.decode_ops import swiglu
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D, T, n, N = _dev(), 14, 2, 128, 12, 6000, 8
    g = torch.Generator(device=dev).manual_seed(10)
    k, v = (torch.randn(1, nkv, n, D, device=dev, generator=g).bfloat16() for _ in range(2))
    qs = [torch.randn(T, nq, D, device=dev, generator=g).bfloat16() for _ in range(N)]
    cu, k_len, gate = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.tensor([n], device=dev), torch.full((T, nq * D), 20.0, device=dev, dtype=torch.bfloat16)
    outs, reads = [torch.empty_like(q) for q in qs], [torch.empty_like(gate) for _ in qs]

    def call(i, wait):
        attn_prompt(qs[i], k, v, outs[i], cu, T, 0.1, k_len=k_len)
        if wait:
            torch.cuda.synchronize()
        swiglu(gate, outs[i].view(T, -1), reads[i])

    for i in range(N):
        call(i, True)
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


@pytest.mark.parametrize("S", [128, 129, 1000])
@pytest.mark.parametrize("lead", [64, 200, 5000])
@pytest.mark.parametrize("slabs", [False, True])
def test_rows_of_no_sequence_before_the_first(S, lead, slabs):
    """Sequences whose first does not start at row 0 (it is empty, too, where keys lie in slabs): rows of none stay as they are, and
    call after call gives the same bits."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D = _dev(), 14, 2, 64
    lens = [(7 * s) % 11 for s in range(S)]
    lens[0], lens[S // 2] = (0 if slabs else 3), 150
    T = sum(lens)
    g = torch.Generator(device=dev).manual_seed(S + lead)
    q = torch.randn(lead + T + 2, nq, D, device=dev, generator=g).bfloat16()
    q[:lead], q[lead + T:] = float("nan"), float("nan")
    cu = [lead + sum(lens[:s]) for s in range(S + 1)]
    cu_d = torch.tensor(cu, dtype=torch.int32, device=dev)
    if slabs:
        k, v = (torch.randn(S, nkv, 160, D, device=dev, generator=g).bfloat16() for _ in range(2))
        n = [9 + s % 150 for s in range(S)]
        kw = dict(k_len=torch.tensor(n, device=dev))
        keys = lambda t, s: t[s, :, : n[s]].transpose(0, 1)        # noqa: E731
    else:
        k, v = (torch.randn(lead + T + 2, nkv, D, device=dev, generator=g).bfloat16() for _ in range(2))
        k[:lead], v[:lead] = float("nan"), float("inf")
        kw = {}
        keys = lambda t, s: t[cu[s]: cu[s + 1]]        # noqa: E731
    outs = [torch.full((lead + T + 2, nq, D), 7.0, device=dev, dtype=torch.bfloat16) for _ in range(10)]
    for o in outs:
        attn_prompt(q, k, v, o, cu_d, 150, 0.125, **kw)
    out = outs[0]
    assert bool((out[:lead] == 7).all()) and bool((out[lead + T:] == 7).all())
    assert all(torch.equal(out, o) for o in outs)
    want = torch.cat([_want(q[cu[s]: cu[s + 1]], keys(k, s), keys(v, s), 0.125, True) for s in range(S) if lens[s]])
    _compare(out[lead: lead + T], want, "all")


def test_status_word_outlives_replays(monkeypatch):
    """The word is made outside a capture (a first call under one is refused) and no replay clears it."""
    from helix_substrate_b200 import packed
    from helix_substrate_b200.prompt_ops import attn_prompt, check_status
    monkeypatch.setattr(packed, "_status_words", {})
    dev, T = _dev(), 40
    q, k = (torch.randn(T, n, 64, device=dev).bfloat16() for n in (4, 2))
    cu, out = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            with pytest.raises(RuntimeError, match="capture"):
                attn_prompt(q, k, k, out, cu, T, 0.1)
        attn_prompt(q, k, k, out, cu, T, 0.1)
        assert check_status(dev) == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attn_prompt(q, k, k, out, cu, T, 0.1)
        packed._status_word(dev).fill_(-7)
        graph.replay()
        assert check_status(dev) == -7 == check_status("cuda:0")


@pytest.mark.parametrize("nq,nkv,D,lens,keys", [(28, 4, 128, [50, 3, 30], None), (128, 4, 64, [700, 37, 300, 900], None), (14, 2, 128, [40, 5], [6000, 5]),
                                                (8, 8, 64, [200], [9000])])
@pytest.mark.parametrize("max_q", [1, 4, 33])
def test_queries_past_max_q_are_left_alone(nq, nkv, D, lens, keys, max_q):
    """Sequences longer than max_q, tiles one to a thread block, two, and with their keys shared out: of each the first max_q queries are
    computed, as the first of all its queries, and no other row of out is touched."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, T, S = _dev(), sum(lens), len(lens)
    g = torch.Generator(device=dev).manual_seed(T + max_q)
    q = torch.randn(T, nq, D, device=dev, generator=g).bfloat16()
    cu = [sum(lens[:s]) for s in range(S + 1)]
    if keys is None:
        k, v = (torch.randn(T, nkv, D, device=dev, generator=g).bfloat16() for _ in range(2))
        kw, of = {}, lambda t, s: t[cu[s]: cu[s + 1]]
    else:
        k, v = (torch.randn(S, nkv, max(keys), D, device=dev, generator=g).bfloat16() for _ in range(2))
        kw, of = dict(k_len=torch.tensor(keys, device=dev)), lambda t, s: t[s, :, : keys[s]].transpose(0, 1)
    for causal in (True, False):
        out = torch.full((T, nq, D), 7.0, device=dev, dtype=torch.bfloat16)
        attn_prompt(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device=dev), max_q, 0.15, causal=causal, **kw)
        for s, (a, b) in enumerate(zip(cu, cu[1:])):
            m = min(max_q, b - a)
            _compare(out[a: a + m], _want(q[a:b], of(k, s), of(v, s), 0.15, causal)[:m], (causal, s))
            assert bool((out[a + m: b] == 7).all()), (causal, s)


@pytest.mark.parametrize("lens,keys", [([61, 9], None), ([700, 400], None), ([9, 3], [3000, 2])])
@pytest.mark.parametrize("loud", [30.0, 3e4])
def test_a_neighbours_scores_change_no_bit(lens, keys, loud):
    """Rows of one tile are other heads', other tokens' and other sequences': whatever the size of theirs, a row's bits stay."""
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, nq, nkv, D, T, S = _dev(), 8, 1, 64, sum(lens), len(lens)
    g = torch.Generator(device=dev).manual_seed(T)
    q = torch.randn(T, nq, D, device=dev, generator=g).bfloat16() * 3
    rows = T if keys is None else max(keys)
    k, v = (torch.randn(*((rows,) if keys is None else (S, nkv, rows)), *((nkv, D) if keys is None else (D,)), device=dev, generator=g).bfloat16() for _ in range(2))
    kw = {} if keys is None else dict(k_len=torch.tensor(keys, device=dev))
    cu = torch.tensor([0, lens[0], T], dtype=torch.int32, device=dev)
    out, other = torch.empty_like(q), torch.empty_like(q)
    attn_prompt(q, k, v, out, cu, max(lens), 1.0, **kw)
    q2 = q.clone()
    q2[:, 0] *= loud             # a head
    q2[::5] *= loud              # tokens
    q2[lens[0]:] *= loud         # the next sequence
    attn_prompt(q2, k, v, other, cu, max(lens), 1.0, **kw)
    same = (q2 == q).all(-1)
    assert bool(same.any()) and torch.equal(out[same], other[same])


@pytest.mark.parametrize("n", [2000, 6000])
@pytest.mark.parametrize("size", [500.0, 2000.0, 20000.0, 60000.0])
def test_reference_points_that_move_among_large_scores(n, size):
    """Scores about `size`, sixteen keys of them as heavy together as half of all, values that nearly cancel: weights count across a move
    of the reference point and across shares of the keys."""
    from math import log
    from helix_substrate_b200.prompt_ops import attn_prompt
    dev, D, T = _dev(), 64, 8
    g = torch.Generator(device=dev).manual_seed(n)
    q = torch.zeros(T, 1, D, device=dev)
    q[:, :, 0] = 256.0
    q[:, :, 1] = 1.0
    big = torch.tensor(size / 256, device=dev).bfloat16()
    k, v = torch.zeros(n, 1, D, device=dev), torch.randn(n, 1, D, device=dev, generator=g) * 0.01
    k[:, :, 0] = big.float()
    k[n // 2: n // 2 + 16, :, 1] = log(n / 2 / 16)
    v[: n // 2] += 1.0
    v[n // 2: n // 2 + 16] -= 1.0
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    out = torch.empty_like(q)
    attn_prompt(q, k, v, out, torch.tensor([0, T], dtype=torch.int32, device=dev), T, 1.0, cu_k=torch.tensor([0, n], dtype=torch.int32, device=dev), causal=False)
    want = _want(q, k, v, 1.0, False)
    # fp32 holds a score of `size` to 2^-24 size; weights are rounded to bf16 (2^-8), the output too; sums of |w v| / w are below 1.1
    assert float((out.double() - want).abs().max()) <= 1.1 * (2.0 ** -8 + size * 2.0 ** -23) + 2.0 ** -8
