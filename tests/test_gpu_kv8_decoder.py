"""The decoder on an 8-bit cache and with fused prompt attention: append, prompt attention, rows back and
single-token attention together, as a serving loop runs them."""

import pytest
import torch

from conftest import rel_l2

pytestmark = pytest.mark.gpu


def _dev():
    return torch.device("cuda:0")


def _pair(world=1, rank=0, batch=2, max_len=320, **kw):
    from helix_substrate_b200.qwen2_decode import Qwen2HxqDecoder, Qwen2Shape
    return Qwen2HxqDecoder(Qwen2Shape.tiny(), _dev(), batch=batch, max_len=max_len, rank=rank, world=world, **kw)


def _same_weights(first, *others):
    """Decoders to be compared share the first one's matrices: the encoder's k-means adds up in no fixed order, so two encodings of one
    weight differ in a few codes."""
    for m in others:
        m.layers = first.layers
    return (first, *others)


@pytest.mark.parametrize("fuse_proj", [True, False])
@pytest.mark.parametrize("chunk", [2048, 100, 64])
def test_prefill_and_steps(fuse_proj, chunk):
    """Prompt of 230 tokens in one piece or several, then steps over a block's end: fused prompt attention on the 16-bit cache agrees
    with the framework's operator to bf16 precision; the 8-bit cache differs by what 8 bits cost (rows are off by 1/254 of their
    block's largest value at most, about 1 % of a row's norm; a logit's error stays of that order)."""
    base, fused, q8 = _same_weights(_pair(fuse_proj=fuse_proj), _pair(fuse_proj=fuse_proj, prompt_attn="fused"), _pair(fuse_proj=fuse_proj, kv_bits=8))
    prompt = torch.randint(0, 1024, (2, 230), device=_dev(), generator=torch.Generator(device=_dev()).manual_seed(3))
    with torch.no_grad():
        logits = []
        for m in (base, fused, q8):
            for a in range(0, 230, chunk):
                b = min(a + chunk, 230)
                pos = torch.arange(a, b, device=_dev())
                out = m.forward_tokens(prompt[:, a:b], pos, pos, b)
            logits.append(out.float().cpu())
        assert rel_l2(logits[1], logits[0]) < 2e-2 and rel_l2(logits[2], logits[0]) < 5e-2
        assert rel_l2(fused.k_cache.float().cpu(), base.k_cache.float().cpu()) < 1e-2
        tok = logits[0].argmax(-1)[:, None].to(_dev())
        for i in range(230, 260):           # position 255 finishes a block
            p = torch.tensor([i], device=_dev())
            steps = [m.step_fused(tok, p).float().cpu() for m in (base, fused, q8)]
            assert rel_l2(steps[1], steps[0]) < 2e-2 and rel_l2(steps[2], steps[0]) < 5e-2, i
            tok = steps[0].argmax(-1)[:, None].to(_dev())


def test_the_cache_holds_the_rows_of_the_16_bit_one():
    """What the 8-bit cache of the first layer reads back is the 16-bit cache's rows to within half a code."""
    from helix_substrate_b200.kv8 import kv8_rows
    base, q8 = _same_weights(_pair(), _pair(kv_bits=8))
    prompt = torch.randint(0, 1024, (2, 200), device=_dev(), generator=torch.Generator(device=_dev()).manual_seed(4))
    base.prefill(prompt)
    q8.prefill(prompt, chunk=90)
    c = q8.kv8[0]
    k, v = (torch.empty(2, 2, 200, 64, device=_dev(), dtype=torch.bfloat16) for _ in range(2))
    kv8_rows(c, torch.tensor([200], device=_dev()), k, v)
    for got, want, scale in ((k, base.k_cache[0], c.k_scale), (v, base.v_cache[0], c.v_scale)):
        want = want[:, :, :200].float()
        assert torch.equal(got[:, :, 192:].float(), want[:, :, 192:]) or rel_l2(got[:, :, 192:].float().cpu(), want[:, :, 192:].cpu()) < 1e-2
        step = scale[:, :, :3].repeat_interleave(64, 2)[..., None]
        want = want[:, :, :192]
        # Half a code, and two bf16 roundings (the rotation's and the read's), 2^-8 of the value each.  The pieces' projections are
        # other calls (180 tokens and 400: another kernel), each rounded to bf16: x differs by 2 * 2^-8 of itself, which a rotation
        # turns into at most 2^-7 (|x0| + |x1|) <= 2^-7 sqrt(2) r, r the pair's length; and their fp32 sums of 256 products run
        # in another order: 2 * 256 * 2^-24 * |x| |w| with |x| = 16 (normalised rows), |w| < 0.5 (256 weights of 0.02): 2.5e-4.
        r = want.unflatten(-1, (2, 32)).square().sum(-2, keepdim=True).sqrt().expand(-1, -1, -1, 2, -1).flatten(-2)
        assert bool(((got[:, :, :192].float() - want).abs() <= 0.5 * step + 2.0 ** -7 * want.abs() + 2.0 ** -7 * 2 ** 0.5 * r + 2.5e-4).all())


@pytest.mark.parametrize("kv_bits,prompt_attn", [(8, "torch"), (16, "fused")])
def test_captured_greedy_decoding_equals_eager_steps(kv_bits, prompt_attn):
    m, n = _same_weights(_pair(kv_bits=kv_bits, prompt_attn=prompt_attn), _pair(kv_bits=kv_bits, prompt_attn=prompt_attn))
    prompt = torch.randint(0, 1024, (2, 120), device=_dev(), generator=torch.Generator(device=_dev()).manual_seed(5))
    with torch.no_grad():
        nxt, n_nxt = m.prefill(prompt), n.prefill(prompt)
        assert torch.equal(nxt, n_nxt)
        if kv_bits == 8:
            before = [t.clone() for c in m.kv8 for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail)]
        run, tok, pos = m.make_graphed_step(2)
        if kv_bits == 8:
            after = [t for c in m.kv8 for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail)]
            assert all(torch.equal(a, b) for a, b in zip(before, after)), "capturing leaves the cache as it is"
        else:
            n.k_cache.copy_(m.k_cache); n.v_cache.copy_(m.v_cache)
        for i in range(12):          # a block ends at position 127
            tok.copy_(nxt[:, None]); pos.fill_(120 + i)
            nxt = run().clone()
            n_nxt = n.step_fused(n_nxt[:, None], torch.tensor([120 + i], device=_dev())).argmax(-1)
            assert torch.equal(nxt, n_nxt), i


def test_sharded_decoder_on_an_8_bit_cache():
    from helix_substrate_b200.qwen2_decode import Qwen2HxqDecoder, Qwen2Shape, run_ranks_in_process
    dev = _dev()
    shp = Qwen2Shape(hidden=256, inter=640, layers=2, heads=14, kv_heads=2, head_dim=64, vocab=512)
    full = Qwen2HxqDecoder(shp, dev, batch=2, max_len=128, build="global", kv_bits=8)
    ranks = [Qwen2HxqDecoder(shp, dev, batch=2, max_len=128, rank=r, world=4, build="global", kv_bits=8) for r in range(4)]
    prompt = torch.randint(0, shp.vocab, (2, 70), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    pos = torch.arange(70, device=dev)
    with torch.no_grad():
        ref = full.forward_tokens(prompt, pos, pos, 70)
        outs = run_ranks_in_process([m.blocks_tokens(prompt, pos, pos, 70) for m in ranks])
        assert all(torch.equal(o, outs[0]) for o in outs) and rel_l2(outs[0].float().cpu(), ref.float().cpu()) < 3e-2
        tok, p1 = ref.argmax(-1)[:, None], torch.tensor([70], device=dev)
        ref = full.step_fused(tok, p1)
        outs = run_ranks_in_process([m.blocks_step(tok, p1, fp32_partials=True) for m in ranks])
        assert all(torch.equal(o, outs[0]) for o in outs) and rel_l2(outs[0].float().cpu(), ref.float().cpu()) < 3e-2


def test_run_decode_reports_the_cache():
    from helix_substrate_b200.qwen2_decode import run_decode
    for kw in (dict(kv_bits=8), dict(kv_bits=8, fill_cache=True), dict(prompt_attn="fused")):
        res = run_decode("tiny", [2, 1], 100, 6, _dev(), **kw)
        assert len(res) == 2 and all(r["tokens_valid"] and r["kv_bits"] == kw.get("kv_bits", 16) and r["prompt_attn"] == "fused" for r in res)


def test_decoder_refuses():
    with pytest.raises(ValueError, match="kv_bits"):
        _pair(kv_bits=4)
    with pytest.raises(ValueError, match="prompt_attn"):
        _pair(prompt_attn="other")
    with pytest.raises(ValueError, match="8-bit"):
        _pair(kv_bits=8).make_graphed_step(2, fused=False)


def test_run_decode_reports_a_wait_that_gave_up():
    from helix_substrate_b200 import _lib, packed
    from helix_substrate_b200.qwen2_decode import run_decode
    word = packed._status_word(_dev())
    assert run_decode("tiny", [1], 70, 3, _dev(), prompt_attn="fused")[0]["kernel_status_word"] == 0
    word.fill_(_lib.HXQ_E_TIMEOUT)
    try:
        assert run_decode("tiny", [1], 70, 3, _dev(), kv_bits=8)[0]["kernel_status_word"] == _lib.HXQ_E_TIMEOUT
    finally:
        word.zero_()
