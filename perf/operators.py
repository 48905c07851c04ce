"""Attention over prompts and over an 8-bit key/value cache, as timed cases.

Four operators of a decoder's attention, the way a serving loop calls them:

* ``prompt``: causal grouped-query attention of packed prompts of different lengths, or of a later piece of a
  prompt over the rows its cache already holds;
* ``append``: rotary embedding of new query and key heads and the append of keys and values to an 8-bit cache, for
  one token a sequence (``step``) or for packed prompts;
* ``decode``: single-query attention over the 8-bit cache;
* ``rows``: rows of the 8-bit cache back as bf16.

The 8-bit cache holds blocks of 64 positions, each with one scale for every KV head; the rows of a sequence's last,
unfinished block are kept in bf16 in a tail.  A scale is max(|x|) / 127 rounded up to bf16 (2**-126 at least), a code
is x / scale rounded to the nearest even integer.  The rotary embedding is rounded once, to bf16.

Head layouts are those of the benchmark's decoders (28 query and 4 KV heads, 40 and 8, of 128; 4 and 2 of 64) and
generic ones.  Queries, keys and values are N(0, 1) with a few louder key channels, as a projection's are.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 64            # positions with one scale
THETA = 1e6           # base of the rotary angles


def listed():
    return [
        # the smallest prompt: one short question to a small model
        dict(name="prompt_37", kind="prompt", nq=4, nkv=2, D=64, lens="37", hist="0"),
        # what a server packs into one call: an empty slot, single tokens, a long prompt among short ones
        dict(name="prompt_packed", kind="prompt", nq=28, nkv=4, D=128, lens="1,733,64,2048,0,7,311,129,1500", hist="0,0,0,0,0,0,0,0,0"),
        # a later piece of two prompts, over the rows that their caches hold already
        dict(name="prompt_chunk", kind="prompt", nq=40, nkv=8, D=128, lens="512,301", hist="6000,2111"),
        # one long document
        dict(name="prompt_16384", kind="prompt", nq=28, nkv=4, D=128, lens="16384", hist="0"),
        # one token's rotary embedding and append, one sequence
        dict(name="append_step_1", kind="append", step=True, nq=28, nkv=4, D=128, max_len=4160, pos="2047"),
        # the same for a busy server, where every sequence finishes a block at this token
        dict(name="append_step_32", kind="append", step=True, nq=28, nkv=4, D=128, max_len=4160, pos=",".join(str(64 * (2 * i + 1) - 1) for i in range(32))),
        # packed prompts: fresh ones and one that continues in the middle of a block
        dict(name="append_prompt", kind="append", step=False, nq=28, nkv=4, D=128, max_len=8320, pos="0,100,0", lens="6000,1000,1191"),
        # one token behind a 2048-token context
        dict(name="decode_1", kind="decode", nq=28, nkv=4, D=128, max_len=2240, pos="2047"),
        # a batch of sequences of many lengths, an idle slot among them
        dict(name="decode_32", kind="decode", nq=28, nkv=4, D=128, max_len=4160, pos="-1," + ",".join(str(131 * i) for i in range(1, 32))),
        # two very long contexts
        dict(name="decode_long", kind="decode", nq=40, nkv=8, D=128, max_len=131072, pos="131071,100000"),
        # a short context back as bf16 for the next piece of its prompt, and long ones
        dict(name="rows_500", kind="rows", nkv=4, D=128, max_len=4160, lens="500"),
        dict(name="rows_long", kind="rows", nkv=8, D=128, max_len=32768, lens="32768,20001,0,9999"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(28, 4), (40, 8), (4, 2), (8, 8), (8, 1), (14, 2), (6, 2), (3, 1)]


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "append", "append", "decode", "decode", "rows"])
    nq, nkv = rng.choice(_HEADS)
    D = rng.choice([128, 128, 64])
    if kind == "prompt":
        n = rng.choice([1, 1, 2, 5, 9])
        lens = [_log(rng, 1, 10000 // n) for _ in range(n)]
        hist = [rng.choice([0, _log(rng, 1, 4000)]) for _ in lens] if rng.random() < 0.4 else [0] * n
        return dict(kind=kind, nq=nq, nkv=nkv, D=D, lens=_text(lens), hist=_text(hist))
    if kind == "append":
        n = rng.choice([1, 2, 4, 17, 48])
        if rng.random() < 0.5:
            last = rng.random() < 0.5        # every sequence finishes its block, or none does
            pos = [64 * rng.randrange(0, 60) + (63 if last else rng.randrange(0, 63)) for _ in range(n)]
            return dict(kind=kind, step=True, nq=nq, nkv=nkv, D=D, max_len=4160, pos=_text(pos))
        n = min(n, 4)
        lens = [_log(rng, 1, 8000 // n) for _ in range(n)]
        pos = [rng.choice([0, rng.randrange(0, 200)]) for _ in lens]
        return dict(kind=kind, step=False, nq=nq, nkv=nkv, D=D, max_len=8320, pos=_text(pos), lens=_text(lens))
    if kind == "decode":
        n = _log(rng, 1, 64)
        longest = _log(rng, 64, 120000 // n + 64)
        pos = [rng.randrange(-1, longest) for _ in range(n)]
        pos[rng.randrange(n)] = longest - 1
        return dict(kind=kind, nq=nq, nkv=nkv, D=D, max_len=BLOCK * (longest // BLOCK + 1 + rng.randrange(0, 8)), pos=_text(pos))
    n = rng.choice([1, 2, 8])
    longest = _log(rng, 1, 60000 // n)
    lens = [rng.randrange(0, longest + 1) for _ in range(n)]
    lens[0] = longest
    return dict(kind=kind, nkv=nkv, D=D, max_len=BLOCK * (longest // BLOCK + 1), lens=_text(lens))


def _text(v):
    return ",".join(str(int(x)) for x in v)


def _ints(text):
    return [int(x) for x in text.split(",")]


def _pairs(lens, hist):
    """(query, key) pairs of causal attention behind ``hist`` earlier rows."""
    return sum(n * h + n * (n + 1) // 2 for n, h in zip(lens, hist))


def work(case):
    D, nkv = case["D"], case["nkv"]
    if case["kind"] == "prompt":
        lens, hist = _ints(case["lens"]), _ints(case["hist"])
        keys = sum(n + h for n, h in zip(lens, hist) if n)
        return {"bytes": 2 * 2 * D * (sum(lens) * case["nq"] + keys * nkv), "flops": 4 * D * case["nq"] * _pairs(lens, hist)}
    if case["kind"] == "append":
        width = (case["nq"] + 2 * nkv) * D
        pos = _ints(case["pos"])
        lens = [1] * len(pos) if case["step"] else _ints(case["lens"])
        old = sum(p % BLOCK for p, n in zip(pos, lens) if p % BLOCK + n >= BLOCK)       # rows of the tail that a finished block takes in
        whole = sum((p + n) // BLOCK - p // BLOCK for p, n in zip(pos, lens))
        rest = sum(min(n, (p + n) % BLOCK) for p, n in zip(pos, lens))
        k_rows = 0 if case["step"] else sum(lens)
        return {"bytes": 2 * sum(lens) * width + 2 * 2 * old * nkv * D + 2 * sum(lens) * case["nq"] * D + 2 * k_rows * nkv * D
                         + 2 * whole * nkv * (BLOCK * D + 4) + 2 * 2 * rest * nkv * D + 2 * 4 * D * sum(lens),
                "flops": 3 * sum(lens) * (case["nq"] + nkv) * D + 2 * 2 * whole * BLOCK * nkv * D}
    lens = [p + 1 for p in _ints(case["pos"])] if case["kind"] == "decode" else _ints(case["lens"])
    whole, rest = sum(n // BLOCK for n in lens), sum(n % BLOCK for n in lens)
    cache = 2 * nkv * (whole * (BLOCK * D + 4) + rest * D * 2)
    if case["kind"] == "decode":
        return {"bytes": cache + 2 * 2 * len(lens) * case["nq"] * D, "flops": 4 * D * case["nq"] * sum(lens)}
    return {"bytes": cache + 2 * 2 * nkv * D * sum(lens), "flops": 2 * nkv * D * sum(lens)}


# ---------------------------------------------------------------------------------------------------- inputs

def _rand(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _loud(gen, nkv, D):
    return torch.exp(0.5 * _rand(gen, nkv, D))         # gain of each key channel


def _tables(max_len, D):
    inv = 1.0 / (THETA ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
    ang = torch.arange(max_len, device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
    both = torch.cat([ang, ang], -1)
    return both.cos().float(), both.sin().float()


def _filled_cache(gen, B, nkv, max_len, D):
    """An 8-bit cache of random rows, and its tails."""
    gain = _loud(gen, nkv, D)
    c = {}
    for name in ("k", "v"):
        codes = torch.empty(B, nkv, max_len, D, device=DEV, dtype=torch.int8)
        scale = torch.empty(B, nkv, max_len // BLOCK, device=DEV)
        for b in range(B):
            x = _rand(gen, nkv, max_len, D)
            x = (x * gain[:, None] if name == "k" else x).bfloat16()
            codes[b], scale[b] = _quantise(x)
        tail = _rand(gen, B, nkv, BLOCK, D)
        c[name], c[name + "_scale"] = codes, scale
        c[name + "_tail"] = (tail * gain[:, None] if name == "k" else tail).bfloat16()
    return c


def _quantise(x):
    """bf16 [nkv, rows, D], whole blocks -> codes int8 of that shape, scales [nkv, rows / 64]."""
    xb = x.float().unflatten(1, (-1, BLOCK))
    s = xb.abs().amax((-1, -2)) / 127.0
    s = ((s.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32).clamp_min(2.0 ** -126)      # up to bf16
    return torch.round(xb / s[..., None, None]).to(torch.int8).flatten(1, 2), s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    D, nkv = case["D"], case["nkv"]
    s = dict(case)
    dev = lambda v, t: torch.tensor(v, device=DEV, dtype=t)        # noqa: E731
    if case["kind"] == "prompt":
        nq, lens, hist = case["nq"], _ints(case["lens"]), _ints(case["hist"])
        T, gain = sum(lens), _loud(gen, nkv, D)
        s.update(lens=lens, hist=hist, scale=D ** -0.5, out=torch.zeros(T, nq, D, device=DEV, dtype=torch.bfloat16))
        s["cu"] = dev([sum(lens[:i]) for i in range(len(lens) + 1)], torch.int32)
        if any(hist):      # keys and values in the cache's rows
            rows = BLOCK * ((max(n + h for n, h in zip(lens, hist)) + BLOCK - 1) // BLOCK)
            s["q"] = _rand(gen, T, nq, D).bfloat16()
            s["k"] = (_rand(gen, len(lens), nkv, rows, D) * gain[:, None]).bfloat16()
            s["v"] = _rand(gen, len(lens), nkv, rows, D).bfloat16()
            s["k_len"] = dev([n + h for n, h in zip(lens, hist)], torch.int64)
        else:              # all three in the projection's output
            qkv = _rand(gen, T, nq + 2 * nkv, D)
            qkv[:, nq: nq + nkv] *= gain
            s["q"], s["k"], s["v"] = qkv.bfloat16().split([nq, nkv, nkv], 1)
            s["k_len"] = None
        return s
    if case["kind"] == "rows":
        lens = _ints(case["lens"])
        s.update(lens=lens, length=dev(lens, torch.int64), cache=_filled_cache(gen, len(lens), nkv, case["max_len"], D))
        for name in ("k_out", "v_out"):
            s[name] = torch.zeros(len(lens), nkv, max(lens), D, device=DEV, dtype=torch.bfloat16)
        return s
    nq, pos = case["nq"], _ints(case["pos"])
    B = len(pos)
    s["cache"] = _filled_cache(gen, B, nkv, case["max_len"], D)
    s["positions"], s["pos"] = pos, dev(pos, torch.int64)
    if case["kind"] == "decode":
        s.update(q=_rand(gen, B, nq * D).bfloat16(), out=torch.empty(B, nq * D, device=DEV, dtype=torch.bfloat16), scale=D ** -0.5)
        return s
    lens = [1] * B if case["step"] else _ints(case["lens"])
    T = sum(lens)
    qkv = _rand(gen, T, nq + 2 * nkv, D)
    qkv[:, nq: nq + nkv] *= _loud(gen, nkv, D)
    s.update(lens=lens, qkv=qkv.bfloat16().flatten(1), q_out=torch.zeros(T, nq * D, device=DEV, dtype=torch.bfloat16),
             k_out=None if case["step"] else torch.zeros(T, nkv, D, device=DEV, dtype=torch.bfloat16),
             cu=dev([sum(lens[:i]) for i in range(B + 1)], torch.int32))
    s["cos"], s["sin"] = _tables(case["max_len"], D)
    s["before"] = {n: s["cache"][n].clone() for n in ("k_tail", "v_tail")}
    # the blocks that this call finishes: (sequence, block)
    done = [(b, j) for b, (p, n) in enumerate(zip(pos, lens)) for j in range(p // BLOCK, (p + n) // BLOCK)]
    s["done"] = tuple(dev([d[i] for d in done], torch.int64) for i in (0, 1)) if done else None
    # a token's place: its sequence, its position; the last rows of each sequence, which stay in the tail
    seq = [b for b, n in enumerate(lens) for _ in range(n)]
    at = [p + i for p, n in zip(pos, lens) for i in range(n)]
    s["seq"], s["at"] = dev(seq, torch.int64), dev(at, torch.int64)
    ends = [p + n for p, n in zip(pos, lens)]
    keep = [t for t in range(T) if at[t] // BLOCK == ends[seq[t]] // BLOCK]
    s["keep"] = dev(keep, torch.int64)
    # for each finished block, where its rows come from: a row of this call, or of the tail (numbered behind them)
    first = [sum(lens[:b]) for b in range(B)]
    src = [[first[b] + j * BLOCK + i - pos[b] if j * BLOCK + i >= pos[b] else T + b * BLOCK + i for i in range(BLOCK)] for b, j in done]
    s["src"] = dev(src, torch.int64) if done else None
    return s


# ------------------------------------------------------------------------------------------------------- run

def run(s):
    return (_run_own if own else _run_plain)(s)


def _handle(s):
    from helix_substrate_b200.kv8 import Kv8Cache
    if "handle" not in s:                  # the cache object that a program keeps
        s["handle"] = Kv8Cache(**s["cache"])
    return s["handle"]


def _run_own(s):
    from helix_substrate_b200 import kv8, prompt_ops
    kind = s["kind"]
    if kind == "prompt":
        return prompt_ops.attn_prompt(s["q"], s["k"], s["v"], s["out"], s["cu"], max(s["lens"]), s["scale"], k_len=s["k_len"])
    cache = _handle(s)
    if kind == "decode":
        return kv8.attn_decode_kv8(s["q"], cache, s["pos"], s["out"], s["nq"], s["scale"])
    if kind == "rows":
        return kv8.kv8_rows(cache, s["length"], s["k_out"], s["v_out"])
    _restore(s)
    if s["step"]:
        kv8.rope_append_kv8(s["qkv"], s["pos"], s["cos"], s["sin"], s["q_out"], cache, s["nq"])
    else:
        kv8.rope_append_prompt_kv8(s["qkv"], s["cu"], max(s["lens"]), s["pos"], s["cos"], s["sin"], s["q_out"], s["k_out"], cache, s["nq"])
    return _appended(s)


def _restore(s):
    """The tails as they were before the call: a prompt that goes on behind its tail would find its own rows there."""
    if not s["step"]:
        for name, t in s["before"].items():
            s["cache"][name].copy_(t)


def _appended(s):
    """What an append leaves: the rotated heads, the tails, and the values of the blocks that it finished."""
    c = s["cache"]
    got = {"q": s["q_out"], "k_tail": c["k_tail"], "v_tail": c["v_tail"]}
    if s["k_out"] is not None:
        got["k"] = s["k_out"]
    if s["done"] is not None:
        b, j = s["done"]
        for name in ("k", "v"):
            got[name + "_blocks"] = c[name].unflatten(2, (-1, BLOCK))[b, :, j] * c[name + "_scale"][b, :, j, None, None]
    return got


def _rotate(x, cos, sin):
    """Rotate-half embedding of [T, heads, D] in 64 bits (a value next to a border of bf16 is rounded as it is), to bf16."""
    x, half = x.double(), x.shape[-1] // 2
    other = torch.cat([-x[..., half:], x[..., :half]], -1)
    return (x * cos[:, None].double() + other * sin[:, None].double()).bfloat16()


def _run_plain(s):
    kind = s["kind"]
    if kind == "prompt":
        return _plain_prompt(s)
    c, D, nkv = s["cache"], s["D"], s["nkv"]
    if kind == "append":
        _restore(s)
        T, nq = s["qkv"].shape[0], s["nq"]
        q, k, v = s["qkv"].view(T, nq + 2 * nkv, D).split([nq, nkv, nkv], 1)
        cos, sin = s["cos"][s["at"]], s["sin"][s["at"]]
        s["q_out"].copy_(_rotate(q, cos, sin).flatten(1))
        k = _rotate(k, cos, sin)
        if s["k_out"] is not None:
            s["k_out"].copy_(k)
        for name, x in (("k", k), ("v", v)):
            if s["done"] is not None:
                b, j = s["done"]
                rows = torch.cat([x, c[name + "_tail"].transpose(1, 2).flatten(0, 1)])[s["src"]]       # [blocks, 64, nkv, D]
                codes, scale = _quantise(rows.permute(2, 0, 1, 3).flatten(1, 2))
                c[name].unflatten(2, (-1, BLOCK))[b, :, j] = codes.unflatten(1, (-1, BLOCK)).transpose(0, 1)
                c[name + "_scale"][b, :, j] = scale.t()
            c[name + "_tail"][s["seq"][s["keep"]], :, s["at"][s["keep"]] % BLOCK] = x[s["keep"]]
        return _appended(s)
    n = [p + 1 for p in s["positions"]] if kind == "decode" else s["lens"]
    rows = max(n)
    if kind == "rows":
        for b, nb in enumerate(n):
            s["k_out"][b, :, :nb] = _cache_rows(c, "k", b, nb).bfloat16()
            s["v_out"][b, :, :nb] = _cache_rows(c, "v", b, nb).bfloat16()
        return s["k_out"], s["v_out"]
    out = s["out"].view(len(n), nkv, s["nq"] // nkv, D)
    for b, nb in enumerate(n):
        if nb == 0:
            out[b] = 0
            continue
        q = s["q"][b].view(nkv, s["nq"] // nkv, D).float()
        p = ((q @ _cache_rows(c, "k", b, nb).transpose(1, 2)) * s["scale"]).softmax(-1)
        out[b] = (p @ _cache_rows(c, "v", b, nb)).bfloat16()
    return s["out"]


def _cache_rows(c, name, b, n):
    """Rows 0 .. n - 1 of sequence b in fp32 [nkv, n, D]."""
    whole = n // BLOCK * BLOCK
    x = c[name][b, :, :whole].float() * c[name + "_scale"][b, :, : whole // BLOCK].repeat_interleave(BLOCK, 1)[..., None]
    return torch.cat([x, c[name + "_tail"][b, :, : n - whole].float()], 1)


def _plain_prompt(s):
    nkv, at = s["nkv"], 0
    G = s["nq"] // nkv
    for b, (n, h) in enumerate(zip(s["lens"], s["hist"])):
        if n == 0:
            continue
        k, v = ((s["k"][b, :, : n + h], s["v"][b, :, : n + h]) if s["k_len"] is not None
                else (s["k"][at: at + n].transpose(0, 1), s["v"][at: at + n].transpose(0, 1)))
        k, v = k.float(), v.float()                                      # [nkv, keys, D]
        step = max(1, (1 << 29) // (s["nq"] * (n + h)))                  # query rows whose scores are held at a time
        for i in range(0, n, step):
            j = min(n, i + step)
            m = h + j                                                    # keys that any of these rows sees
            q = s["q"][at + i: at + j].float().unflatten(1, (nkv, G)).permute(1, 2, 0, 3).flatten(1, 2)
            w = ((q @ k[:, :m].transpose(1, 2)) * s["scale"]).unflatten(1, (G, j - i))
            unseen = torch.arange(m, device=DEV) > (h + torch.arange(i, j, device=DEV))[:, None]
            w = w.masked_fill(unseen, -math.inf).softmax(-1)
            o = w.flatten(1, 2) @ v[:, :m]
            s["out"][at + i: at + j] = o.unflatten(1, (G, j - i)).permute(2, 0, 1, 3).flatten(1, 2).bfloat16()
        at += n
    return s["out"]


# ----------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    f64 = torch.float64
    D, nkv = case["D"], case["nkv"]
    if case["kind"] == "prompt":
        G, at = case["nq"] // nkv, 0
        out = torch.zeros(s["out"].shape, device=DEV, dtype=f64)
        for b, (n, h) in enumerate(zip(s["lens"], s["hist"])):
            for head in range(case["nq"]):
                if s["k_len"] is not None:
                    k, v = s["k"][b, head // G, : n + h], s["v"][b, head // G, : n + h]
                else:
                    k, v = s["k"][at: at + n, head // G], s["v"][at: at + n, head // G]
                for i in range(0, n, 4096):
                    j = min(n, i + 4096)
                    e = torch.einsum("id,jd->ij", s["q"][at + i: at + j, head].to(f64), k.to(f64)).div_(math.sqrt(D))
                    seen = torch.ones(j - i, n + h, device=DEV, dtype=torch.bool).tril_(h + i)
                    e = torch.where(seen, e, torch.full((), -math.inf, device=DEV, dtype=f64))
                    e = (e - e.max(1, keepdim=True).values).exp()
                    out[at + i: at + j, head] = torch.einsum("ij,jd->id", e, v.to(f64)) / e.sum(1, keepdim=True)
            at += n
        return out
    c = s["cache"]

    def row_values(name, b, n):
        x = c[name][b].to(f64).reshape(nkv, -1, BLOCK, D) * c[name + "_scale"][b].to(f64)[:, :, None, None]
        x = x.reshape(nkv, -1, D)[:, :n].clone()
        if n % BLOCK:
            x[:, n - n % BLOCK:] = c[name + "_tail"][b, :, : n % BLOCK].to(f64)
        return x

    if case["kind"] == "rows":
        res = []
        for name in ("k", "v"):
            o = torch.zeros(s[name + "_out"].shape, device=DEV, dtype=f64)
            for b, n in enumerate(s["lens"]):
                o[b, :, :n] = row_values(name, b, n)
            res.append(o)
        return tuple(res)
    if case["kind"] == "decode":
        out = torch.zeros(len(s["positions"]), nkv, case["nq"] // nkv, D, device=DEV, dtype=f64)
        for b, p in enumerate(s["positions"]):
            if p < 0:
                continue
            k, v = row_values("k", b, p + 1), row_values("v", b, p + 1)
            e = torch.einsum("hgd,hpd->hgp", s["q"][b].to(f64).reshape(nkv, -1, D), k) / math.sqrt(D)
            e = (e - e.amax(-1, keepdim=True)).exp()
            out[b] = torch.einsum("hgp,hpd->hgd", e, v) / e.sum(-1, keepdim=True)
        return out.reshape(len(s["positions"]), -1)

    # append: sequence by sequence, position by position of its rows
    nq, x = case["nq"], s["qkv"].to(f64).reshape(s["qkv"].shape[0], -1, D)
    turned = x[:, : nq + nkv]
    a, b = turned[..., : D // 2], turned[..., D // 2:]
    co, si = s["cos"].to(f64)[s["at"]][:, None], s["sin"].to(f64)[s["at"]][:, None]
    turned = torch.cat([a * co[..., : D // 2] - b * si[..., : D // 2], b * co[..., D // 2:] + a * si[..., D // 2:]], -1)
    res = {"q": turned[:, :nq].reshape(x.shape[0], -1)}
    if s["k_out"] is not None:
        res["k"] = turned[:, nq:]
    start = 0
    blocks = {"k": [], "v": []}
    tails = {n: c[n + "_tail"].to(f64) for n in ("k", "v")}
    for i, (p, n) in enumerate(zip(s["positions"], s["lens"])):
        for name, new in (("k", turned[:, nq:].bfloat16().to(f64)), ("v", x[:, nq + nkv:])):       # the cache is given bf16 rows
            rows = torch.cat([tails[name][i, :, : p % BLOCK], new[start: start + n].transpose(0, 1)], 1)
            full = rows.shape[1] // BLOCK
            for j in range(full):
                y = rows[:, j * BLOCK: (j + 1) * BLOCK]
                m, e = torch.frexp(y.abs().amax((1, 2)) / 127)
                step = torch.ldexp(torch.ceil(m * 256) / 256, e).clamp_min(2.0 ** -126)[:, None, None]
                blocks[name].append(torch.round(y / step) * step)
            left = rows.shape[1] - full * BLOCK
            # (a tail keeps what it held in the rows that the unfinished block has not reached)
            lo = p % BLOCK if full == 0 else 0
            tails[name][i, :, lo: left] = rows[:, full * BLOCK + lo:]
        start += n
    for name in ("k", "v"):
        res[name + "_tail"] = tails[name]
        if blocks[name]:
            res[name + "_blocks"] = torch.stack(blocks[name])
    return res
