"""Plain 64-bit implementations of the 8-bit key/value cache and of attention, for the tests."""

import math

import torch

BLOCK = 64


def quantise(x):
    """bf16 [..., rows, D], whole blocks -> (codes int8, scales float64 [..., rows / 64])."""
    y = x.double().unflatten(-2, (-1, BLOCK))
    m, e = torch.frexp(y.abs().amax((-1, -2)) / 127)
    s = torch.ldexp(torch.ceil(m * 256) / 256, e).clamp_min(2.0 ** -126)
    return torch.round(y / s[..., None, None]).to(torch.int8).flatten(-3, -2), s


def rotate(x, cos, sin):
    """Rotate-half embedding of [..., D] in 64 bits, rounded to bf16."""
    half = x.shape[-1] // 2
    x = x.double()
    other = torch.cat([-x[..., half:], x[..., :half]], -1)
    return (x * cos.double() + other * sin.double()).bfloat16()


class RefCache:
    """What a Kv8Cache has to hold: per slot and head the rows given so far, in 64 bits; values() as it reads back."""

    def __init__(self, slots, nkv, D):
        self.rows = {n: [torch.zeros(nkv, 0, D, dtype=torch.bfloat16) for _ in range(slots)] for n in ("k", "v")}

    def append(self, slot, k, v):        # bf16 [n, nkv, D]
        for n, x in (("k", k), ("v", v)):
            self.rows[n][slot] = torch.cat([self.rows[n][slot], x.cpu().transpose(0, 1)], 1)

    def length(self, slot):
        return self.rows["k"][slot].shape[1]

    def values(self, name, slot, n=None):
        x = self.rows[name][slot][:, : n]
        whole = x.shape[1] // BLOCK * BLOCK
        codes, s = quantise(x[:, :whole])
        return torch.cat([codes.double() * s.repeat_interleave(BLOCK, 1)[..., None], x[:, whole:].double()], 1)


def attention(q, k, v, scale, seen=None):
    """q [nq, lq, D], k and v [nkv, lk, D] in 64 bits, seen [lq, lk] (None: all) -> [nq, lq, D]; an empty row is zero.
    What a row does not see takes no part in it, whatever it holds."""
    nq, nkv = q.shape[0], k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(nq // nkv, 0), v.double().repeat_interleave(nq // nkv, 0)
    s = torch.einsum("hid,hjd->hij", q, k) * scale
    if seen is not None:
        s = torch.where(seen, s, torch.full((), -math.inf, dtype=torch.float64, device=s.device))
    m = s.amax(-1, keepdim=True) if s.shape[-1] else torch.zeros(*s.shape[:2], 1, dtype=torch.float64, device=s.device)
    e = (s - torch.where(m == -math.inf, 0.0, m)).exp()
    fine = torch.isfinite(v)
    o = torch.einsum("hij,hjd->hid", e, torch.where(fine, v, 0.0))
    if not bool(fine.all()):
        for h, j, d in (~fine).nonzero().tolist():          # 0 * inf is not asked of a row that does not see it
            rows = slice(None) if seen is None else seen[:, j]
            o[h, rows, d] += v[h, j, d]
    tot = e.sum(-1, keepdim=True)
    return torch.where(tot == 0, 0.0, o / tot)


def tables(max_len, D, device):
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    ang = torch.arange(max_len, dtype=torch.float64)[:, None] * inv[None, :]
    both = torch.cat([ang, ang], -1)
    return both.cos().float().to(device), both.sin().float().to(device)
