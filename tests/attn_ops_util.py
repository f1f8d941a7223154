"""Plain 64-bit forms of the attention operators and their error bounds.

u(t): half a step of type t relative to the value (one rounding to nearest).
"""
import ctypes as C
import math

import torch

DT = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
U = {t: torch.finfo(d).eps / 2 for t, d in DT.items()}
U32 = 2.0 ** -24


def ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def rope_ref(x, pos, turn, mscale, half, sign=1.0):
    """x [rows, heads, dim] float64 -> (rotated, |x0| + |x1| of every rotated place)."""
    n = 2 * len(turn)
    ang = 2 * math.pi * torch.remainder(pos.double()[:, None] * turn.to(x.device)[None, :], 1.0)
    c, s = (f(ang)[:, None, :] * mscale for f in (torch.cos, torch.sin))
    s = s * sign
    a, b = (slice(0, n // 2), slice(n // 2, n)) if half else (slice(0, n, 2), slice(1, n, 2))
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * mscale
    return y, size


def attn_ref(q, k, v, seen, scale):
    """One head: q [m, d], k and v [n, d] float64, seen [m, n] -> (out, bound without the type's roundings,
    sum of p |v|).  What is not seen takes no part, whatever it holds."""
    d = q.shape[1]
    z = (q @ torch.nan_to_num(k).T) * scale
    big = (q.abs() @ torch.nan_to_num(k).abs().T) * abs(scale)
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(1, keepdim=True) if z.shape[1] else z.new_full((len(z), 1), -math.inf)
    p = torch.exp(z - torch.where(torch.isfinite(top), top, 0.0)) * seen
    l = p.sum(1, keepdim=True)
    p = p / torch.where(l > 0, l, 1.0)
    out, av = p @ torch.nan_to_num(v), p @ torch.nan_to_num(v).abs()
    # a score's error: d fp32 additions of products (each rounded; operands of 22 bits or more, which
    # adds at most 2^-20 of every product) and the scaling; exp2's argument and result add a few units of
    # its size.  Weights are off by twice that (numerator and sum), sums over n slots add n/2 more roundings
    # (partial sums of at least two lanes).
    worst = (big * seen).amax(1, keepdim=True) if z.shape[1] else z.new_zeros(len(z), 1)
    score = worst * ((d + 8) * U32 + 2.0 ** -20) + (z.masked_fill(~seen, 0.0).abs().amax(1, keepdim=True) * 2 if z.shape[1] else 0) * 4 * U32
    rel = 2 * score + (z.shape[1] / 2 + 40) * U32
    return out, rel * av, av


def close(got, out, bound, av, t):
    """Elementwise: |got - out| <= bound + the roundings to type t: of the weights (16-bit types only, u of each,
    so u * sum p|v|), and of the result.  f16's smallest step (2^-24) rounds off by half of it at worst."""
    u = U[t]
    tol = bound + (u * av * 1.05 if t else 0.0) + u * out.abs() * 1.05 + u * bound + (2.0 ** -25 if t == 1 else 1e-37)
    g = got.double()
    assert torch.isfinite(g).all()
    bad = (g - out).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((g - out).abs() / tol).max()))


class Cache:
    """A paged cache with a table of its own; unused places hold NaN."""

    def __init__(self, cw, t, seqs, slots, page, n_kv, dim, layers=1, seed=0, device="cuda", spare=2):
        g = torch.Generator().manual_seed(seed)
        self.cw, self.t, self.page, self.dev = cw, t, page, device
        self.stride = max(1, -(-slots // page))
        n = seqs * self.stride + spare
        self.table_h = torch.randperm(n, generator=g)[:seqs * self.stride].view(seqs, self.stride).int()
        self.table = self.table_h.to(device)
        shape = (layers, n, page, n_kv, dim)
        self.k, self.v = (torch.full(shape, math.nan, dtype=DT[t], device=device) for _ in range(2))
        self.desc = cw.Kv(t, layers, n, page, n_kv, dim, self.k.data_ptr(), self.v.data_ptr())

    def rows(self, s, slots):
        """Flat pool rows of a sequence's slots."""
        slots = torch.as_tensor(list(slots), dtype=torch.long)
        return (self.table_h[s].long()[slots // self.page] * self.page + slots % self.page).to(self.dev)

    def flat(self, which, layer=0):
        x = (self.k if which == "k" else self.v)[layer]
        return x.view(-1, *x.shape[2:])
