"""Attention with shaped scores in 64 bits, with elementwise bounds on what a
kernel that holds P in bfloat16 and sums in 32 bits may be off.

A rounding to bfloat16 is off by at most h = 2**-8 of the value.  With
absolute sums S(x) of the terms of a product:
  out    P is rounded, the result once:        e_o + h |out|
         e_o = h P|V| + h |out|
  dV     P is rounded, the result:             2 h P^T|dO| + h |dV|
  delta  sum of dO * out and its remainder:    e_d = sum_d |dO| e_o
  dS     P (dP - delta) u:                     e_s = u P e_d + h |dS|
  dQ     scale (e_s |K|) + h |dQ|              dK: scale (e_s^T |Q|) + h |dK|
The kernels divide by the sum of the rounded terms p_j (1 + e_j), |e_j| <= h.
That sum is (1 + m) sum p_j with the weighted mean m = sum p_j e_j / sum p_j,
so |m| <= h too, and a weight of the values is P_j (1 + e_j) / (1 + m): off by
h of each term and m of the whole, which is e_o.  The log-sum holds the same
1 + m, so the backward's P is P_j / (1 + m): m more on top of its own rounding
in dV, and m |dS| in dS, which goes on as two bfloat16 (2**-16 of it).
The 32-bit sums add n * 2**-24 of the absolute sum, the hardware's exp2 and
reciprocal and the tanh 2e-5 of a probability at these sizes: both are covered
by 10 per cent on every bound (0.1 * 2**-8 = 4e-4) and 1e-6 for sums that
cancel to nothing.
"""
import numpy as np
import torch

H8 = 2.0 ** -8


def visible(B, Tq, Tk, causal=False, seg_q=None, seg_k=None, prefix=None,
            kv_len=None, off=0):
    """[B, Tq, Tk] truth values, one pair at a time by the definition."""
    ok = np.zeros((B, Tq, Tk), bool)
    pos = np.zeros((B, Tq), np.int64)
    for b in range(B):
        o = int(off[b]) if np.ndim(off) else int(off)
        for i in range(Tq):
            p = i + o
            pos[b, i] = p
            j = np.arange(Tk)
            see = np.ones(Tk, bool)
            if causal:
                see = j <= p
                if prefix is not None:
                    see |= j < int(prefix[b])
            if kv_len is not None:
                see &= j < int(kv_len[b])
            if seg_q is not None:
                see &= (np.asarray(seg_k[b]) == int(seg_q[b][i])) \
                    & (int(seg_q[b][i]) >= 0)
            ok[b, i] = see
    return torch.from_numpy(ok), torch.from_numpy(pos)


def reference(q, k, v, dout, H, Hkv, ok, pos, scale=None, cap=None,
              slopes=None):
    """q, k, v, dout as CPU tensors; returns {name: (value, bound)}."""
    B, Tq, HD = q.shape
    Tk, D, G = k.shape[1], HD // H, H // Hkv
    scale = D ** -0.5 if scale is None else scale
    # places that no query sees may hold anything
    dead_k = ~ok.any(1)
    dead_q = ~ok.any(2)
    q, k, v = q.double(), k.double(), v.double()
    q = torch.where(dead_q[:, :, None], torch.zeros_like(q), q)
    k = torch.where(dead_k[:, :, None], torch.zeros_like(k), k)
    v = torch.where(dead_k[:, :, None], torch.zeros_like(v), v)

    def split(x, n):
        return x.reshape(B, x.shape[1], n, D).transpose(1, 2)

    qh = split(q, H)
    kh = split(k, Hkv).repeat_interleave(G, 1)
    vh = split(v, Hkv).repeat_interleave(G, 1)
    s = qh @ kh.transpose(-1, -2) * scale
    u = torch.ones_like(s)
    if cap is not None:
        t = torch.tanh(s / cap)
        s, u = cap * t, 1 - t * t
    if slopes is not None:
        dist = (pos[:, :, None] - torch.arange(Tk)).abs().double()
        s = s - slopes.double()[None, :, None, None] * dist[:, None]
    m = ok[:, None].expand_as(s)
    s = torch.where(m, s, torch.full_like(s, -float("inf")))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(s - top)
    z = e.sum(-1, keepdim=True)
    p = torch.where(z > 0, e / z, torch.zeros_like(e))

    def merge(x):
        return x.transpose(1, 2).reshape(B, x.shape[2], -1)

    def group(x):
        return x.reshape(B, Hkv, G, Tk, D).sum(2)

    out = p @ vh
    e_o = H8 * (p @ vh.abs()) + H8 * out.abs()
    out_b = 1.1 * (e_o + H8 * out.abs()) + 1e-6
    res = {"out": (merge(out), merge(out_b))}
    if dout is None:
        return res
    g = dout.double()
    g = torch.where(dead_q[:, :, None], torch.zeros_like(g), g)
    gh = split(g, H)
    dp = gh @ vh.transpose(-1, -2)
    delta = (gh * out).sum(-1, keepdim=True)
    ds = p * (dp - delta) * u
    e_s = u * p * (gh.abs() * e_o).sum(-1, keepdim=True) + H8 * ds.abs()
    dq = scale * ds @ kh
    dk = group(scale * ds.transpose(-1, -2) @ qh)
    dv = group(p.transpose(-1, -2) @ gh)
    sc = abs(scale)
    dq_b = 1.1 * (sc * e_s @ kh.abs() + H8 * dq.abs()) + 1e-6
    dk_b = 1.1 * (group(sc * e_s.transpose(-1, -2) @ qh.abs())
                  + H8 * dk.abs()) + 1e-6
    dv_b = 1.1 * (group(2 * H8 * p.transpose(-1, -2) @ gh.abs())
                  + H8 * dv.abs()) + 1e-6
    res.update(dq=(merge(dq), merge(dq_b)), dk=(merge(dk), merge(dk_b)),
               dv=(merge(dv), merge(dv_b)))
    return res


def check(name, got, ref):
    want, bound = ref
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got - want).abs() / bound).max()
    assert over <= 1.0, f"{name}: {float(over):.3f} times its bound"
