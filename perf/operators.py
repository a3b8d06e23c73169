"""Operators of a language model's training step and of its single-token
steps, with their plain forms and the cases they are measured on.

  attention   scores capped by a tanh, a bias that falls with distance,
              document and prefix masks, shared key/value heads; forward with
              its backward (``kind="train"``)
  decode      the same attention for a few new tokens over a long cache
              whose sequences have lengths of their own (``kind="decode"``)
  embedding   row lookup with a scale, and the gradient of the table
  clip        the global norm of many gradients, and their clipping by it

``run`` computes the plain form (elementary torch operations in 32 bits, or
in 64 where sums are long) and, where ``own`` is true, makes the calls of
``anand_mxnet_amd``.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}


# ---------------------------------------------------------------- cases

def _train(name, B, T, H, Hkv, D, docs=0, prefix=False, causal=True, cap=0.0,
           slopes=False, layout=0):
    return {"name": name, "kind": "train", "B": B, "T": T, "H": H,
            "Hkv": Hkv, "D": D, "docs": docs, "prefix": prefix,
            "causal": causal, "cap": cap, "slopes": slopes,
            "layout": layout}


def _decode(name, B, Tq, Tk, H, Hkv, D, cap=0.0, slopes=False, low=0.5,
            layout=0):
    return {"name": name, "kind": "decode", "B": B, "Tq": Tq, "Tk": Tk,
            "H": H, "Hkv": Hkv, "D": D, "cap": cap, "slopes": slopes,
            "low": low, "layout": layout}


def _embed(name, vocab, D, tokens, dtype, scale, skew):
    return {"name": name, "kind": "embedding", "vocab": vocab, "D": D,
            "tokens": tokens, "dtype": dtype, "scale": scale, "skew": skew}


def _clip(name, model, dtype, layers, units, ratio):
    return {"name": name, "kind": "clip", "model": model, "dtype": dtype,
            "layers": layers, "units": units, "ratio": ratio}


def listed():
    return [
        # a short odd batch through the smallest zoo configuration (2 heads
        # of 64): latency of the whole forward and backward
        _train("train_tiny", 2, 77, 2, 2, 64, docs=3, cap=30.0, layout=1),
        # the transformer-big training shape (16 heads of 64, 512 tokens,
        # batch 32) on packed documents with capped scores
        _train("train_packed512", 32, 512, 16, 16, 64, docs=4, cap=50.0,
               layout=2),
        # a prefix language model over 4095 tokens, four query heads to a
        # key head, bias by distance, no cap
        _train("train_prefix4k", 2, 4095, 16, 4, 128, prefix=True,
               slopes=True, layout=3),
        # long-context training: 16384 tokens in a few long documents
        _train("train_long16k", 1, 16384, 16, 8, 128, docs=3, cap=50.0,
               layout=4),
        # one sequence, one token: what an interactive user waits for
        _decode("decode_one", 1, 1, 2048, 16, 16, 64, cap=50.0, low=0.7,
                layout=5),
        # a serving batch with ragged lengths, grouped heads
        _decode("decode_batch", 64, 1, 8192, 16, 4, 128, cap=30.0,
                slopes=True, low=0.05, layout=6),
        # few very long sequences, three tokens a step (drafted tokens)
        _decode("decode_long", 4, 3, 131071, 16, 8, 128, cap=50.0, low=0.8,
                layout=7),
        # token types: a table of two rows that every token of a batch hits
        _embed("embed_types", 2, 768, 16384, "bf16", 1.0, 0.5),
        # word table of transformer-big, batch 32 of 512, scaled by 32
        _embed("embed_words", 32768, 1024, 16384, "bf16", 32.0, 1.1),
        # fine-tuning with a small odd batch, single precision table
        _embed("embed_small", 30528, 768, 333, "fp32", 1.0, 1.1),
        # gradients of a bottleneck convolution network: many small ones
        _clip("clip_conv", "conv", "fp32", 16, 64, 0.25),
        # gradients of transformer-big: large matrices in bf16
        _clip("clip_transformer", "transformer", "bf16", 12, 1024, 0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["train", "train", "decode", "decode", "embedding",
                       "clip"])
    layout = rng.randrange(1 << 20)
    if kind == "train":
        Hkv = rng.choice([1, 2, 4, 8, 16])
        H = Hkv * rng.choice([1, 2, 4, 8])
        T = _log_int(rng, 1, 16384)
        c = _train("", max(1, min(32, _log_int(rng, 1, 16384) // T)), T,
                   min(H, 32), min(Hkv, 32),
                   rng.choice([32, 64, 64, 80, 96, 128, 128]),
                   docs=rng.choice([0, 1, 3, 7]),
                   prefix=rng.random() < 0.4, causal=rng.random() < 0.8,
                   cap=rng.choice([0.0, 20.0, 50.0]),
                   slopes=rng.random() < 0.5, layout=layout)
    elif kind == "decode":
        Hkv = rng.choice([1, 2, 4, 8, 16])
        H = Hkv * rng.choice([1, 2, 4, 8])
        Tk = _log_int(rng, 1, 131072)
        c = _decode("", max(1, min(96, _log_int(rng, 64, 524288) // Tk)),
                    rng.choice([1, 1, 1, 2, 5, 8]), Tk, min(H, 32), Hkv,
                    rng.choice([32, 64, 64, 80, 96, 128, 128]),
                    cap=rng.choice([0.0, 30.0, 50.0]),
                    slopes=rng.random() < 0.5,
                    low=rng.choice([0.0, 0.3, 0.9]), layout=layout)
    elif kind == "embedding":
        c = _embed("", _log_int(rng, 1, 65536), _log_int(rng, 1, 1100),
                   _log_int(rng, 1, 32768),
                   rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                   rng.choice([1.0, 32.0, 22.627416997969522, 0.125]),
                   rng.choice([0.0, 0.6, 1.1]))
    else:
        c = _clip("", rng.choice(["conv", "transformer"]),
                  rng.choice(["bf16", "fp16", "fp32", "mixed"]),
                  rng.randint(1, 12), _log_int(rng, 17, 1024),
                  rng.choice([0.01, 0.5, 2.0]))
    del c["name"]
    return c


def _dense(c):
    if c["kind"] != "train":
        return 0
    return c["B"] * c["H"] * c["T"] ** 2


def draw(rng):
    top = listed()
    limit = {}
    for t in top:
        w = work(t)
        o = limit.setdefault(t["kind"], [0, 0, 0])
        o[0] = max(o[0], w["bytes"])
        o[1] = max(o[1], w["flops"])
        o[2] = max(o[2], _dense(t))
    while True:
        c = _draw_once(rng)
        w = work(c)
        m = limit[c["kind"]]
        if w["bytes"] <= m[0] and w["flops"] <= m[1] and _dense(c) <= m[2]:
            return c


# ---------------------------------------------------------------- layouts

def _doc_lengths(c):
    """Document lengths of each packed row of the batch; what is left of
    the row is padding (its tokens have the id -1)."""
    r = random.Random(c["layout"])
    rows = []
    for _ in range(c["B"]):
        cuts = sorted(r.randint(0, c["T"]) for _ in range(c["docs"] - 1))
        end = c["T"] - r.randint(0, c["T"] // 16)
        cuts = [x for x in cuts if x < end]
        edges = [0] + cuts + [end]
        rows.append([b - a for a, b in zip(edges, edges[1:])])
    return rows


def _prefixes(c):
    r = random.Random(c["layout"] + 1)
    return [r.randint(0, c["T"] // 2) for _ in range(c["B"])]


def _cache_lengths(c):
    r = random.Random(c["layout"] + 2)
    lo = int(c["low"] * c["Tk"])
    return [r.randint(lo, c["Tk"]) for _ in range(c["B"])]


def _pairs(c):
    """Pairs of a query and a key that the masks let meet, over the batch
    (one head)."""
    if c["kind"] == "decode":
        n = 0
        for length in _cache_lengths(c):
            for i in range(c["Tq"]):
                n += max(0, length - c["Tq"] + i + 1)
        return n
    T = c["T"]
    pre = _prefixes(c) if c["prefix"] else [0] * c["B"]
    rows = _doc_lengths(c) if c["docs"] else [[T]] * c["B"]
    total = 0
    for lens, p in zip(rows, pre):
        a = 0
        for n in lens:
            b = a + n
            if not c["causal"]:
                total += n * n
            else:
                i = np.arange(a, b, dtype=np.int64)
                last = np.maximum(i + 1, min(p, b))
                total += int((last - a).sum())
            a = b
    return total


def work(c):
    kind = c["kind"]
    if kind == "train":
        n = c["B"] * c["T"] * c["D"]
        # q, dout read and out, dq written; k, v read and dk, dv written
        return {"bytes": 2 * (4 * n * c["H"] + 4 * n * c["Hkv"]),
                "flops": 14 * _pairs(c) * c["H"] * c["D"]}
    if kind == "decode":
        q = 2 * c["B"] * c["Tq"] * c["H"] * c["D"]
        kv = sum(_cache_lengths(c)) * c["Hkv"] * c["D"] * 2 * 2
        return {"bytes": 2 * q + kv + 8 * c["B"],
                "flops": 4 * _pairs(c) * c["H"] * c["D"]}
    if kind == "embedding":
        size = 4 if c["dtype"] == "fp32" else 2
        rows = min(c["vocab"], c["tokens"])
        return {"bytes": size * c["D"] * (rows + 2 * c["tokens"] + c["vocab"])
                + 8 * c["tokens"],
                "flops": 2 * c["D"] * c["tokens"]}
    n = size = 0
    for shape, dt in _clip_shapes(c):
        k = math.prod(shape)
        n += k
        size += k * (4 if dt == "fp32" else 2)
    return {"bytes": 2 * size, "flops": 3 * n}


def _clip_shapes(c):
    u = c["units"]
    shapes = []
    if c["model"] == "conv":
        shapes.append((u, 7, 7, 3))
        stages = [(u, 3), (2 * u, 4), (4 * u, 6), (8 * u, 3)]
        done, width = 0, u
        for mid, blocks in stages:
            for b in range(blocks):
                if done == c["layers"]:
                    break
                shapes += [(mid, 1, 1, width), (mid,), (mid,),
                           (mid, 3, 3, mid), (mid,), (mid,),
                           (4 * mid, 1, 1, mid), (4 * mid,), (4 * mid,)]
                if b == 0:
                    shapes += [(4 * mid, 1, 1, width), (4 * mid,),
                               (4 * mid,)]
                width = 4 * mid
                done += 1
        shapes += [(1000, width), (1000,)]
    else:
        shapes += [(32 * u, u), (u,)]
        for _ in range(c["layers"]):
            shapes += [(u, u), (u,)] * 4
            shapes += [(4 * u, u), (4 * u,), (u, 4 * u), (u,)]
            shapes += [(u,)] * 4
    out = []
    for s in shapes:
        dt = c["dtype"]
        if dt == "mixed":  # normalisation in single precision
            dt = "fp32" if len(s) == 1 else "bf16"
        out.append((s, dt))
    return out


# ---------------------------------------------------------------- inputs

def _slopes(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


def _segments(c):
    seg = np.full((c["B"], c["T"]), -1, np.int32)
    for b, lens in enumerate(_doc_lengths(c)):
        a = 0
        for i, n in enumerate(lens):
            seg[b, a:a + n] = i
            a += n
    return torch.from_numpy(seg)


def _buckets(tensors):
    """One zeroed buffer for each type, and a view of it for each tensor,
    as data-parallel training keeps its gradients; views begin at multiples
    of 64 elements."""
    starts, size = [], {}
    for t in tensors:
        a = size.get(t.dtype, 0)
        starts.append(a)
        size[t.dtype] = a + (t.numel() + 63) // 64 * 64
    flat = {dt: torch.zeros(n, dtype=dt, device=DEV)
            for dt, n in size.items()}
    views = [flat[t.dtype][a:a + t.numel()].view(t.shape)
             for t, a in zip(tensors, starts)]
    return list(flat.values()), views


def _rand(g, shape, dtype, std=1.0):
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    return (x * std).to(dtype)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind = c["kind"]
    s = {"case": c}
    if kind in ("train", "decode"):
        B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
        Tq, Tk = (c["T"], c["T"]) if kind == "train" else (c["Tq"], c["Tk"])
        # scores of a trained layer spread over several units: enough for
        # the cap to bend the largest ones
        s["q"] = _rand(g, (B, Tq, H * D), torch.bfloat16, 2.0)
        s["k"] = _rand(g, (B, Tk, Hkv * D), torch.bfloat16, 2.0)
        s["v"] = _rand(g, (B, Tk, Hkv * D), torch.bfloat16)
        if c["slopes"]:
            s["slopes"] = torch.tensor(_slopes(H), device=DEV,
                                       dtype=torch.float32)
        if kind == "train":
            s["dout"] = _rand(g, (B, Tq, H * D), torch.bfloat16)
            if c["docs"]:
                s["seg"] = _segments(c).to(DEV)
            if c["prefix"]:
                s["prefix"] = torch.tensor(_prefixes(c), device=DEV,
                                           dtype=torch.int32)
        else:
            s["length"] = torch.tensor(_cache_lengths(c), device=DEV,
                                       dtype=torch.int32)
            s["offset"] = s["length"] - Tq
    elif kind == "embedding":
        dt = DTYPES[c["dtype"]]
        V, N = c["vocab"], c["tokens"]
        # token frequencies fall as a power of the rank, ranks are spread
        # over the table
        p = torch.arange(1, V + 1, device=DEV, dtype=torch.float64)
        p = torch.cumsum(p.pow(-c["skew"]), 0)
        u = torch.rand(N, generator=g, device=DEV, dtype=torch.float64)
        rank = torch.searchsorted(p, u * p[-1]).clamp_(max=V - 1)
        perm = torch.randperm(V, generator=g, device=DEV)
        s["idx"] = perm[rank]
        s["weight"] = _rand(g, (V, c["D"]), dt, c["D"] ** -0.5)
        s["dout"] = _rand(g, (N, c["D"]), dt, 1e-2)
    else:
        s["grads"] = [_rand(g, sh, DTYPES[dt], 1e-3)
                      for sh, dt in _clip_shapes(c)]
        n = sum(t.numel() for t in s["grads"])
        s["max_norm"] = c["ratio"] * 1e-3 * math.sqrt(n)
        s["flat"], s["clipped"] = _buckets(s["grads"])
    if own:
        _wrap(s)
    return s


def _wrap(s):
    from anand_mxnet_amd import nd
    for key in ("q", "k", "v", "dout", "seg", "prefix", "slopes", "length",
                "offset", "idx", "weight"):
        if key in s:
            s["nd_" + key] = nd.from_torch(s[key])
    for key in ("grads", "clipped"):
        if key in s:
            s["nd_" + key] = [nd.from_torch(t) for t in s[key]]
    if s["case"]["kind"] == "train":
        for key in ("nd_q", "nd_k", "nd_v"):
            s[key].attach_grad()
    if s["case"]["kind"] == "embedding":
        s["nd_weight"].attach_grad()


# ---------------------------------------------------------------- run

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from anand_mxnet_amd import autograd, nd
    c = s["case"]
    kind = c["kind"]
    if kind == "train":
        with autograd.record():
            out = nd.multi_head_attention(
                s["nd_q"], s["nd_k"], s["nd_v"], c["H"], causal=c["causal"],
                num_kv_heads=c["Hkv"], logit_cap=c["cap"] or None,
                distance_slopes=s.get("nd_slopes"),
                segment_ids=s.get("nd_seg"),
                prefix_length=s.get("nd_prefix"))
        out.backward(s["nd_dout"])
        return [out._t.detach(), s["nd_q"].grad._t, s["nd_k"].grad._t,
                s["nd_v"].grad._t]
    if kind == "decode":
        out = nd.multi_head_attention(
            s["nd_q"], s["nd_k"], s["nd_v"], c["H"], causal=True,
            num_kv_heads=c["Hkv"], logit_cap=c["cap"] or None,
            distance_slopes=s.get("nd_slopes"), kv_length=s["nd_length"],
            query_offset=s["nd_offset"])
        return out._t
    if kind == "embedding":
        with autograd.record():
            out = nd.Embedding(s["nd_idx"], s["nd_weight"],
                               input_dim=c["vocab"], output_dim=c["D"],
                               scale=c["scale"])
        out.backward(s["nd_dout"])
        return [out._t.detach(), s["nd_weight"].grad._t]
    norm = nd.multi_clip_global_norm(s["nd_grads"], s["max_norm"],
                                     out=s["nd_clipped"])
    return [norm._t] + s["flat"]


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "train":
        return _plain_train(s)
    if kind == "decode":
        return _plain_decode(s)
    if kind == "embedding":
        w = s["weight"]
        out = (w[s["idx"]].float() * c["scale"]).to(w.dtype)
        # a frequent token sums many rows: in 64 bits
        g = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
        g.index_add_(0, s["idx"], s["dout"].double())
        return [out, (g * c["scale"]).to(w.dtype)]
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for t in s["grads"]:
        total = total + t.double().square().sum()
    norm = total.sqrt()
    f = torch.clamp(s["max_norm"] / (norm + 1e-8), max=1.0).float()
    for t, o in zip(s["grads"], s["clipped"]):
        o.copy_(t.float() * f)
    return [norm.float()] + s["flat"]


def _visible(s, b, i0, i1, Tk):
    """[i1 - i0, Tk] truth values: which keys the queries i0..i1 of
    sequence b may see; and their distances."""
    c = s["case"]
    j = torch.arange(Tk, device=DEV)
    pos = torch.arange(i0, i1, device=DEV)
    if "offset" in s:
        pos = pos + s["offset"][b]
    dist = pos[:, None] - j[None, :]
    ok = torch.ones_like(dist, dtype=torch.bool)
    if c.get("causal", True):
        ok = dist >= 0
        if "prefix" in s:
            ok = ok | (j < s["prefix"][b])[None, :]
    if "length" in s:
        ok = ok & (j < s["length"][b])[None, :]
    if "seg" in s:
        sq = s["seg"][b, i0:i1]
        ok = ok & (sq[:, None] == s["seg"][b][None, :]) & (sq >= 0)[:, None]
    return ok, dist


def _heads(x, n):
    """[T, n*D] -> [n, T, D] in 32 bits."""
    T, W = x.shape
    return x.float().reshape(T, n, W // n).transpose(0, 1).contiguous()


def _probs(s, q, k, ok, dist, h0, h1):
    c = s["case"]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * c["D"] ** -0.5
    t = None
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x = t * c["cap"]
    if "slopes" in s:
        x = x - s["slopes"][h0:h1, None, None] * dist.abs().float()[None]
    x = x.masked_fill(~ok[None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(x - m)
    z = p.sum(-1, keepdim=True)
    return p / torch.where(z > 0, z, torch.ones_like(z)), t


def _plain_train(s):
    c = s["case"]
    B, T, H, Hkv, D = c["B"], c["T"], c["H"], c["Hkv"], c["D"]
    G = H // Hkv
    out, dq = torch.empty_like(s["q"]), torch.empty_like(s["q"])
    dk, dv = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    # heads at a time, so that their scores fit comfortably
    step = max(1, min(Hkv, (1 << 30) // max(1, G * T * T)))
    for b in range(B):
        ok, dist = _visible(s, b, 0, T, T)
        q, do = _heads(s["q"][b], H), _heads(s["dout"][b], H)
        k, v = _heads(s["k"][b], Hkv), _heads(s["v"][b], Hkv)
        O, DQ = torch.empty_like(q), torch.empty_like(q)
        DK, DV = torch.empty_like(k), torch.empty_like(v)
        for a in range(0, Hkv, step):
            e = min(Hkv, a + step)
            h0, h1 = a * G, e * G
            kk = k[a:e].repeat_interleave(G, 0)
            vv = v[a:e].repeat_interleave(G, 0)
            p, t = _probs(s, q[h0:h1], kk, ok, dist, h0, h1)
            O[h0:h1] = torch.matmul(p, vv)
            dp = torch.matmul(do[h0:h1], vv.transpose(-1, -2).contiguous())
            dvh = torch.matmul(p.transpose(-1, -2).contiguous(), do[h0:h1])
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            if t is not None:
                ds = ds * (1.0 - t * t)
            ds = ds * D ** -0.5
            DQ[h0:h1] = torch.matmul(ds, kk)
            dkh = torch.matmul(ds.transpose(-1, -2).contiguous(), q[h0:h1])
            DK[a:e] = dkh.reshape(e - a, G, T, D).sum(1)
            DV[a:e] = dvh.reshape(e - a, G, T, D).sum(1)
        out[b] = O.transpose(0, 1).reshape(T, H * D)
        dq[b] = DQ.transpose(0, 1).reshape(T, H * D)
        dk[b] = DK.transpose(0, 1).reshape(T, Hkv * D)
        dv[b] = DV.transpose(0, 1).reshape(T, Hkv * D)
    return [out, dq, dk, dv]


def _plain_decode(s):
    c = s["case"]
    B, Tq, Tk, H, Hkv = c["B"], c["Tq"], c["Tk"], c["H"], c["Hkv"]
    G = H // Hkv
    out = torch.empty_like(s["q"])
    for b in range(B):
        ok, dist = _visible(s, b, 0, Tq, Tk)
        q = _heads(s["q"][b], H)
        k = _heads(s["k"][b], Hkv).repeat_interleave(G, 0)
        v = _heads(s["v"][b], Hkv).repeat_interleave(G, 0)
        p, _ = _probs(s, q, k, ok, dist, 0, H)
        out[b] = torch.matmul(p, v).transpose(0, 1).reshape(Tq, -1)
    return out


# ---------------------------------------------------------------- exact

def exact(case, seed):
    """The definition in 64 bits, head by head, gradients by automatic
    differentiation of it."""
    if case["kind"] == "train" and _dense(case) > 20 * 16384 ** 2:
        return None
    s = prepare(case, seed)
    c = s["case"]
    kind = c["kind"]
    if kind == "embedding":
        rows = s["weight"].double().index_select(0, s["idx"]) * c["scale"]
        order = torch.argsort(s["idx"])
        tok, d = s["idx"][order], s["dout"].double()[order] * c["scale"]
        g = torch.zeros(c["vocab"], c["D"], dtype=torch.float64, device=DEV)
        uniq, counts = torch.unique_consecutive(tok, return_counts=True)
        run_sum = torch.segment_reduce(d, "sum", lengths=counts, axis=0)
        g[uniq] = run_sum
        return [rows, g]
    if kind == "clip":
        flat = torch.cat([t.double().flatten() for t in s["grads"]])
        norm = torch.linalg.vector_norm(flat)
        f = min(1.0, s["max_norm"] / (float(norm) + 1e-8))
        return [norm] + _buckets_of([t.double() * f for t in s["grads"]],
                                    [t.dtype for t in s["grads"]])
    return _exact_attention(s, kind == "train")


def _buckets_of(values, dtypes):
    parts = {}
    for x, dt in zip(values, dtypes):
        pad = torch.zeros(-x.numel() % 64, dtype=x.dtype, device=DEV)
        parts.setdefault(dt, []).extend([x.flatten(), pad])
    return [torch.cat(p) for p in parts.values()]


def _exact_attention(s, train):
    c = s["case"]
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    Tq, Tk = s["q"].shape[1], s["k"].shape[1]

    def leaf(x, n):
        x = x.double().reshape(B, x.shape[1], n, D)
        return x.requires_grad_(train)

    q, k, v = leaf(s["q"], H), leaf(s["k"], Hkv), leaf(s["v"], Hkv)
    out = torch.zeros(B, Tq, H, D, dtype=torch.float64, device=DEV)
    i = torch.arange(Tq, device=DEV)[:, None]
    j = torch.arange(Tk, device=DEV)[None, :]
    for b in range(B):
        pos = i if train else i + int(s["offset"][b])
        see = torch.full((Tq, Tk), True, device=DEV)
        if c.get("causal", True):
            edge = pos
            if "prefix" in s:
                edge = torch.maximum(pos, s["prefix"][b].long() - 1)
            see &= j <= edge
        if not train:
            see &= j < int(s["length"][b])
        if "seg" in s:
            sg = s["seg"][b]
            see &= (sg[:, None] == sg[None, :]) & (sg[None, :] >= 0)
        some = see.any(1)
        for h in range(H):
            kv = h * Hkv // H
            with torch.set_grad_enabled(train):
                x = (q[b, :, h] @ k[b, :, kv].t()) / math.sqrt(D)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if c["slopes"]:
                    x = x + (-_slopes(H)[h]) * (pos - j).abs().double()
                x = x.where(see, torch.full_like(x, -1e300))
                p = torch.softmax(x, 1) * some[:, None]
                o = p @ v[b, :, kv]
            if train:
                o.backward(s["dout"][b].reshape(Tq, H, D)[:, h].double())
            out[b, :, h] = o.detach()
            del x, p, o
    out = out.reshape(B, Tq, H * D)
    if not train:
        return out
    return [out] + [t.grad.reshape(B, t.shape[1], -1) for t in (q, k, v)]
