"""Operators of networks beside a scene: attention, layer norm and embedding lookup, as timed cases.

Three kinds of calls, each with or without its gradients:

  attend  ttsplat.attention.attention: gaussians or view tokens (queries) over a view's tokens
  norm    ttsplat.norm.layer_norm: one row of features a gaussian or token
  embed   ttsplat.embedding.embedding: codes of gaussians or view tokens from a table

Token counts are those of the benchmark scenes: gaussians (2000, 100 000, 1 000 000) and 16x16
image tiles (64 at 128x128, 2500 at 800x800, 8040 at 1920x1072).  Where `own` is false `run` takes
the plain formulas in 32 bits; where it is true, the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # Serving: one new token a view over its frame's 8040 tile tokens, shared key heads.
        dict(name="attend_1x8040_bf16", kind="attend", B=8, Hq=8, Hkv=2, Nq=1, Nk=8040, D=64,
             dtype="bf16", causal=False, live=0.9, rows_major=True, grad=False),
        # The smallest scene in the framework's own type: 2000 gaussians over the 64 tile tokens of
        # a 128x128 view, forward and gradients.
        dict(name="attend_2000x64_fp32_grad", kind="attend", B=1, Hq=4, Hkv=4, Nq=2000, Nk=64,
             D=32, dtype="fp32", causal=False, live=1.0, rows_major=True, grad=True),
        # A headline scene's gaussians over an odd number of view tokens, some left out.
        dict(name="attend_100kx257_bf16_grad", kind="attend", B=1, Hq=4, Hkv=4, Nq=100000, Nk=257,
             D=32, dtype="bf16", causal=False, live=0.75, rows_major=True, grad=True),
        # Tile tokens of two 800x800 views among themselves.
        dict(name="attend_2500x2500_bf16_grad", kind="attend", B=2, Hq=8, Hkv=8, Nq=2500, Nk=2500,
             D=64, dtype="bf16", causal=False, live=1.0, rows_major=False, grad=True),
        # Tokens in order, the new ones behind a longer past; odd lengths and head size.
        dict(name="attend_531x1207_fp16_grad", kind="attend", B=3, Hq=6, Hkv=2, Nq=531, Nk=1207,
             D=72, dtype="fp16", causal=True, live=1.0, rows_major=True, grad=True),
        # The largest frame's tile tokens among themselves, shared key heads, some tiles left out.
        dict(name="attend_8040x8040_bf16_grad", kind="attend", B=1, Hq=16, Hkv=4, Nq=8040, Nk=8040,
             D=128, dtype="bf16", causal=False, live=0.9, rows_major=True, grad=True),
        # A handful of tokens: latency.
        dict(name="norm_64x64_fp32", kind="norm", R=64, D=64, dtype="fp32", wtype="fp32",
             grad=False),
        # Wide rows of an odd size, forward and gradients.
        dict(name="norm_8040x1003_fp16_grad", kind="norm", R=8040, D=1003, dtype="fp16",
             wtype="fp16", grad=True),
        # A row for each of a million gaussians, weights held in 32 bits.
        dict(name="norm_1mx64_bf16_grad", kind="norm", R=1000000, D=64, dtype="bf16",
             wtype="fp32", grad=True),
        # The codes of one view's tokens: latency.
        dict(name="embed_257_fp32", kind="embed", N=257, V=1000, D=64, dtype="fp32", grad=False),
        # A code for each gaussian of the headline scene, a few codes shared by many.
        dict(name="embed_100k_fp32_grad", kind="embed", N=100000, V=4096, D=32, dtype="fp32",
             grad=True),
        # A million gaussians and a large table.
        dict(name="embed_1m_bf16_grad", kind="embed", N=1000000, V=100003, D=128, dtype="bf16",
             grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    kind = rng.choice(["attend", "attend", "norm", "embed"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    grad = rng.random() < 0.7
    if kind == "norm":
        D = _log(rng, 1, 4096)
        return dict(kind="norm", R=_log(rng, 1, min(1000000, 64000000 // D)), D=D, dtype=dtype,
                    wtype=rng.choice([dtype, "fp32"]), grad=grad)
    if kind == "embed":
        D = _log(rng, 1, 512)
        return dict(kind="embed", N=_log(rng, 1, min(1000000, 128000000 // D)),
                    V=_log(rng, 1, 100003), D=D, dtype=dtype, grad=grad)
    while True:
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 1, 2, 3, 4])
        B = rng.choice([1, 1, 2, 3, 8])
        shape = rng.choice(["few", "cross", "self"])
        Nk = _log(rng, 1, 8040)
        Nq = _log(rng, 1, 8) if shape == "few" else _log(rng, 1, 8040)
        if shape == "cross":
            Nq, Nk = _log(rng, 100, 100000), _log(rng, 1, 512)
        D = rng.choice([8, 16, 32, 40, 64, 64, 72, 96, 128])
        cost = B * Hq * Nq * Nk * D * (16 if dtype == "fp32" else 1)
        if cost <= 16 * 8040 * 8040 * 128 and B * Hq * Nq * D <= 100000000:
            return dict(kind="attend", B=B, Hq=Hq, Hkv=Hkv, Nq=Nq, Nk=Nk, D=D, dtype=dtype,
                        causal=rng.random() < 0.3, live=rng.choice([1.0, 1.0, 0.9, 0.5]),
                        rows_major=rng.random() < 0.6, grad=grad)


# ------------------------------------------------------------------------------------ inputs --
def _heads(B, H, N, D, dtype, rows_major, gen):
    """[B, H, N, D]; rows_major: a view of memory ordered [B, N, H, D]."""
    if rows_major:
        t = torch.randn(B, N, H, D, device="cuda", generator=gen).to(dtype)
        return t.transpose(1, 2)
    return torch.randn(B, H, N, D, device="cuda", generator=gen).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    st = dict(case=case)
    if case["kind"] == "attend":
        B, D, rm = case["B"], case["D"], case["rows_major"]
        st["q"] = _heads(B, case["Hq"], case["Nq"], D, dt, rm, gen)
        st["k"] = _heads(B, case["Hkv"], case["Nk"], D, dt, rm, gen)
        st["v"] = _heads(B, case["Hkv"], case["Nk"], D, dt, rm, gen)
        st["do"] = _heads(B, case["Hq"], case["Nq"], D, dt, rm, gen) if case["grad"] else None
        st["mask"] = None
        if case["live"] < 1.0:
            st["mask"] = torch.rand(B, case["Nk"], device="cuda", generator=gen) < case["live"]
        leaves = ("q", "k", "v")
    elif case["kind"] == "norm":
        R, D = case["R"], case["D"]
        # rows away from zero mean, as features after a few layers are
        st["x"] = (torch.randn(R, D, device="cuda", generator=gen) * 1.5
                   + torch.randn(R, 1, device="cuda", generator=gen)).to(dt)
        wt = _DT[case["wtype"]]
        st["w"] = (1 + 0.1 * torch.randn(D, device="cuda", generator=gen)).to(wt)
        st["b"] = (0.1 * torch.randn(D, device="cuda", generator=gen)).to(wt)
        st["dy"] = (torch.randn(R, D, device="cuda", generator=gen).to(dt)
                    if case["grad"] else None)
        leaves = ("x", "w", "b")
    else:
        N, V, D = case["N"], case["V"], case["D"]
        st["table"] = torch.randn(V, D, device="cuda", generator=gen).to(dt)
        # a few codes shared by many, and 2 % of the entries without a code (-1)
        u = torch.rand(N, device="cuda", generator=gen)
        ids = ((V * u.pow(4)).long().clamp(max=V - 1) * 7919) % V
        none = torch.rand(N, device="cuda", generator=gen) < 0.02
        st["ids"] = torch.where(none, torch.full_like(ids, -1), ids).to(torch.int32)
        st["scale"] = math.sqrt(D)
        st["dy"] = (torch.randn(N, D, device="cuda", generator=gen).to(dt)
                    if case["grad"] else None)
        leaves = ("table",)
    if case["grad"]:
        for n in leaves:
            st[n] = st[n].detach().requires_grad_(True)
    return st


# -------------------------------------------------------------------------------- the passes --
def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"attend": _plain_attend, "norm": _plain_norm, "embed": _plain_embed}[
            state["case"]["kind"]](state)


def _own(st):
    pkg = os.path.join(os.getcwd(), "tt-splat_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    case = st["case"]
    if case["kind"] == "attend":
        from ttsplat.attention import attention
        out = attention(st["q"], st["k"], st["v"], key_mask=st["mask"], causal=case["causal"])
        if not case["grad"]:
            return dict(out=out)
        dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"])
        return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)
    if case["kind"] == "norm":
        from ttsplat.norm import layer_norm
        y = layer_norm(st["x"], st["w"], st["b"])
        if not case["grad"]:
            return dict(out=y)
        dx, dw, db = torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"])
        return dict(out=y.detach(), dx=dx, dw=dw, db=db)
    from ttsplat.embedding import embedding
    y = embedding(st["table"], st["ids"], scale=st["scale"])
    if not case["grad"]:
        return dict(out=y)
    (dt,) = torch.autograd.grad(y, (st["table"],), st["dy"])
    return dict(out=y.detach(), dtable=dt)


def _plain_attend(st):
    case, q, k, v, do = st["case"], st["q"], st["k"], st["v"], st["do"]
    B, Hq, Hkv, Nq, Nk, D = (case[n] for n in ("B", "Hq", "Hkv", "Nq", "Nk", "D"))
    grp, c = Hq // Hkv, 1.0 / math.sqrt(D)
    qf = q.float().reshape(B * Hkv, grp * Nq, D)
    kf = k.float().reshape(B * Hkv, Nk, D)
    vf = v.float().reshape(B * Hkv, Nk, D)
    dof = do.float().reshape(B * Hkv, grp * Nq, D) if case["grad"] else None
    o = torch.empty_like(qf)
    dq, dk, dv = ((torch.empty_like(qf), torch.empty_like(kf), torch.empty_like(vf))
                  if case["grad"] else (None, None, None))
    step = max(1, (1 << 28) // max(1, grp * Nq * Nk))       # heads at once, by their scores' size
    for a in range(0, B * Hkv, step):
        z = min(a + step, B * Hkv)
        s = torch.matmul(qf[a:z], kf[a:z].transpose(1, 2).contiguous()) * c
        if st["mask"] is not None:
            m = st["mask"].repeat_interleave(Hkv, 0)[a:z, None, :]
            s = s.masked_fill(~m, -math.inf)
        if case["causal"]:
            i = torch.arange(Nq, device=q.device).repeat(grp)[:, None]
            j = torch.arange(Nk, device=q.device)[None, :]
            s = s.masked_fill(j > i + (Nk - Nq), -math.inf)
        top = s.max(2, keepdim=True).values
        p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
        tot = p.sum(2, keepdim=True)
        p = p / tot.masked_fill(tot == 0, 1.0)
        o[a:z] = torch.matmul(p, vf[a:z])
        if case["grad"]:
            dv[a:z] = torch.matmul(p.transpose(1, 2).contiguous(), dof[a:z])
            dp = torch.matmul(dof[a:z], vf[a:z].transpose(1, 2).contiguous())
            ds = p * (dp - (dof[a:z] * o[a:z]).sum(2, keepdim=True)) * c
            dq[a:z] = torch.matmul(ds, kf[a:z])
            dk[a:z] = torch.matmul(ds.transpose(1, 2).contiguous(), qf[a:z])
    out = dict(out=o.reshape(q.shape).to(q.dtype))
    if case["grad"]:
        out.update(dq=dq.reshape(q.shape).to(q.dtype), dk=dk.reshape(k.shape).to(k.dtype),
                   dv=dv.reshape(v.shape).to(v.dtype))
    return out


def _plain_norm(st):
    x, w, b = st["x"].float(), st["w"].float(), st["b"].float()
    m = x.mean(1, keepdim=True)
    xc = x - m
    r = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
    xh = xc * r
    out = dict(out=(xh * w + b).to(st["x"].dtype))
    if st["case"]["grad"]:
        dy = st["dy"].float()
        g = dy * w
        dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out.update(dx=dx.to(st["x"].dtype), dw=(dy * xh).sum(0).to(st["w"].dtype),
                   db=dy.sum(0).to(st["b"].dtype))
    return out


def _plain_embed(st):
    table, ids, s = st["table"], st["ids"].long(), st["scale"]
    V = table.shape[0]
    ok = (ids >= 0) & (ids < V)
    y = table[ids.clamp(0, V - 1)].float() * s
    out = dict(out=torch.where(ok[:, None], y, torch.zeros_like(y)).to(table.dtype))
    if st["case"]["grad"]:
        dt = torch.zeros(V + 1, table.shape[1], device=table.device)
        dt.index_add_(0, torch.where(ok, ids, torch.full_like(ids, V)), st["dy"].float())
        out["dtable"] = (dt[:V] * s).to(table.dtype)
    return out


# ---------------------------------------------------------------------- the formulas in 64 bits --
@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, st)
    if case["kind"] == "norm":
        x = st["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        n = (x - mean) / sd
        res = dict(out=n * st["w"].double() + st["b"].double())
        if case["grad"]:
            g = st["dy"].double()
            gw = g * st["w"].double()
            proj = (gw * n).sum(1, keepdim=True) / case["D"]
            res.update(dx=(gw - gw.sum(1, keepdim=True) / case["D"] - n * proj) / sd,
                       dw=torch.einsum("rd,rd->d", g, n), db=g.sum(0))
        return res
    ids, V = st["ids"].long(), case["V"]
    known = ((ids >= 0) & (ids < V)).nonzero().flatten()
    res = dict(out=torch.zeros(case["N"], case["D"], device="cuda", dtype=torch.float64))
    res["out"][known] = st["table"].double()[ids[known]] * st["scale"]
    if case["grad"]:
        acc = torch.zeros(V, case["D"], device="cuda", dtype=torch.float64)
        acc.index_put_((ids[known],), st["dy"].double()[known] * st["scale"], accumulate=True)
        res["dtable"] = acc
    return res


def _exact_attend(case, st):
    q, k, v = st["q"], st["k"], st["v"]
    B, Hq, Hkv, Nq, Nk, D = (case[n] for n in ("B", "Hq", "Hkv", "Nq", "Nk", "D"))
    res = dict(out=torch.zeros(q.shape, device="cuda", dtype=torch.float64))
    if case["grad"]:
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            res[n] = torch.zeros(t.shape, device="cuda", dtype=torch.float64)
    rows = max(1, (1 << 26) // Nk)
    for b in range(B):
        for h in range(Hq):
            g = h // (Hq // Hkv)
            K, Vv = k[b, g].double(), v[b, g].double()
            for a in range(0, Nq, rows):
                Q = q[b, h, a:a + rows].double()
                n = Q.shape[0]
                seen = torch.ones(n, Nk, dtype=torch.bool, device="cuda")
                if st["mask"] is not None:
                    seen &= st["mask"][b]
                if case["causal"]:
                    pos = torch.arange(a, a + n, device="cuda") + Nk - Nq
                    seen &= torch.arange(Nk, device="cuda") <= pos[:, None]
                sc = (Q @ K.T) / D ** 0.5
                sc = torch.where(seen, sc, torch.full_like(sc, -math.inf))
                lse = torch.logsumexp(sc, 1)
                pr = torch.where(seen, torch.exp(sc - lse[:, None]), torch.zeros_like(sc))
                O = pr @ Vv
                res["out"][b, h, a:a + n] = O
                if case["grad"]:
                    G = st["do"][b, h, a:a + n].double()
                    res["dv"][b, g] += pr.T @ G
                    t = G @ Vv.T
                    t = pr * (t - (t * pr).sum(1)[:, None]) / D ** 0.5
                    res["dq"][b, h, a:a + n] = t @ K
                    res["dk"][b, g] += t.T @ Q
    return res


# ------------------------------------------------------------------------------------- floors --
def work(case):
    """Bytes and flops one pass cannot do without."""
    e = _SIZE[case["dtype"]]
    if case["kind"] == "norm":
        R, D = case["R"], case["D"]
        wb = 2 * D * _SIZE[case["wtype"]]
        if not case["grad"]:
            return {"bytes": 2 * R * D * e + wb, "flops": 8 * R * D}
        return {"bytes": 4 * R * D * e + 2 * wb, "flops": 24 * R * D}
    if case["kind"] == "embed":
        N, V, D = case["N"], case["V"], case["D"]
        # distinct rows of the table that the draw reaches, at most
        rows = min(N, V)
        if not case["grad"]:
            return {"bytes": 4 * N + (rows + N) * D * e, "flops": N * D}
        return {"bytes": 4 * N + (rows + 2 * N + V) * D * e, "flops": 2 * N * D}
    B, Hq, Hkv, Nq, Nk, D = (case[n] for n in ("B", "Hq", "Hkv", "Nq", "Nk", "D"))
    if case["causal"]:
        lo, hi = Nk - Nq + 1, Nk                    # keys of the first and the last row
        n = min(Nq, hi)
        pairs = n * (max(lo, 1) + hi) / 2.0
    else:
        pairs = Nq * Nk
    pairs *= B * Hq * case["live"]
    qo, kv = B * Hq * Nq * D * e, B * Hkv * Nk * D * e
    if not case["grad"]:
        return {"bytes": 2 * qo + 2 * kv, "flops": 4 * pairs * D}
    return {"bytes": 4 * qo + 4 * kv, "flops": 14 * pairs * D}
