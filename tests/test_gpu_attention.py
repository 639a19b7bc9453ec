"""Attention (ttsplat.attention), forward and backward, against the formula in 64 bits, on the GPU.

Tolerances, relative to the size of each tensor (its root mean square rms and, entry by entry, its
own value): with u the unit roundoff of the type (2^-24, 2^-11, 2^-8),
  * half types: every entry is rounded once (u |x|) and is a sum of products whose P or dS factor was
    rounded (u a term, signs independent): the error of a sum of n terms is about u times the root
    of the sum of their squares, at most u times the rms-size of the result times a few; D is
    computed from the rounded output.  Entry by entry |err| <= 2 u |x| + 10 u rms, where rms is that
    of the largest tensor row the entry's terms come from; in the mean, rms(err) <= 2 u rms(x).
  * fp32: exp2 of an argument of size a is off by 2^-24 a, with a <= 40 here; sums of up to 1e4
    terms by less than 1e-5: |err| <= 2e-5 (|x| + rms)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def formula(q, k, v, do, mask, causal, scale):
    """out, lse, dq, dk, dv in 64 bits; hidden keys are cut out of the products."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    B, Hq, Nq, D = q.shape
    Hkv, Nk = k.shape[1], k.shape[2]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros(k.shape, **opts(k)), torch.zeros(k.shape, **opts(k))
    lse = torch.full((B, Hq, Nq), -math.inf, **opts(q))
    for b in range(B):
        sel = torch.arange(Nk, device=q.device) if mask is None else mask[b].nonzero().flatten()
        if sel.numel() == 0 or Nq == 0:
            continue
        for h in range(Hq):
            g = h // (Hq // Hkv)
            K, V = k[b, g][sel], v[b, g][sel]
            s = scale * (q[b, h] @ K.T)
            if causal:
                i = torch.arange(Nq, device=q.device)[:, None]
                s = s.masked_fill(sel[None, :] > i + (Nk - Nq), -math.inf)
            L = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - L.masked_fill(L == -math.inf, 0.0))
            lse[b, h] = L[:, 0]
            out[b, h] = p @ V
            dp = do[b, h] @ V.T
            ds = scale * p * (dp - (p * dp).sum(1, keepdim=True))
            dq[b, h] = ds @ K
            dk[b, g].index_add_(0, sel, ds.T @ q[b, h])
            dv[b, g].index_add_(0, sel, p.T @ do[b, h])
    return out, lse, dq, dk, dv


def opts(t):
    return dict(device=t.device, dtype=t.dtype)


def close(got, want, what, dtype):
    assert got.dtype == dtype and got.shape == want.shape, what
    if want.numel() == 0:
        return
    u = U[dtype]
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(err).all()), f"{what}: not finite"
    rms = want.pow(2).mean(-1, keepdim=True).sqrt().amax()    # of the largest row
    lim = 2e-5 * (want.abs() + rms) if dtype == torch.float32 else 2 * u * want.abs() + 10 * u * rms
    assert bool((err <= lim + 1e-30).all()), \
        f"{what}: max err {float(err.max()):.3e}, largest row's rms {float(rms):.3e}"
    if dtype != torch.float32:
        assert float(err.pow(2).mean().sqrt()) <= 2 * u * float(want.pow(2).mean().sqrt()) + 1e-30 \
            + 2.0 ** -24, what


def heads(B, H, N, D, dtype, rows_major, gen):
    if rows_major:
        return torch.randn(B, N, H, D, device="cuda", generator=gen).to(dtype).transpose(1, 2)
    return torch.randn(B, H, N, D, device="cuda", generator=gen).to(dtype)


def inputs(B, Hq, Hkv, Nq, Nk, D, dtype, rows_major=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q, do = (heads(B, Hq, Nq, D, dtype, rows_major, gen) for _ in range(2))
    k, v = (heads(B, Hkv, Nk, D, dtype, rows_major, gen) for _ in range(2))
    return q, k, v, do


def check(q, k, v, do, mask=None, causal=False, scale=None, ref=None):
    from ttsplat import kernels
    from ttsplat.attention import attention
    c = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    ql, kl, vl = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention(ql, kl, vl, mask, causal, scale)
    grads = torch.autograd.grad(out, (ql, kl, vl), do)
    want = ref or formula(q, k, v, do, None if mask is None else mask != 0, causal, c)
    close(out.detach(), want[0], "out", q.dtype)
    for g, w, n in zip(grads, want[2:], ("dq", "dk", "dv")):
        close(g, w, n, q.dtype)
    with torch.no_grad():
        assert torch.equal(attention(q, k, v, mask, causal, scale), out)
    lse = torch.empty(q.shape[:3], device="cuda")
    kernels.attention_fwd(q.contiguous(), k, v, mask, causal, scale, lse=lse)
    w = want[1]
    assert torch.equal(lse == -math.inf, w == -math.inf)
    f = w > -math.inf
    assert bool(((lse.double() - w).abs()[f] <= 2e-5 * (1 + w.abs()[f])).all())
    return out.detach(), grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,Nq,Nk,D", [
    (1, 1, 1, 1, 1, 8), (1, 1, 1, 1, 1, 1), (1, 2, 1, 3, 5, 3), (2, 1, 1, 1, 700, 32),
    (1, 4, 2, 1, 65, 64), (1, 8, 1, 4, 300, 40), (1, 1, 1, 33, 31, 16), (1, 2, 2, 64, 64, 32),
    (2, 3, 1, 65, 129, 72), (1, 1, 1, 128, 128, 64), (1, 6, 2, 131, 257, 128),
    (1, 1, 1, 127, 63, 96), (1, 2, 1, 200, 33, 127), (3, 2, 2, 50, 20, 12), (1, 1, 1, 513, 1, 64),
    (1, 2, 2, 1500, 40, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_sizes(B, Hq, Hkv, Nq, Nk, D, dtype, causal):
    print(f"[attend] B={B} H={Hq}/{Hkv} {Nq}x{Nk} D={D} {dtype} causal={causal}", flush=True)
    check(*inputs(B, Hq, Hkv, Nq, Nk, D, dtype, rows_major=bool((Nq + D) % 2)), causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,Nq,Nk,D,live", [
    (2, 4, 2, 70, 300, 64, 0.5), (3, 2, 1, 1, 1000, 32, 0.1), (2, 2, 2, 300, 77, 96, 0.9),
    (1, 4, 4, 5000, 64, 32, 0.7), (2, 8, 2, 2, 4500, 64, 0.02)])
@pytest.mark.parametrize("causal", [False, True])
def test_key_masks(B, Hq, Hkv, Nq, Nk, D, live, dtype, causal):
    """Random masks; the last batch sees nothing, the first batch's second half is hidden; hidden keys
    hold NaN and infinities, which reach neither the results nor the gradients."""
    print(f"[attend] mask B={B} H={Hq}/{Hkv} {Nq}x{Nk} D={D} {dtype} causal={causal}", flush=True)
    q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, dtype)
    gen = torch.Generator(device="cuda").manual_seed(9)
    mask = torch.rand(B, Nk, device="cuda", generator=gen) < live
    mask[0, Nk // 2:] = False
    if B > 1:
        mask[B - 1] = False
    hole = (~mask)[:, None, :, None]
    k = k.masked_fill(hole, float("nan"))
    v = v.masked_fill(hole, float("inf"))
    _, (dq, dk, dv) = check(q, k, v, do, mask, causal)
    gone = hole.expand_as(dk)
    assert bool((dk[gone] == 0).all()) and bool((dv[gone] == 0).all())
    if B > 1:
        assert bool((dq[B - 1] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,Nq,Nk,D", [(4, 4, 1000, 1000, 64), (6, 2, 531, 1207, 72),
                                             (2, 1, 257, 2500, 128), (4, 4, 20000, 257, 32),
                                             (16, 4, 1, 8040, 64), (2, 2, 3000, 4, 16)])
def test_longer(Hq, Hkv, Nq, Nk, D, dtype):
    print(f"[attend] H={Hq}/{Hkv} {Nq}x{Nk} D={D} {dtype}", flush=True)
    check(*inputs(1, Hq, Hkv, Nq, Nk, D, dtype), causal=Nq < Nk and Nq > 1)


def test_more_queries_than_keys_causal():
    """Rows before the first key see nothing: zeros, no gradient."""
    q, k, v, do = inputs(1, 2, 2, 200, 50, 32, torch.float32)
    out, (dq, _, _) = check(q, k, v, do, causal=True)
    assert bool((out[:, :, :150] == 0).all()) and bool((dq[:, :, :150] == 0).all())


def test_strides():
    """Heads inside a row, a shared batch by stride zero, a slice of wider rows at odd addresses, a last
    axis that is not contiguous, every other position, an expanded gradient."""
    g = torch.Generator(device="cuda").manual_seed(2)
    for dtype in DTYPES:
        qkv = torch.randn(2, 90, 3, 4, 24, device="cuda", generator=g).to(dtype)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        do = torch.randn(2, 4, 90, 24, device="cuda", generator=g).to(dtype)
        check(q, k, v, do)
        check(q, k[:1].expand(2, 4, 90, 24), v[:1].expand(2, 4, 90, 24), do)
        check(q, k[:, :, ::2], v[:, :, 1::2], do)
        check(q[..., 1:18], k[..., 3:20], v[..., 5:22], do[..., :17])
        check(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, do)
        check(q, k, v, do[:, :1, :1].expand(2, 4, 90, 24))


def test_offsets_past_32_bits():
    """Rows a million elements apart: the last ones lie 8 GB behind the first."""
    q, k, v, do = inputs(1, 2, 2, 70, 2100, 32, torch.bfloat16)
    wide = torch.empty(2100, 1 << 21, device="cuda", dtype=torch.bfloat16)   # 8.8 GB, written in part
    views = []
    for i, t in enumerate((k, v)):
        w = wide[:, 4096 * i:4096 * i + 64].view(2100, 2, 32).permute(1, 0, 2)[None]
        w.copy_(t)
        views.append(w)
    check(q, *views, do)
    check(views[0], k[:, :, :90], v[:, :, :90], views[1])       # as query rows and their gradient
    qg = torch.cat([views[0], views[1]], 1)                      # grouped heads over far rows
    check(qg, k[:, :, :50], v[:, :, :50], qg.flip(2))


def test_large_scores():
    """Scores of several hundred: the softmax is taken from each row's maximum; a row's largest few
    keys carry it, and the rest underflow to zero."""
    q, k, v, do = inputs(1, 2, 2, 100, 200, 64, torch.float32)
    from ttsplat.attention import attention
    out = attention(q * 30, k, v)
    want = formula(q * 30, k, v, do, None, False, 0.125)
    # exponents of size 400 * log2(e) carry 2^-24 of that: 4e-5 a probability, and the products' sums
    assert float((out.double() - want[0]).abs().max()) <= 5e-4
    assert bool(torch.isfinite(out).all())


def test_scale():
    q, k, v, do = inputs(1, 2, 1, 60, 90, 32, torch.float32)
    check(q, k, v, do, scale=0.5)
    check(q, k, v, do, scale=0.01)


def test_a_row_with_nan_stays_alone():
    from ttsplat.attention import attention
    q, k, v, _ = inputs(1, 2, 2, 100, 70, 32, torch.bfloat16)
    q = q.clone()
    q[0, 1, 17, 3] = float("nan")
    out = attention(q, k, v)
    bad = ~torch.isfinite(out).all(3)
    assert bad.nonzero().tolist() == [[0, 1, 17]]


def test_no_tokens():
    from ttsplat.attention import attention
    q, k, v, do = inputs(2, 4, 2, 5, 0, 16, torch.bfloat16)
    check(q, k, v, do)
    q, k, v, do = inputs(2, 4, 2, 0, 5, 16, torch.bfloat16)
    check(q, k, v, do)
    assert attention(q[:0], k[:0], v[:0]).shape == (0, 4, 0, 16)


def test_gradients_against_differences():
    """Central differences of the 64-bit loss of the kernel's own fp32 forward, step 1e-2: error
    h^2 / 6 of the third derivative and 2^-24 / h of rounding, well below 1e-2 of the largest."""
    from ttsplat.attention import attention
    q, k, v, do = inputs(1, 2, 1, 3, 4, 8, torch.float32, rows_major=False, seed=4)
    mask = torch.tensor([[True, False, True, True]], device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(attention(*leaves, mask, True), leaves, do)
    for n, g in enumerate(grads):
        num = torch.zeros_like(g)
        for i in range(g.numel()):
            val = []
            for s in (1e-2, -1e-2):
                t = [x.clone() for x in (q, k, v)]
                t[n].view(-1)[i] += s
                val.append((attention(*t, mask, True).double() * do.double()).sum())
            num.view(-1)[i] = float(val[0] - val[1]) / 2e-2
        assert float((num - g).abs().max()) <= 1e-2 * float(g.abs().max())


@pytest.mark.parametrize("Hq,Hkv,Nq,Nk", [(4, 2, 700, 300), (4, 4, 9000, 30), (8, 2, 1, 5000)])
def test_same_bits_and_parts(Hq, Hkv, Nq, Nk):
    """Two runs agree bit for bit, and so does each gradient asked for alone."""
    from ttsplat import kernels
    q, k, v, do = inputs(1, Hq, Hkv, Nq, Nk, 64, torch.bfloat16)
    lse = torch.empty(q.shape[:3], device="cuda")
    out = kernels.attention_fwd(q, k, v, lse=lse)
    ref = kernels.attention_bwd(q, k, v, out, lse, do)
    for need in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        got = kernels.attention_bwd(q, k, v, out, lse, do, need_dq=bool(need[0]),
                                    need_dk=bool(need[1]), need_dv=bool(need[2]))
        for a, b, n in zip(got, ref, need):
            assert torch.equal(a, b) if n else a is None


def test_another_stream_and_graph():
    from ttsplat import kernels
    q, k, v, do = inputs(1, 4, 2, 300, 700, 64, torch.bfloat16)
    mask = torch.rand(1, 700, device="cuda") < 0.6
    lse = torch.empty(q.shape[:3], device="cuda")
    out = kernels.attention_fwd(q, k, v, mask, lse=lse)
    ref = kernels.attention_bwd(q, k, v, out, lse, do, mask)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        o2 = kernels.attention_fwd(q, k, v, mask)
    s.synchronize()
    assert torch.equal(out, o2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3 = kernels.attention_fwd(q, k, v, mask, lse=lse)
        g3 = kernels.attention_bwd(q, k, v, o3, lse, do, mask)
    for _ in range(3):
        o3.zero_()
        [t.zero_() for t in g3]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o3) and all(torch.equal(a, b) for a, b in zip(ref, g3))


def test_refusals():
    from ttsplat import _lib, kernels
    from ttsplat.attention import attention
    q, k, v, do = inputs(1, 4, 2, 5, 6, 16, torch.float32)
    mask = torch.ones(1, 6, dtype=torch.bool, device="cuda")
    wide = torch.zeros(1, 2, 6, 160, device="cuda")
    for bad in (lambda: attention(q.cpu(), k, v), lambda: attention(q.half(), k, v),
                lambda: attention(q.double(), k.double(), v.double()),
                lambda: attention(q[:, :3], k, v), lambda: attention(q, k, v[:, :, :5]),
                lambda: attention(q[0], k, v), lambda: attention(q, k[..., :8], v),
                lambda: attention(wide, wide, wide), lambda: attention(q, k, v, scale=0.0),
                lambda: attention(q, k, v, scale=float("nan")),
                lambda: attention(q, k, v, scale=-1.0),
                lambda: attention(q, k, v, mask[:, :5]), lambda: attention(q, k, v, mask.float()),
                lambda: attention(q, k, v, mask.cpu()),
                lambda: kernels.attention_fwd(q.transpose(2, 3), k, v),
                lambda: kernels.attention_fwd(q, k, v, lse=torch.zeros(1, 4, 6, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    shape = kernels._attn_shape(q, k, v, q, None, False, 0.25, q, q, k, v)
    with pytest.raises(_lib.TTSError):       # no workspace
        _lib.call("tts_attention_bwd", shape, *(_lib.ptr(t) for t in (q, k, v)), None,
                  _lib.ptr(q), None, _lib.ptr(q), _lib.ptr(q), _lib.ptr(q), None, None, None, 0,
                  _lib.stream())
