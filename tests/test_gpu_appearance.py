"""View-dependent colours by codes, norms and attention (ttsplat.appearance): the network against
the same formulas in 64 bits, and a scene fitted to views of different looks.

Tolerances are those of the framework's renders: values within 1e-4 of the largest, gradients
within 1e-3 relative L2 (fp32); bf16 rows carry 2^-8 a rounding and a handful of them follow one
another: 2e-2 and 5e-2."""
import math

import pytest
import torch

from helpers import config_inputs, rel_l2
from ttsplat import binned
from ttsplat.model import GaussianModel

pytestmark = pytest.mark.gpu


def norm64(x, wb):
    m = x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5) * wb[0] + wb[1]


def offsets64(app, leaves, ids, view, mask):
    p = dict(zip(app.names, leaves))
    ok = ids >= 0
    x = torch.where(ok[:, None], p["codes"][ids.clamp(min=0).long()], 0.0) * app.scale
    t = norm64(p["views"][view * app.tokens:(view + 1) * app.tokens] * app.scale, p["norm_t"])
    h = norm64(x, p["norm_x"])
    H, Hk = app.heads, app.kv_heads
    q = (h @ p["wq"]).view(len(ids), H, -1)
    k = (t @ p["wk"]).view(app.tokens, Hk, -1).repeat_interleave(H // Hk, 1)
    v = (t @ p["wv"]).view(app.tokens, Hk, -1).repeat_interleave(H // Hk, 1)
    s = torch.einsum("ghd,thd->ght", q, k) / math.sqrt(q.shape[2])
    if mask is not None:
        s = s.masked_fill(~mask[None, None, :], -math.inf)
    o = torch.einsum("ght,thd->ghd", torch.softmax(s, 2), v).reshape(len(ids), -1)
    return norm64(x + o @ p["wo"], p["norm_y"]) @ p["wc"]


@pytest.mark.parametrize("dtype,vtol,gtol", [(torch.float32, 1e-4, 1e-3), (torch.bfloat16, 2e-2, 5e-2)])
@pytest.mark.parametrize("masked", [False, True])
def test_network_against_64_bits(dtype, vtol, gtol, masked):
    from ttsplat.appearance import Appearance
    app = Appearance(50, 3, tokens=9, width=48, heads=6, kv_heads=2, dtype=dtype, seed=1)
    with torch.no_grad():
        app.wc.copy_(torch.randn(48, 3, generator=torch.Generator().manual_seed(2)) * 0.2)
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, 50, (777,), generator=gen).to(torch.int32).cuda()
    mask = torch.tensor([1, 1, 0, 1, 1, 0, 1, 1, 1], dtype=torch.bool).cuda() if masked else None
    R = torch.randn(777, 3, generator=gen).cuda()
    out = app.offsets(ids, 1, mask)
    grads = torch.autograd.grad((out * R).sum(), app.leaves())
    l64 = [t.detach().double().requires_grad_(True) for t in app.leaves()]
    ref = offsets64(app, l64, ids, 1, mask)
    rgrads = torch.autograd.grad((ref * R.double()).sum(), l64)
    assert float((out.double() - ref).abs().max()) <= vtol * float(ref.abs().max())
    for n, g, r in zip(app.names, grads, rgrads):
        assert rel_l2(g, r) <= gtol, n


def test_a_scene_of_two_looks():
    """Two views of a scene, one of them tinted and darker: the network learns the difference, which
    one set of colours cannot show, and the dress of each view stays its own."""
    from ttsplat.appearance import Appearance, cell_codes, fit_appearance
    cfg, P, cam = config_inputs("c1_ref")
    model = GaussianModel(P.cuda())
    tint = P.clone()
    tint[:, 10:13] += torch.tensor([-0.9, -0.2, 0.5])
    tmap = binned.TileMap(cam.H, cam.W)
    with torch.no_grad():
        looks = [binned.render_binned_device(GaussianModel(p.cuda()), cam, tmap) for p in (P, tint)]
    app = Appearance(64, 2, tokens=4, width=32, heads=4)
    ids = cell_codes(model.means3d, 64, cell=0.5)
    assert ids.dtype == torch.int32 and int(ids.min()) >= 0 and int(ids.max()) < 64
    before = model.params.clone()
    history = fit_appearance(model, app, ids, [cam, cam], looks, iters=120)
    assert torch.equal(model.params, before)
    assert history[-1] < 0.25 * history[0], history[::20]
    with torch.no_grad():
        imgs = [binned.render_binned_device(app.dress(model, ids, i), cam, tmap) for i in range(2)]
    for i in range(2):
        own = float((imgs[i] - looks[i]).abs().mean())
        other = float((imgs[i] - looks[1 - i]).abs().mean())
        assert own < 0.5 * other


def test_zero_start_and_refusals():
    from ttsplat.appearance import Appearance, cell_codes
    app = Appearance(8, 2)
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    assert torch.equal(app.offsets(ids, 0), torch.zeros(5, 3, device="cuda"))
    for bad in (lambda: app.offsets(ids, 2), lambda: Appearance(8, 2, width=30, heads=4),
                lambda: Appearance(8, 2, heads=4, kv_heads=3), lambda: Appearance(0, 2),
                lambda: Appearance(8, 2, dtype=torch.float64),
                lambda: cell_codes(torch.zeros(3, 3), 0, 1.0)):
        with pytest.raises(ValueError):
            bad()
    m = torch.tensor([[0.1, 0.2, 0.3], [float("nan"), 0.0, 0.0]])
    assert cell_codes(m, 4, 0.5).tolist()[1] == -1
