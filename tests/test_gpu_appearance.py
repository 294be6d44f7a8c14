"""GPU checks of the decode with the row tables: the colour head conditioned on a camera's learned row
(appearance_dim > 0), its gradients, and a model rendered from features held in 8 bits."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from horizongs_amd import decode as HD
from horizongs_amd import embedding as E
from horizongs_amd import rowcache as R
from oracle import decode_ref as D
from oracle.checks import close, cond_close

pytestmark = pytest.mark.gpu
DEV = "cuda"
APP, N_OFF, F = 16, 10, 32


def model(A, n_cam, view_dim, color_dim, seed, scale=1.0):
    """An anchor model of the reference's shape, with an appearance table, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, sd=1.0: torch.randn(*s, generator=g) * sd
    k = F + view_dim
    t = dict(anchor=r(A, 3, sd=2.0), feat=r(A, F, sd=0.3), offset=r(A, N_OFF, 3, sd=0.1),
             scaling_raw=np.log(0.01) + r(A, 6, sd=0.1), table=r(n_cam, APP))
    for h, o, kk in (("opacity", N_OFF, k), ("cov", 7 * N_OFF, k), ("color", color_dim * N_OFF, k + APP)):
        t.update({f"{h}_w1": r(F, kk, sd=kk ** -0.5), f"{h}_b1": r(F, sd=0.1), f"{h}_w2": r(o, F, sd=F ** -0.5),
                  f"{h}_b2": r(o, sd=0.1)})
    return t


def head(t, h, tanh=False):
    def lin(w, b):
        m = torch.nn.Linear(w.shape[1], w.shape[0], device=DEV)
        m.weight.data.copy_(w), m.bias.data.copy_(b)
        return m
    seq = [lin(t[f"{h}_w1"], t[f"{h}_b1"]), torch.nn.ReLU(), lin(t[f"{h}_w2"], t[f"{h}_b2"])]
    return torch.nn.Sequential(*seq, *([torch.nn.Tanh()] if tanh else []))


def as_object(t, view_dim, color_dim, scale):
    p = lambda x: torch.nn.Parameter(x.to(DEV))
    table = E.Embedding(t["table"].shape[0], APP, scale, device=DEV)
    table.embedding.weight.data.copy_(t["table"])
    return SimpleNamespace(get_anchor=p(t["anchor"]), get_anchor_feat=p(t["feat"]), get_offset=p(t["offset"]),
                           _scaling=p(t["scaling_raw"]), get_opacity_mlp=head(t, "opacity", True),
                           get_cov_mlp=head(t, "cov"), get_color_mlp=head(t, "color"), view_dim=view_dim,
                           n_offsets=N_OFF, color_dim=color_dim, active_sh_degree=0, appearance_dim=APP,
                           embedding_appearance=table)


CAM = torch.tensor([0.3, -0.5, 6.0])


def formula(t, uid, scale, view_dim, color_dim, vis, dtype):
    """The decode with the row written out to every anchor, as the model defines it; t: leaves."""
    c = {k: v.to(dtype).requires_grad_(True) for k, v in t.items()}
    a, f = c["anchor"][vis], c["feat"][vis]
    mlps = {k: v for k, v in c.items() if k.endswith(("w1", "w2", "b1", "b2"))}
    plain = dict(mlps, color_w1=mlps["color_w1"][:, :F + view_dim])
    xyz, offs, _, op, sc, rot, mask = D.decode_torch(a, f, c["offset"][vis], c["scaling_raw"][vis], CAM.to(dtype), plain,
                                                     view_dim, N_OFF, color_dim)
    v = a - CAM.to(dtype)
    x = torch.cat([f, v / v.norm(dim=1, keepdim=True)], 1) if view_dim else f
    row = c["table"][uid] * scale if 0 <= uid < t["table"].shape[0] else torch.zeros(APP, dtype=dtype)
    x = torch.cat([x, row.expand(x.shape[0], APP)], 1)
    h = torch.relu(x @ mlps["color_w1"].T + mlps["color_b1"])
    col = (h @ mlps["color_w2"].T + mlps["color_b2"]).reshape(-1, color_dim)[mask]
    return c, (xyz, offs, col, op, sc, rot, mask)


@pytest.mark.parametrize("view_dim,color_dim,uid,scale", [(3, 3, 4, 1.0), (0, 3, 0, 0.5), (3, 27, 7, 4.0), (3, 3, 99, 1.0)])
def test_appearance_conditioned_decode(view_dim, color_dim, uid, scale):
    A, n_cam = 700, 8
    t = model(A, n_cam, view_dim, color_dim, seed=uid + color_dim)
    vis = torch.rand(A, generator=torch.Generator().manual_seed(1)) < 0.6
    m = as_object(t, view_dim, color_dim, scale)
    cam = SimpleNamespace(camera_center=CAM.to(DEV), uid=uid)
    xyz, offs, col, op, sc, rot, _, mask = HD.generate_neural_gaussians(m, cam, vis.to(DEV))
    col = col.reshape(col.shape[0], -1)
    c64, w64 = formula(t, uid, scale, view_dim, color_dim, vis, torch.float64)
    c32, w32 = formula(t, uid, scale, view_dim, color_dim, vis, torch.float32)
    np.testing.assert_array_equal(mask.cpu().numpy(), w64[6].numpy())
    for name, got, want in zip(("xyz", "offs", "color", "opacity", "scaling", "rot"), (xyz, offs, col, op, sc, rot), w64):
        close(got.detach().cpu().numpy(), want.detach().numpy(), name=name)
    # gradients of the whole run: table row, both parts of the colour head, every other leaf
    g = torch.Generator().manual_seed(5)
    cs = [torch.randn(w.shape, generator=g, dtype=torch.float64) for w in (w64[0], w64[2], w64[3], w64[4], w64[5])]
    pick = lambda o: (o[0], o[2], o[3], o[4], o[5])
    sum((x * c.float().to(DEV)).sum() for x, c in zip((xyz, col, op, sc, rot), cs)).backward()
    sum((x * c).sum() for x, c in zip(pick(w64), cs)).backward()
    sum((x * c.float()).sum() for x, c in zip(pick(w32), cs)).backward()
    got = {"table": m.embedding_appearance.embedding.weight.grad, "feat": m.get_anchor_feat.grad,
           "offset": m.get_offset.grad, "anchor": m.get_anchor.grad, "scaling_raw": m._scaling.grad}
    for h, mod in (("opacity", m.get_opacity_mlp), ("cov", m.get_cov_mlp), ("color", m.get_color_mlp)):
        got.update({f"{h}_w1": mod[0].weight.grad, f"{h}_b1": mod[0].bias.grad, f"{h}_w2": mod[2].weight.grad,
                    f"{h}_b2": mod[2].bias.grad})
    for k, v in got.items():
        a, b = c32[k].grad, c64[k].grad
        a, b = (torch.zeros_like(c64[k]), torch.zeros_like(c64[k])) if b is None else (a, b)
        cond_close(v.cpu().numpy(), a.numpy(), b.numpy(), k)
    rest = torch.ones(n_cam, dtype=torch.bool)
    if uid < n_cam:
        rest[uid] = False
    assert not got["table"].cpu()[rest].any()  # the other cameras' rows


def test_appearance_id_and_adam():
    """Another camera's row by appearance_id; a few fused Adam steps move the rendered cameras' rows only."""
    from horizongs_amd.optim import Adam
    t = model(300, 6, 3, 3, seed=2)
    m = as_object(t, 3, 3, 1.0)
    cam = lambda u: SimpleNamespace(camera_center=CAM.to(DEV), uid=u)
    with torch.no_grad():
        a = HD.generate_neural_gaussians(m, cam(5))[2]
        b = HD.generate_neural_gaussians(m, cam(0), appearance_id=5)[2]
        c = HD.generate_neural_gaussians(m, cam(0))[2]
    assert torch.equal(a, b) and not torch.equal(a, c)
    w = m.embedding_appearance.embedding.weight
    opt, before = Adam([w], lr=0.1, eps=1e-15), w.detach().clone()
    for u in (1, 3):
        HD.generate_neural_gaussians(m, cam(u))[2].sum().backward()
        opt.step()
        opt.zero_grad()
    moved = (w != before).any(1).cpu()
    assert moved.tolist() == [False, True, False, True, False, False]


def test_unfit_appearance_is_refused():
    t = model(20, 3, 3, 3, seed=0)
    w = {k: v.to(DEV) for k, v in t.items()}
    args = (w["anchor"], w["feat"], w["offset"], w["scaling_raw"], CAM.to(DEV), w)
    with pytest.raises(ValueError, match="appearance row"):
        HD.decode(*args)
    with pytest.raises(ValueError, match="does not fit"):
        HD.decode(*args, appearance=torch.zeros(APP + 1, device=DEV))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decode_from_a_row_cache(fmt):
    """A model written into a cache decodes as the model whose features are what the cache holds."""
    A = 900
    t = {k: v.to(DEV) for k, v in model(A, 4, 3, 3, seed=9).items()}
    cache = R.rowcache_alloc(A, F, fmt, 32, DEV)
    order = torch.randperm(A, device=DEV)
    for part in order.split(250):  # chunk by chunk, in any order
        R.rowcache_write(cache, t["feat"][part], part)
    feat = R.rowcache_read(cache)
    row = E.embedding(t["table"], torch.tensor([2], device=DEV))[0]
    vis = torch.rand(A, device=DEV) < 0.5
    idx = torch.nonzero(vis).reshape(-1)
    buf = torch.full((A,), -7, dtype=torch.int32, device=DEV)
    buf[:idx.numel()] = idx.int()
    lazy = HD.VisibleIndex(buf, torch.tensor([0, idx.numel()], device=DEV), vis)
    for v in (None, vis, idx, lazy):
        a = HD.decode(t["anchor"], cache, t["offset"], t["scaling_raw"], CAM.to(DEV), t, v, appearance=row)
        b = HD.decode(t["anchor"], feat, t["offset"], t["scaling_raw"], CAM.to(DEV), t,
                      idx if v is lazy else v, appearance=row)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    with pytest.raises(NotImplementedError, match="rendering"):
        HD.decode(t["anchor"].clone().requires_grad_(True), cache, t["offset"], t["scaling_raw"], CAM.to(DEV), t, vis,
                  appearance=row)
    with pytest.raises(ValueError, match="slots"):
        HD.decode(t["anchor"], R.rowcache_alloc(3, F, fmt, 32, DEV), t["offset"], t["scaling_raw"], CAM.to(DEV), t,
                  appearance=row)
