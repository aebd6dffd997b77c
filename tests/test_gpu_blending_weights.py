"""What a Gaussian contributes to a view, the sum of alpha * T over the pixels that blend it, against the compositing
restated per pixel in 64 bits, and what the accumulation and the eviction make of it.

Tolerance of the weights: the bar of every gradient here, 1e-4 of the value and 1e-6 of the largest (the weights come out of
the backward blend, which recovers T by divisions)."""
import numpy as np
import pytest
import torch

import synth
from dense_ref import dense_render
from gpu_util import scene_to_torch

pytestmark = pytest.mark.gpu

RAW = ("xyz", "opacity", "scaling", "rotation")


def _raw(sc):
    """The raw parameters of a scene, float32 on the GPU."""
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32, device="cuda:0")
    op = np.clip(sc["opacities"].reshape(-1, 1).astype(np.float64), 1e-3, 1 - 1e-3)
    return dict(xyz=t(sc["means3D"]), opacity=t(np.log(op / (1 - op))), scaling=t(np.log(sc["scales"])), rotation=t(sc["rotations"]) * 1.7)


def _dense_inputs(raw):
    """The activated parameters as the rasterizer gets them, in 64 bits."""
    P = raw["xyz"].shape[0]
    act = dict(means3D=raw["xyz"], opacities=torch.sigmoid(raw["opacity"]), scales=torch.exp(raw["scaling"]),
               rotations=torch.nn.functional.normalize(raw["rotation"]))
    return dict({k: v.detach().cpu().double() for k, v in act.items()}, means2D=torch.zeros(P, 3, dtype=torch.float64))


def _definition(raw, cam, aa):
    """Three Gaussians at a time are painted red, green and blue and all others black, on a black background: the sum
    of a channel is then the sum of its Gaussian's weights."""
    inp = _dense_inputs(raw)
    P = inp["means3D"].shape[0]
    out = torch.zeros(P, dtype=torch.float64)
    for g in range(0, P, 3):
        col = torch.zeros(P, 3, dtype=torch.float64)
        for c in range(min(3, P - g)):
            col[g + c, c] = 1.0
        img = dense_render(dict(inp, colors_precomp=col), cam, (0.0, 0.0, 0.0), 0, antialiasing=aa)["color"]
        out[g:g + 3] = img.sum((1, 2))[:min(3, P - g)]
    return out


def _by_autograd(raw, cam, aa):
    """The same by differentiating the 64-bit image (for more Gaussians)."""
    inp = _dense_inputs(raw)
    col = torch.zeros(inp["means3D"].shape[0], 3, dtype=torch.float64, requires_grad=True)
    dense_render(dict(inp, colors_precomp=col), cam, (0.0, 0.0, 0.0), 0, antialiasing=aa)["color"][1].sum().backward()
    return col.grad[:, 1]


def _close(got, want):
    return bool(((got.cpu().double() - want).abs() <= 1e-4 * want.abs() + 1e-6 * want.abs().max() + 1e-12).all())


@pytest.mark.parametrize("name,kw,aa", [("aa", dict(P=48, width=56, height=40, seed=21, spread=1.2), True),
                                        ("plain", dict(P=48, width=37, height=29, seed=22, spread=1.2, scale=0.3), False),
                                        ("deep", None, True)], ids=["aa", "plain", "deep"])
def test_weights_are_those_of_the_compositing(name, kw, aa):
    from diff_gaussian_rasterization import GaussianRasterizer
    sc = synth.deep_scene(P=120) if kw is None else synth.tiny_scene(**kw)
    rs, _ = scene_to_torch(sc, bg=(0.3, 0.6, 0.1), antialiasing=aa)
    raw = _raw(sc)
    for p in raw.values():
        p.requires_grad_(True)
    r = GaussianRasterizer(rs)
    w = r.blending_weights(*[raw[k] for k in RAW])
    assert w.shape == (len(sc["means3D"]),) and w.dtype == torch.float32 and w.is_contiguous() and not w.requires_grad
    assert all(p.grad is None for p in raw.values())
    want = _definition(raw, sc["camera"], aa)
    assert float(want.max()) > 1 and int((want == 0).sum()) > 0 or kw is None
    assert _close(w, want)
    assert bool((w.cpu()[want == 0] == 0).all()) and bool((w >= 0).all())
    # a pixel's weights sum to what it lets through less than all: the sum over pixels of 1 - T
    color, radii, invd, gsum, gcnt, _ = r(means3D=raw["xyz"].detach(), means2D=torch.zeros_like(raw["xyz"]), opacities=torch.sigmoid(raw["opacity"]).detach(),
                                          colors_precomp=torch.ones_like(raw["xyz"]), scales=torch.exp(raw["scaling"]).detach(),
                                          rotations=torch.nn.functional.normalize(raw["rotation"]).detach())
    dense = dense_render(dict(_dense_inputs(raw), colors_precomp=torch.zeros(w.shape[0], 3, dtype=torch.float64)), sc["camera"], (0, 0, 0), 0, antialiasing=aa)
    covered = float((1.0 - dense["final_T"]).sum())
    assert abs(float(w.double().sum()) - covered) <= 1e-4 * covered and covered <= rs.image_height * rs.image_width
    # what gauss_sum and the opacity give is never less
    bound = torch.sigmoid(raw["opacity"]).detach().view(-1).double() * gsum.double()
    assert bool((w.double() <= bound * (1 + 1e-4) + 1e-6 * float(w.max())).all())


def test_nothing_to_render():
    from diff_gaussian_rasterization import GaussianRasterizer
    sc = synth.tiny_scene(P=10, seed=2)
    rs, _ = scene_to_torch(sc)
    raw = _raw(sc)
    assert GaussianRasterizer(rs).blending_weights(*[raw[k][:0] for k in RAW]).shape == (0,)
    raw["xyz"] = raw["xyz"] * 0 - 100.0     # behind the camera, all of them
    w = GaussianRasterizer(rs).blending_weights(*[raw[k] for k in RAW])
    assert w.shape == (10,) and bool((w == 0).all())


def test_the_eviction_keeps_what_the_images_are_made_of():
    """A splat below a pixel's size of high opacity, and one of several pixels that is nearly transparent: by opacity
    times transmittance over the tested pixels the first weighs more, in the image the second does."""
    import gsplat_optim as G
    from diff_gaussian_rasterization import GaussianRasterizer
    sc = synth.tiny_scene(P=2, width=96, height=96, seed=3)
    sc["means3D"] = np.array([[-0.45, 0.0, 0.0], [0.45, 0.0, 0.0]], np.float32)
    sc["scales"] = np.array([[0.002] * 3, [0.11] * 3], np.float32)
    sc["opacities"] = np.array([[0.95], [0.05]], np.float32)
    sc["camera"] = synth.make_camera(96, 96, 0.9, (0.0, 0.0, -2.5), (0.0, 0.0, 1.0))
    rs, _ = scene_to_torch(sc)
    raw = _raw(sc)
    r = GaussianRasterizer(rs)
    want = _definition(raw, sc["camera"], False)
    assert float(want[1]) > 2 * float(want[0]) > 0
    w = G.accumulate_weights(torch.zeros(2, device="cuda:0"), r.blending_weights(*[raw[k] for k in RAW]))
    assert _close(w, want)
    assert G.evict_rows(w, 1)[0].tolist() == [1]
    gsum = r(means3D=raw["xyz"], means2D=torch.zeros_like(raw["xyz"]), opacities=torch.sigmoid(raw["opacity"]), colors_precomp=torch.ones_like(raw["xyz"]),
             scales=torch.exp(raw["scaling"]), rotations=torch.nn.functional.normalize(raw["rotation"]))[3]
    bound = G.accumulate_weights(torch.zeros(2, device="cuda:0"), gsum, raw["opacity"])
    assert bool((bound >= w * (1 - 1e-4)).all()) and float(bound[0]) > float(bound[1])


def test_a_training_run_evicts_by_its_blending_weights():
    """Views, weights, clipped steps and evictions as a training program strings them together.  The rows are chosen
    exactly as the accumulated weights say, and these are the compositing's, restated in 64 bits from the same parameters."""
    import gsplat_optim as G
    from diff_gaussian_rasterization import GaussianRasterizationSettings, GaussianRasterizer
    dev, W, H, P = "cuda:0", 64, 48, 300
    sc = synth.tiny_scene(P=P, width=W, height=H, seed=21, scale=0.08)
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32, device=dev)
    raw = _raw(sc)
    init = dict(xyz=raw["xyz"], f_dc=t(sc["shs"][:, :1]), f_rest=t(sc["shs"][:, 1:]), opacity=raw["opacity"], scaling=raw["scaling"],
                rotation=raw["rotation"], reps=t(sc["reps"]))
    names = list(init)
    cams = [synth.make_camera(W, H, 0.9, (0.3 * v, -0.05, -2.5), (0.0, 0.0, 1.0)) for v in range(2)]
    settings = [GaussianRasterizationSettings(
        image_height=H, image_width=W, tanfovx=cam["tanfovx"], tanfovy=cam["tanfovy"], bg=torch.zeros(3, device=dev), scale_modifier=1.0,
        viewmatrix=t(cam["viewmatrix"]), projmatrix=t(cam["projmatrix"]), sh_degree=3, campos=t(cam["campos"]), prefiltered=False, debug=False,
        antialiasing=True) for cam in cams]
    params = {k: torch.nn.Parameter(v.detach().clone().contiguous()) for k, v in init.items()}
    opt = G.FusedGaussianAdam([{"params": [params[k]], "lr": 1e-3, "name": k} for k in names], lr=0.0, eps=1e-15)
    for budget, recent in ((250, 20), (180, 0)):
        for it in range(2):
            for rs in settings:
                m2 = torch.zeros_like(params["xyz"], requires_grad=True)
                img = GaussianRasterizer(rs).forward_params(params["xyz"], m2, *[params[k] for k in names[1:]])[0]
                (img.square().mean() * 50).backward()
            opt.clipped_step(0.1)
            opt.zero_grad()
        n = params["xyz"].shape[0]
        weights, plain = torch.zeros(n, device=dev), torch.zeros(n, dtype=torch.float64)
        for rs, cam in zip(settings, cams):
            G.accumulate_weights(weights, [GaussianRasterizer(rs).blending_weights(*[params[k] for k in RAW])], decay=0.9)
            plain = plain * 0.9 + _by_autograd({k: params[k] for k in RAW}, cam, True)
        assert _close(weights, plain)
        old = {k: params[k].detach().clone() for k in names}
        params, rows, new = G.evict_optimizer(opt, weights, budget, recent, dict(weights=weights))
        order = np.lexsort((np.arange(n - recent), -weights[:n - recent].cpu().double().numpy()))
        chosen = np.sort(np.concatenate([order[:budget - recent], np.arange(n - recent, n)]))
        assert np.array_equal(rows.cpu().numpy(), chosen)
        # and by the 64-bit weights no dropped row is heavier than a kept one, but for the tolerance of both
        kept = np.zeros(n, bool)
        kept[chosen] = True
        tol = 1e-4 * plain.numpy() + 1e-6 * float(plain.max()) + 1e-12
        candidates = np.arange(n) < n - recent
        assert (plain.numpy() + tol)[kept & candidates].min() >= (plain.numpy() - tol)[~kept].max()
        assert all(torch.equal(params[k], old[k][rows.long()]) for k in names) and torch.equal(new["weights"], weights[rows.long()])
    assert params["xyz"].shape == (180, 3)
