"""Accumulated blending weights and the eviction to a row budget, against plain formulations: the weights in 64 bits,
the selection with a stable sort on the CPU (exact), the copied rows bit for bit."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("N", [1, 3, 255, 256, 257, 70001])
@pytest.mark.parametrize("views", [0, 1, 2, 8, 9, 33, 70])
@pytest.mark.parametrize("opacity", [None, 1, 2])
def test_accumulated_weights(N, views, opacity):
    """Roundings: views - 1 additions of non-negative terms, the sigmoid's exponential (one unit in the last place,
    2u), its sum and the quotient, the decay and its product, the sum, and views / 32 more sums and products where the
    views take several passes."""
    import gsplat_optim as G
    gen = torch.Generator(device="cuda").manual_seed(N * 100 + views)
    w = torch.rand(N, device="cuda", generator=gen) * 10
    c = [torch.rand(N, device="cuda", generator=gen) * 100 * (torch.rand(N, device="cuda", generator=gen) < 0.5) for _ in range(views)]
    o = None if opacity is None else torch.randn((N, 1)[:opacity] if opacity == 2 else (N,), device="cuda", generator=gen) * 4
    before = w.double()
    add = sum((x.double() for x in c), torch.zeros(N, dtype=torch.float64, device="cuda"))
    if o is not None:
        add = add * torch.sigmoid(o.double().view(-1))
    want = before * 0.9 + add
    assert G.accumulate_weights(w, c, o, 0.9) is w
    tol = 1.01 * U * ((views + 7 + views // 32) * add + (3 + views // 32) * before)
    assert bool(((w.double() - want).abs() <= tol).all())


def test_weights_at_odd_addresses_and_strides():
    import gsplat_optim as G
    buf = torch.full((1100,), 5.0, device="cuda")
    w = buf[3:1003]
    table = torch.rand(1000, 3, device="cuda")
    col = torch.rand(2000, device="cuda")[1::2]
    G.accumulate_weights(w, [table[:, 1], col, table[:, 2].contiguous()[:]], None, 0.5)
    want = 2.5 + table[:, 1].double() + col.double() + table[:, 2].double()
    assert bool(((w.double() - want).abs() <= 8 * U * want).all())
    assert bool((buf[:3] == 5).all()) and bool((buf[1003:] == 5).all())
    single = torch.zeros(1000, 1, device="cuda")
    G.accumulate_weights(single, table[:, 0])
    assert torch.equal(single.view(-1), table[:, 0])
    # saturated opacities: exp overflows to infinity, the weight is zero, not NaN
    z = torch.zeros(3, device="cuda")
    G.accumulate_weights(z, [torch.ones(3, device="cuda")], torch.tensor([-200.0, 0.0, 200.0], device="cuda"))
    assert z.tolist() == [0.0, 0.5, 1.0]


def test_weight_refusals():
    import gsplat_optim as G
    w = torch.zeros(10, device="cuda")
    for bad in (torch.zeros(9, device="cuda"), torch.zeros(10), torch.zeros(10, device="cuda", dtype=torch.float64),
                torch.zeros(2, 5, device="cuda")):
        with pytest.raises(RuntimeError, match="one entry per"):
            G.accumulate_weights(w, [bad])
    with pytest.raises(RuntimeError, match="one entry per"):
        G.accumulate_weights(w, [], torch.zeros(10))
    for aliases in ([w], [torch.ones(10, device="cuda"), w], [w.view(10, 1)]):
        with pytest.raises(RuntimeError, match="share memory"):
            G.accumulate_weights(w, aliases)
    with pytest.raises(RuntimeError, match="contiguous"):
        G.accumulate_weights(torch.zeros(20, device="cuda")[::2], [torch.ones(10, device="cuda")])
    with pytest.raises(RuntimeError, match="decay"):
        G.accumulate_weights(w, [], None, math.nan)
    assert float(w.abs().max()) == 0.0
    G.accumulate_weights(torch.zeros(0, device="cuda"), [torch.zeros(0, device="cuda")])


# ------------------------------------------------------------------ selection
def _reference(w, budget, recent):
    """By definition: order by (NaN last, larger weight, lower index), on the CPU."""
    w = w.cpu().numpy().astype(np.float64)
    N = len(w)
    recent, keep = min(recent, N), min(budget, N)
    old = N - recent
    v = w[:old] + 0.0
    order = np.lexsort((np.arange(old), np.where(np.isnan(v), 0.0, -v), np.isnan(v)))
    return np.sort(np.concatenate([order[:keep - recent], np.arange(old, N)])).astype(np.int32)


def _weights(kind, N, gen):
    r = lambda: torch.rand(N, device="cuda", generator=gen)
    if kind == "random":
        return torch.randn(N, device="cuda", generator=gen)
    if kind == "equal":
        return torch.full((N,), 0.25, device="cuda")
    if kind == "zeros":
        return r() * (r() < 0.05)
    if kind == "few_values":
        return (r() * 5).floor() - 2
    if kind == "near":      # equal in their upper bits: the last histogram decides
        return torch.tensor(1.0, device="cuda") + (r() * 500).floor() * 2.0 ** -23
    w = torch.randn(N, device="cuda", generator=gen)
    for val, share in ((math.nan, 0.2), (math.inf, 0.1), (-math.inf, 0.1), (0.0, 0.1), (-0.0, 0.1), (1e-44, 0.05), (-1e-44, 0.05)):
        w[r() < share] = val
    return w


@pytest.mark.parametrize("kind", ["random", "equal", "zeros", "few_values", "near", "special"])
@pytest.mark.parametrize("N", [1, 2, 63, 256, 1000, 4095, 4096, 4097, 8191, 8192, 8193, 70001])
def test_selection(kind, N):
    import gsplat_optim as G
    gen = torch.Generator(device="cuda").manual_seed(N)
    w = _weights(kind, N, gen)
    for budget in sorted({0, 1, N // 3, N // 2, N - 1, N, N + 5}):
        for recent in sorted({0, min(1, budget), budget // 2, budget}):
            rows, kept = G.evict_rows(w, budget, recent)
            assert rows.dtype == torch.int32 and rows.is_cuda and kept == []
            assert np.array_equal(rows.cpu().numpy(), _reference(w, budget, recent)), (budget, recent)


def test_selection_of_a_large_model():
    import gsplat_optim as G
    gen = torch.Generator(device="cuda").manual_seed(3)
    N = 3_000_017
    for kind in ("random", "zeros"):
        w = _weights(kind, N, gen)
        rows, _ = G.evict_rows(w, 2_000_000, 100_000)
        assert np.array_equal(rows.cpu().numpy(), _reference(w, 2_000_000, 100_000))


@pytest.mark.parametrize("kind", ["random", "equal", "zeros", "few_values", "near", "special"])
@pytest.mark.parametrize("N,offset", [(2_200_003, 1), (2_097_153, 0), (9_000_001, 0)])
def test_selection_in_several_steps_and_tiles(kind, N, offset):
    """More rows than the workgroups take at once: several loads a thread, several tiles a workgroup."""
    import gsplat_optim as G
    gen = torch.Generator(device="cuda").manual_seed(N)
    w = torch.empty(N + offset, device="cuda")[offset:]
    w.copy_(_weights(kind, N, gen))
    for budget, recent in ((N - 1, 0), (N // 3, N // 5 + 1), (17, 3)):
        rows, _ = G.evict_rows(w, budget, recent)
        # the same order on the GPU: NaN last, then larger weights, then lower rows (two stable sorts)
        old = N - recent
        v = w[:old] + 0.0
        order = torch.sort(torch.where(v.isnan(), -math.inf, v), descending=True, stable=True).indices
        order = order[torch.sort(v[order].isnan().to(torch.uint8), stable=True).indices]
        want = torch.cat((order[:budget - recent].sort().values, torch.arange(old, N, device="cuda"))).to(torch.int32)
        assert torch.equal(rows, want), (budget, recent)


def test_selection_of_the_largest_list():
    """2^31 - 1 rows: byte offsets beyond 32 bits in weights and rows."""
    import gsplat_optim as G
    N = (1 << 31) - 1
    w = torch.zeros(N, device="cuda")
    at = [5, 1 << 30, (1 << 30) + 7, N - 260, N - 1]
    w[at] = torch.tensor([3.0, 2.0, -1.0, -2.0, 1.0], device="cuda")
    assert G.evict_rows(w, 3)[0].tolist() == [5, 1 << 30, N - 1]
    assert G.evict_rows(w, 4, 2)[0].tolist() == [5, 1 << 30, N - 2, N - 1]
    rows = G.evict_rows(w, N - 2)[0]
    a, b = at[2], at[3]
    assert rows.shape == (N - 2,)
    assert rows[[0, a - 1, a, b - 2, b - 1, N - 3]].tolist() == [0, a - 1, a + 1, b - 1, b + 1, N - 1]
    assert int((rows[1:] - rows[:-1]).max()) == 2 and int((rows[1:] - rows[:-1]).min()) == 1
    with pytest.raises(RuntimeError, match="2\\^31"):
        G.evict_rows(torch.zeros(1, device="cuda").expand(1 << 31).contiguous(), 5)


def test_selection_takes_a_column_and_any_address():
    import gsplat_optim as G
    base = torch.randn(5003, device="cuda")
    for off in (1, 2, 3):
        w = base[off:]
        assert np.array_equal(G.evict_rows(w, 100)[0].cpu().numpy(), _reference(w, 100, 0))
    w = torch.randn(300, 1, device="cuda")
    assert np.array_equal(G.evict_rows(w, 100)[0].cpu().numpy(), _reference(w.view(-1), 100, 0))
    w = torch.randn(300, 2, device="cuda")[:, 1]
    assert np.array_equal(G.evict_rows(w, 100)[0].cpu().numpy(), _reference(w, 100, 0))


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("N,budget", [(1, 1), (7, 3), (1000, 1000), (1000, 0), (5001, 4000), (70001, 69999)])
def test_rows_of_any_tensor(N, budget):
    import gsplat_optim as G
    gen = torch.Generator(device="cuda").manual_seed(N)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    wide = r(N, 9)
    tensors = [r(N, 3), r(N, 15, 3), r(N), r(N, 1), r(N, 4), r(N, 3).to(torch.bfloat16), r(N, 7).half(), r(N, 2).double(),
               (r(N) > 0), (r(N, 5) > 0), torch.arange(N, device="cuda"), torch.arange(N, device="cuda", dtype=torch.int32),
               (r(N, 3) * 50).to(torch.int8), r(N, 0), r(N, 3, 0), wide[:, 2:7], wide[:, 4], wide[:, 1:].to(torch.bfloat16)[:, 1:],
               r(3, N).t(), r(1, 6).expand(N, 6), r(N + 1, 3)[1:], r(N + 1)[1:].to(torch.bfloat16), r(N, 301),
               (r(N * 3 + 1) * 50).to(torch.int8)[1:].view(N, 3), r(N, 16).to(torch.bfloat16)]
    w = torch.rand(N, device="cuda", generator=gen)
    rows, kept = G.evict_rows(w, budget, min(2, budget), tensors)
    for t, k in zip(tensors, kept):
        assert k.is_contiguous() and k.dtype == t.dtype and torch.equal(k, t[rows.long()]), (t.shape, t.dtype, t.stride())


def test_many_tensors():
    import gsplat_optim as G
    N = 333
    tensors = [torch.randn(N, 1 + k % 17, device="cuda") for k in range(250)]
    rows, kept = G.evict_rows(torch.rand(N, device="cuda"), 111, 0, tensors)
    assert all(torch.equal(k, t[rows.long()]) for t, k in zip(tensors, kept))


def test_tensors_beyond_32_bit_offsets():
    """4-byte units beyond 2^32 and bytes beyond 2^34 in source and copy; every value names its place."""
    import gsplat_optim as G
    N, M = 36_000_000, 128
    t = torch.empty(N, M, dtype=torch.int32, device="cuda")
    t[:, 0] = torch.arange(N, device="cuda", dtype=torch.int32)
    t[:, M - 1] = torch.arange(N, device="cuda", dtype=torch.int32) + 1
    w = torch.ones(N, device="cuda")
    w[::50] = 0.5
    budget = N - N // 50
    rows, (k,) = G.evict_rows(w, budget, 0, [t])
    assert k.numel() > 1 << 32
    assert torch.equal(k[:, 0], rows) and torch.equal(k[:, M - 1], rows + 1)
    assert torch.equal(rows, torch.nonzero(w == 1.0).view(-1).to(torch.int32))


def test_eviction_refusals():
    import gsplat_optim as G
    w = torch.rand(10, device="cuda")
    for budget, recent in ((-1, 0), (5, 6), (5, -1)):
        with pytest.raises(RuntimeError, match="budget"):
            G.evict_rows(w, budget, recent)
    with pytest.raises(RuntimeError, match="float32"):
        G.evict_rows(w.double(), 5)
    with pytest.raises(RuntimeError, match="one entry per row"):
        G.evict_rows(torch.rand(10, 2, device="cuda"), 5)
    for bad in (torch.rand(9, device="cuda"), torch.rand(10), torch.tensor(1.0, device="cuda")):
        with pytest.raises(RuntimeError, match="one row per weight"):
            G.evict_rows(w, 5, 0, [bad])
    empty, kept = G.evict_rows(torch.zeros(0, device="cuda"), 5, 2, [torch.zeros(0, 3, device="cuda")])
    assert empty.shape == (0,) and kept[0].shape == (0, 3)


def test_on_a_side_stream_and_in_a_graph():
    """Replays on new weights with eager calls between them; two captured graphs that do not share scratch memory."""
    import gsplat_optim as G
    N, budget, recent = 20011, 15000, 500
    gen = torch.Generator(device="cuda").manual_seed(8)
    w, t, c = torch.rand(N, device="cuda", generator=gen), torch.randn(N, 3, device="cuda"), torch.rand(N, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rows, kept = G.evict_rows(w, budget, recent, [t])
    torch.cuda.current_stream().wait_stream(side)
    assert np.array_equal(rows.cpu().numpy(), _reference(w, budget, recent))
    graphs = []
    for b in (budget, budget // 2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            G.accumulate_weights(w, [c], None, 0.5)
            out = G.evict_rows(w, b, recent, [t])
        graphs.append((g, b, out))
    for k in range(3):
        for g, b, (rows, kept) in graphs:
            c.copy_(torch.rand(N, device="cuda", generator=gen) * (torch.rand(N, device="cuda", generator=gen) < 0.5))
            w.copy_(torch.rand(N, device="cuda", generator=gen))
            eager_w = w.clone()
            g.replay()
            G.accumulate_weights(eager_w, [c], None, 0.5)
            eager_rows, eager_kept = G.evict_rows(eager_w, b, recent, [t])
            torch.cuda.synchronize()
            assert torch.equal(w, eager_w) and torch.equal(rows, eager_rows) and torch.equal(kept[0], eager_kept[0])
            assert np.array_equal(rows.cpu().numpy(), _reference(w, b, recent))


# ------------------------------------------------------------------ the optimizer, and a run of all of them
def _optimizer(N, steps=1):
    from gsplat_optim import FusedGaussianAdam
    gen = torch.Generator().manual_seed(5)
    shapes = dict(xyz=(N, 3), f_dc=(N, 1, 3), f_rest=(N, 15, 3), opacity=(N, 1), scaling=(N, 3), rotation=(N, 4), reps=(N, 4))
    opt = FusedGaussianAdam([{"params": [torch.nn.Parameter(torch.randn(*s, generator=gen).cuda())], "lr": 1e-3, "name": n}
                             for n, s in shapes.items()], lr=0.0, eps=1e-15)
    for _ in range(steps):
        for g in opt.param_groups:
            g["params"][0].grad = torch.randn(*g["params"][0].shape, generator=gen).cuda()
        opt.step()
    return opt


@pytest.mark.parametrize("steps", [0, 2])
def test_evict_optimizer(steps):
    import gsplat_optim as G
    N, budget = 3001, 2000
    a, b = _optimizer(N, steps), _optimizer(N, steps)
    w = torch.rand(N, device="cuda")
    stats = dict(weights=w, max_radii2D=torch.rand(N, device="cuda"), radii=torch.arange(N, device="cuda", dtype=torch.int32))
    got, rows, new = G.evict_optimizer(a, w, budget, 100, stats)
    assert np.array_equal(rows.cpu().numpy(), _reference(w, budget, 100))
    mask = torch.zeros(N, dtype=torch.bool, device="cuda")
    mask[rows.long()] = True
    G.prune_optimizer(b, mask)
    for ga, gb in zip(a.param_groups, b.param_groups):
        pa, pb = ga["params"][0], gb["params"][0]
        assert got[ga["name"]] is pa and isinstance(pa, torch.nn.Parameter) and pa.requires_grad and pa.grad is None
        assert torch.equal(pa, pb)
        if steps:
            for k in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(a.state[pa][k], b.state[pb][k])
            assert float(a.state[pa]["step"]) == steps
    assert len(a.state) == (len(a.param_groups) if steps else 0)
    assert all(torch.equal(new[k], stats[k][rows.long()]) for k in stats)
    for g in a.param_groups:
        g["params"][0].grad = torch.randn_like(g["params"][0])
    a.step()
    # one tensor that does not match: nothing moves
    a.param_groups[3]["params"][0] = torch.nn.Parameter(torch.zeros(7, 1, device="cuda"))
    before = [g["params"][0] for g in a.param_groups]
    with pytest.raises(RuntimeError, match="opacity"):
        G.evict_optimizer(a, new["weights"], 10)
    assert all(x is g["params"][0] for x, g in zip(before, a.param_groups))


def test_a_training_run_within_its_bounds():
    """Views, accumulated weights, clipped steps and evictions as a training program strings them together, next to the
    same run with the plain operations in between: the chosen rows are equal, the parameters to the roundings of a
    few steps (the gradients' atomics alone differ by more from run to run, so the plain run gets the same gradients)."""
    import gsplat_optim as G
    import synth
    from diff_gaussian_rasterization import GaussianRasterizationSettings, GaussianRasterizer, ParamGradSink
    dev, W, H, P = "cuda:0", 96, 64, 1200
    sc = synth.tiny_scene(P=P, width=W, height=H, seed=21, scale=0.08)
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32, device=dev)
    op = np.clip(sc["opacities"].reshape(-1, 1), 1e-3, 1 - 1e-3)
    init = dict(xyz=t(sc["means3D"]), f_dc=t(sc["shs"][:, :1]), f_rest=t(sc["shs"][:, 1:]), opacity=t(np.log(op / (1 - op))),
                scaling=t(np.log(sc["scales"])), rotation=t(sc["rotations"]), reps=t(sc["reps"]))
    names = list(init)
    cams = []
    for v in range(2):
        cam = synth.make_camera(W, H, 0.9, (0.3 * v, -0.05, -2.5), (0.0, 0.0, 1.0))
        cams.append(GaussianRasterizationSettings(
            image_height=H, image_width=W, tanfovx=cam["tanfovx"], tanfovy=cam["tanfovy"], bg=torch.zeros(3, device=dev),
            scale_modifier=1.0, viewmatrix=t(cam["viewmatrix"]), projmatrix=t(cam["projmatrix"]), sh_degree=3,
            campos=t(cam["campos"]), prefiltered=False, debug=False, antialiasing=True))
    params = {k: torch.nn.Parameter(v.clone().contiguous()) for k, v in init.items()}
    opt = G.FusedGaussianAdam([{"params": [params[k]], "lr": 1e-3, "name": k} for k in names], lr=0.0, eps=1e-15)
    plain = {k: [params[k].detach().double(), None, None] for k in names}
    steps = 0
    weights = torch.zeros(P, device=dev)
    plain_w = torch.zeros(P, device=dev, dtype=torch.float64)
    for budget in (1000, 900):
        sink = ParamGradSink(*[params[k] for k in names], defer=True)
        for it in range(3):
            sink.begin_step()
            sums = []
            for rs in cams:
                m2 = torch.zeros_like(params["xyz"], requires_grad=True)
                img, radii, invd, gsum, gcnt, reps = GaussianRasterizer(rs).forward_params(
                    params["xyz"], m2, *[params[k] for k in names[1:]], grad_sink=sink)
                (img.square().mean() * 50 + reps.abs().mean()).backward()
                sums.append(gsum.detach())
            sink.flush()
            G.accumulate_weights(weights, sums, params["opacity"], 0.9)
            plain_w = plain_w * 0.9 + torch.sigmoid(plain["opacity"][0].view(-1)) * sum(s.double().view(-1) for s in sums)
            norm = opt.clipped_step(0.1)
            wide = {k: params[k].grad.double() for k in names}
            ref = math.sqrt(sum(float(g.square().sum()) for g in wide.values()))
            assert ref > 0 and abs(float(norm) - ref) <= 1e-6 * ref
            steps += 1
            for k in names:
                p, m, v = plain[k]
                g = wide[k] * min(1.0, 0.1 / (ref + 1e-6))
                m = 0.1 * g if m is None else 0.9 * m + 0.1 * g
                v = 0.001 * g * g if v is None else 0.999 * v + 0.001 * g * g
                plain[k] = [p - 1e-3 / (1 - 0.9 ** steps) * m / ((v / (1 - 0.999 ** steps)).sqrt() + 1e-15), m, v]
        n = weights.shape[0]
        params, rows, new = G.evict_optimizer(opt, weights, budget, 50, dict(weights=weights))
        gap = (torch.sort(plain_w[:n - 50], descending=True).values[budget - 51:budget - 49])
        if float(gap[0] - gap[1]) > 1e-4 * float(gap[0]):   # the border is wider than the roundings of either side
            assert np.array_equal(rows.cpu().numpy(), _reference(plain_w, budget, 50))
        weights = new["weights"]
        plain_w = plain_w[rows.long()]
        plain = {k: [x[rows.long()] for x in plain[k]] for k in names}
        for k in names:
            assert params[k].shape[0] == budget
            # gradients of rows that no pixel reached are zero on both sides; a first step is lr * g / |g| however
            # small g is, so a gradient near the float32 underflow decides its own size: leave those elements out
            sure = plain[k][2] > 1e-30
            # at most 6 steps of 1e-3, each off by 40 roundings of the update (cancellation in the first moment aside,
            # which the bound of the update, lr / sqrt(1 - beta2), covers: 0.032 per step) and one of the parameter
            bound = 6 * (0.032 * 40 * U) + 6 * U * plain[k][0].abs()
            assert bool(((params[k].double() - plain[k][0]).abs() <= bound)[sure].all()), k


@pytest.mark.parametrize("shape,dtype", [((40, 40001), torch.float32), ((40, 40000), torch.float32), ((33, 70001), torch.bfloat16),
                                         ((33, 33333), torch.int8), ((17, 20002), torch.float32)])
def test_wide_rows(shape, dtype):
    import gsplat_optim as G
    t = (torch.randn(shape, device="cuda") * 40).to(dtype)
    rows, (k,) = G.evict_rows(torch.rand(shape[0], device="cuda"), shape[0] - 9, 0, [t])
    assert torch.equal(k, t[rows.long()])


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 8])
@pytest.mark.parametrize("row_bytes,pitch", [(12, 12), (16, 16), (16, 20), (5, 5), (6, 8), (180, 180), (4, 4), (1, 1), (1, 3), (64, 0)])
def test_c_abi_copies_to_any_address(offset, row_bytes, pitch):
    """Through the C ABI the copy may start anywhere; what lies around it stays."""
    import ctypes as C
    from _gsplat_lib import check, lib
    N, K = 700, 411
    gen = torch.Generator(device="cuda").manual_seed(offset)
    src = torch.randint(0, 250, (N * max(pitch, 1) + row_bytes + 64,), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    dst = torch.full((K * row_bytes + 64,), 255, dtype=torch.uint8, device="cuda")
    rows = torch.randperm(N, device="cuda", generator=gen)[:K].sort().values.to(torch.int32)
    entry = (C.c_int64 * 4)(src.data_ptr() + offset, dst.data_ptr() + offset, row_bytes, pitch)
    check(lib().gso_gather_rows_multi(1, C.addressof(entry), rows.data_ptr(), K, torch.cuda.current_stream().cuda_stream), "gather")
    at = offset + rows.long()[:, None] * pitch + torch.arange(row_bytes, device="cuda")[None]
    torch.cuda.synchronize()
    assert torch.equal(dst[offset:offset + K * row_bytes].view(K, row_bytes), src[at])
    assert bool((dst[:offset] == 255).all()) and bool((dst[offset + K * row_bytes:] == 255).all())


def test_two_evictions_at_once_on_two_streams():
    import gsplat_optim as G
    ws = [torch.rand(200_003, device="cuda") for _ in range(2)]
    ts = [torch.randn(200_003, 45, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in ws]
    torch.cuda.synchronize()
    out = []
    for w, t, st in zip(ws, ts, streams):
        with torch.cuda.stream(st):
            out.append(G.evict_rows(w, 150_000, 1000, [t]))
    torch.cuda.synchronize()
    for w, t, (rows, kept) in zip(ws, ts, out):
        assert np.array_equal(rows.cpu().numpy(), _reference(w, 150_000, 1000)) and torch.equal(kept[0], t[rows.long()])


def test_lazy_conjugates_and_a_single_tensor():
    import gsplat_optim as G
    z = torch.randn(100, 3, device="cuda", dtype=torch.complex64)
    w = torch.rand(100, device="cuda")
    rows, kept = G.evict_rows(w, 60, 0, [z.conj(), z.conj().imag, z.conj().real])
    at = rows.long()
    assert torch.equal(kept[0], z[at].conj()) and torch.equal(kept[1], -z.imag[at]) and torch.equal(kept[2], z.real[at])
    rows, kept = G.evict_rows(w, 60, 0, z)
    assert len(kept) == 1 and torch.equal(kept[0], z[rows.long()])
    lazy = torch.complex(w, -w).conj().imag
    assert lazy.is_neg() is True
    assert np.array_equal(G.evict_rows(lazy, 60)[0].cpu().numpy(), _reference(w, 60, 0))
    acc = torch.zeros(100, device="cuda")
    G.accumulate_weights(acc, [lazy])
    assert torch.equal(acc, w)


@pytest.mark.parametrize("row_bytes,pitch", [(1, 1), (2, 2), (4, 4), (8, 8), (3, 3), (6, 6), (12, 12), (16, 16), (180, 180), (4, 12), (1, 0)])
@pytest.mark.parametrize("order", ["repeats", "descending", "random", "pairs"])
def test_c_abi_copies_rows_in_any_order(row_bytes, pitch, order):
    """Repeated and unordered rows: a vector of the copy whose first and last row are as far apart as in a run of rows
    need not be one."""
    import ctypes as C
    from _gsplat_lib import check, lib
    N, K = 500, 1003
    gen = torch.Generator(device="cuda").manual_seed(row_bytes)
    src = torch.randint(0, 250, (N * max(pitch, row_bytes),), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    dst = torch.full((K * row_bytes,), 255, dtype=torch.uint8, device="cuda")
    if order == "repeats":      # 5 5 7 8, 9 9 11 12, ...: ascending, the span of a run
        rows = (torch.arange(K, device="cuda") + 5 - (torch.arange(K, device="cuda") % 4 == 1).long()) % (N - 8)
    elif order == "descending":
        rows = torch.arange(K, device="cuda").flip(0) % N
    elif order == "random":
        rows = torch.randint(0, N, (K,), device="cuda", generator=gen)
    else:                       # 0 2 1 3, 4 6 5 7, ...
        k = torch.arange(K, device="cuda")
        rows = (k + (k % 4 == 1).long() - (k % 4 == 2).long()) % (N - 8)
    rows = rows.to(torch.int32)
    assert int(rows.min()) >= 0 and int(rows.max()) < N
    entry = (C.c_int64 * 4)(src.data_ptr(), dst.data_ptr(), row_bytes, pitch)
    check(lib().gso_gather_rows_multi(1, C.addressof(entry), rows.data_ptr(), K, torch.cuda.current_stream().cuda_stream), "gather")
    at = rows.long()[:, None] * pitch + torch.arange(row_bytes, device="cuda")[None]
    torch.cuda.synchronize()
    assert torch.equal(dst.view(K, row_bytes), src[at])


@pytest.mark.parametrize("over", [0, 7])
@pytest.mark.parametrize("steps", [0, 2])
def test_a_model_within_its_budget_stays_as_it_is(steps, over):
    import gsplat_optim as G
    N = 3001
    opt = _optimizer(N, steps)
    old = {g["name"]: g["params"][0] for g in opt.param_groups}
    for p in old.values():
        p.grad = torch.randn_like(p)
    grads = {k: p.grad for k, p in old.items()}
    state = {k: dict(opt.state[p]) for k, p in old.items()} if steps else {}
    values = {k: p.detach().clone() for k, p in old.items()}
    w = torch.rand(N, device="cuda")
    stats = dict(weights=w, radii=torch.arange(N, device="cuda", dtype=torch.int32))
    got, rows, new = G.evict_optimizer(opt, w, N + over, 100, stats)
    assert rows.dtype == torch.int32 and torch.equal(rows, torch.arange(N, device="cuda", dtype=torch.int32))
    assert list(got) == list(old) and list(new) == list(stats) and all(new[k] is stats[k] for k in stats)
    for g in opt.param_groups:
        k = g["name"]
        assert got[k] is old[k] and g["params"][0] is old[k] and old[k].grad is grads[k] and torch.equal(old[k], values[k])
        if steps:
            assert all(opt.state[old[k]][n] is t for n, t in state[k].items())
    assert len(opt.state) == (len(old) if steps else 0)
    opt.step()
    # what an eviction refuses is refused here too
    for bad in (torch.rand(N - 1, device="cuda"), torch.rand(N), torch.tensor(1.0, device="cuda")):
        with pytest.raises(RuntimeError, match="one row per weight"):
            G.evict_optimizer(opt, w, N + over, 0, dict(bad=bad))
    with pytest.raises(RuntimeError, match="recent"):
        G.evict_optimizer(opt, w, N, N + 1)
    with pytest.raises(RuntimeError, match="float32"):
        G.evict_optimizer(opt, w.double(), N)
