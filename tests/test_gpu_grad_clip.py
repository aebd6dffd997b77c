"""The global gradient norm, clipping and the Adam step under a ceiling, against the formulas in 64 bits.

Tolerances, from the roundings: u = 2^-24 is half a step of float32.  The sums are held in 64 bits, so the norm is off
by its one rounding, u, and n * 2^-53 for n terms.  The coefficient is rounded once (u), the product with a gradient in
float32 once (u), and to the gradient's type once more (2^-8 for bfloat16, 2^-11 for float16; below the normal range
half a step of the type's subnormals)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUBNORMAL = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
SHAPES = dict(xyz=(3,), f_dc=(1, 3), f_rest=(15, 3), opacity=(1,), scaling=(3,), rotation=(4,), reps=(4,))


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def _norm64(grads, p):
    """The definition, in 64 bits on the CPU."""
    flat = np.concatenate([g.detach().double().cpu().numpy().ravel() for g in grads] + [np.zeros(0)])
    if p == 2.0:
        return math.sqrt(float(np.sum(flat * flat)))
    if p == 1.0:
        return float(np.sum(np.abs(flat)))
    return float(np.max(np.abs(flat))) if flat.size else 0.0


def _make(sizes, dtypes, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * scale).to(dtypes[k % len(dtypes)]).cuda() for k, s in enumerate(sizes)]


LISTS = [[1], [0, 5, 0], [4095, 4096, 4097], [63, 64, 65, 255, 256, 257], [100003], [(1000, 3), (1000, 15, 3), (1000, 1), ()],
         [(k * 37) % 611 for k in range(300)], [1 << 20, 1, 1048577]]
TYPES = [[torch.float32], [torch.bfloat16], [torch.float16], [torch.float32, torch.bfloat16, torch.float16]]


@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtypes", TYPES, ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("sizes", LISTS, ids=[str(i) for i in range(len(LISTS))])
def test_norm_and_clip(sizes, dtypes, norm_type):
    import gsplat_optim as G
    grads = _make(sizes, dtypes, seed=len(sizes))
    params = _params(grads)
    n = sum(g.numel() for g in grads)
    ref = _norm64(grads, norm_type)
    before = [g.clone() for g in grads]
    got = G.grad_norm(params, norm_type)
    assert got.shape == () and got.dtype == torch.float32 and got.is_cuda
    tol = U + 4 * n * 2.0 ** -53
    assert abs(float(got) - ref) <= tol * ref
    # under the ceiling: nothing moves
    kept = G.clip_grad_norm_(params, 2.0 * ref + 1.0, norm_type)
    assert torch.equal(kept, got) and all(torch.equal(a, b) for a, b in zip(grads, before))
    # over it
    ceiling = 0.3 * ref
    kept = G.clip_grad_norm_(params, ceiling, norm_type)
    assert torch.equal(kept, got)
    c = min(1.0, ceiling / (ref + 1e-6))
    for g, b in zip(grads, before):
        want = b.double() * c
        bound = want.abs() * (HALF_STEP[g.dtype] + 3 * U) + SUBNORMAL[g.dtype]
        assert bool(((g.double() - want).abs() <= bound).all())


def test_same_bits_as_torch_semantics_for_a_single_tensor_and_generators():
    import gsplat_optim as G
    g = _make([1000], [torch.float32])[0]
    p = _params([g])[0]
    n = G.grad_norm(p)
    assert torch.equal(n, G.grad_norm(x for x in [p, torch.nn.Parameter(torch.empty(3, device="cuda"))]))
    z = G.clip_grad_norm_([torch.nn.Parameter(torch.empty(3, device="cuda"))], 1.0)
    assert z.shape == () and float(z) == 0.0
    assert float(G.grad_norm([])) == 0.0
    q = torch.nn.Parameter(p.detach().clone())
    q.grad = g.clone()
    a, b = G.clip_grad_norm_(p, 0.5), torch.nn.utils.clip_grad_norm_(q, 0.5)
    assert abs(float(a) - float(b)) <= 1e-5 * float(b)
    assert torch.allclose(p.grad, q.grad, rtol=1e-5, atol=0)


@pytest.mark.parametrize("scale", [3e38, 1e-30, 1e-44, 0.0])
@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
def test_extreme_sizes_do_not_overflow_or_vanish(scale, norm_type):
    import gsplat_optim as G
    g = torch.full((5001,), scale, device="cuda")
    if scale == 3e38:
        g[1:] = 1e36
    ref = _norm64([g], norm_type)
    got = float(G.grad_norm(_params([g]), norm_type))
    if ref > float(np.finfo(np.float32).max):
        assert got == math.inf
        ref64 = ref
    else:
        assert abs(got - ref) <= ref * (U + 1e-11) + SUBNORMAL[torch.float32]
        ref64 = ref
    before = g.clone()
    G.clip_grad_norm_(_params([g]), 0.25 * ref64 if ref64 < 1e38 else 1e37, norm_type)
    c = min(1.0, (0.25 * ref64 if ref64 < 1e38 else 1e37) / (ref64 + 1e-6))
    want = before.double() * c
    assert bool(((g.double() - want).abs() <= want.abs() * 3 * U + c * 0 + SUBNORMAL[torch.float32] + before.double().abs() * 2.0 ** -150).all())


@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite_gradients(norm_type, bad):
    import gsplat_optim as G
    grads = _make([3000, 5000, 17], [torch.float32, torch.bfloat16, torch.float16], seed=2)
    grads[1][4321] = bad
    before = [g.clone() for g in grads]
    with pytest.raises(RuntimeError, match="nothing was changed"):
        G.clip_grad_norm_(_params(grads), 1.0, norm_type, error_if_nonfinite=True)
    same = lambda: all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(grads, before))
    assert same()
    n = G.clip_grad_norm_(_params(grads), 1.0, norm_type)
    if math.isnan(bad):
        assert math.isnan(float(n)) and all(bool(g.isnan().all()) for g in grads)
    else:
        assert math.isinf(float(n)) and float(n) > 0
        assert bool(grads[1][4321].isnan()) and int(grads[1].isnan().sum()) == 1
        assert all(float(torch.nan_to_num(g.float(), nan=0.0).abs().max()) == 0.0 for g in grads)
    # an infinite ceiling never clips
    h = _make([100], [torch.float32])[0]
    was = h.clone()
    G.clip_grad_norm_(_params([h]), math.inf)
    assert torch.equal(h, was)
    G.clip_grad_norm_(_params([h]), 0.0)
    assert float(h.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_neighbours_of_a_gradient_are_neither_counted_nor_touched(dtype, offset):
    """Gradients that start at any element of a wider buffer, next to NaN."""
    import gsplat_optim as G
    for n in (1, 2, 7, 8, 9, 4096 - offset, 4096, 4097, 10001):
        buf = torch.full((n + offset + 9,), math.nan, dtype=dtype, device="cuda")
        g = buf[offset:offset + n]
        g.copy_(_make([n], [dtype], seed=n)[0])
        before = g.clone()
        ref = _norm64([g], 2.0)
        got = G.clip_grad_norm_(_params([g]), 0.5 * ref)
        assert abs(float(got) - ref) <= ref * (U + 1e-11)
        assert bool(buf[:offset].isnan().all()) and bool(buf[offset + n:].isnan().all())
        want = before.double() * (0.5 * ref / (ref + 1e-6))
        assert bool(((g.double() - want).abs() <= want.abs() * (HALF_STEP[dtype] + 3 * U) + SUBNORMAL[dtype]).all())


def test_gradients_of_other_layouts():
    import gsplat_optim as G
    wide = torch.randn(500, 8, device="cuda")
    keep = wide.clone()
    turned = torch.randn(70, 30, device="cuda")
    sparse = torch.randn(40, 40, device="cuda")
    grads = [wide[:, 2:5], turned.t(), sparse[::2, ::3]]
    refs = [g.clone() for g in grads]
    ref = _norm64(grads, 2.0)
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, device="cuda"))
        p.grad = g
        params.append(p)
    got = G.clip_grad_norm_(params, 0.1)
    assert abs(float(got) - ref) <= ref * (U + 1e-11)
    c = 0.1 / (ref + 1e-6)
    for p, r in zip(params, refs):
        assert bool(((p.grad.double() - r.double() * c).abs() <= r.double().abs() * c * 3 * U + SUBNORMAL[torch.float32]).all())
    assert torch.equal(wide[:, :2], keep[:, :2]) and torch.equal(wide[:, 5:], keep[:, 5:])


def test_refusals_on_the_gpu():
    import gsplat_optim as G
    g = torch.ones(10, device="cuda")
    a, b = _params([g, g])
    with pytest.raises(RuntimeError, match="share memory"):
        G.clip_grad_norm_([a, b], 1.0)
    c, d = _params([g[:6], g[5:]])
    with pytest.raises(RuntimeError, match="share memory"):
        G.clip_grad_norm_([d, c], 1.0)
    assert float(G.grad_norm([a, a])) == pytest.approx(math.sqrt(20.0))   # only read: counted twice, as torch does
    e = torch.nn.Parameter(torch.ones(10, device="cuda"))
    e.grad = torch.ones(1, device="cuda").expand(10)
    assert float(G.grad_norm(e)) == pytest.approx(math.sqrt(10.0))
    with pytest.raises(RuntimeError, match="expanded"):
        G.clip_grad_norm_(e, 1.0)
    f = _params([torch.ones(3, device="cuda", dtype=torch.float64)])
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        G.grad_norm(f)
    with pytest.raises(RuntimeError, match="norm_type"):
        G.grad_norm(a, 3.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(RuntimeError, match="max_norm"):
            G.clip_grad_norm_(a, bad)
    cpu = torch.nn.Parameter(torch.ones(3))
    cpu.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="one device|no CPU path"):
        G.clip_grad_norm_([a, cpu], 1.0)
    assert torch.equal(g, torch.ones(10, device="cuda"))


def test_more_than_2_31_elements():
    """Offsets beyond 32 bits: a bfloat16 tensor of 2^31 + 12345 elements, zero but for a few at its ends."""
    import gsplat_optim as G
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, (1 << 31) - 1, 1 << 31, (1 << 31) + 7, n - 1], device="cuda")
    g[at] = 3.0
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = g
    assert float(G.grad_norm(p)) == float(np.float32(math.sqrt(54.0)))
    assert float(G.grad_norm(p, 1.0)) == 18.0 and float(G.grad_norm(p, math.inf)) == 3.0
    G.clip_grad_norm_(p, 6.0, 1.0)     # c = 6 / 18.000001
    assert bool((g[at].float() == 1.0).all())
    assert int(torch.count_nonzero(g)) == 6


def test_on_a_side_stream_and_in_a_graph():
    """A captured clip replays on new gradients, with eager calls of the same leaves between the replays."""
    import gsplat_optim as G
    grads = _make([4097, 300, 100003], [torch.float32, torch.bfloat16, torch.float32], seed=9)
    params = _params(grads)
    source = [g.clone() for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for g in grads:
            g.mul_(2.0)
        n_side = G.clip_grad_norm_(params, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(n_side) - 2 * _norm64(source, 2.0)) <= 2 * _norm64(source, 2.0) * (U + 1e-9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = G.clip_grad_norm_(params, 1.0)
    with pytest.raises(RuntimeError, match="capture"):
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other):
            G.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    for k in range(4):
        for g, s in zip(grads, source):
            g.copy_(s * (k + 1))
        eager_in = [g.clone() for g in grads]
        eager_params = _params(eager_in)
        graph.replay()
        eager = G.clip_grad_norm_(eager_params, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)
        assert all(torch.equal(a, b) for a, b in zip(grads, eager_in))


# ------------------------------------------------------------------ Adam under the ceiling
def _optimizer(N, cls, seed=1, steps=3, extra=False):
    gen = torch.Generator().manual_seed(seed)
    groups = [{"params": [torch.nn.Parameter(torch.randn(N, *s, generator=gen).cuda())], "lr": 10.0 ** -(1 + k % 4), "name": n}
              for k, (n, s) in enumerate(SHAPES.items())]
    if extra:
        groups.append({"params": [torch.nn.Parameter(torch.randn(5, 3, 4, generator=gen).cuda())], "lr": 1e-3, "name": "exposure"})
    opt = cls(groups, lr=0.0, eps=1e-15)
    for _ in range(steps):
        _fill(opt, gen)
        opt.step()
    _fill(opt, gen)
    return opt


def _fill(opt, gen):
    for g in opt.param_groups:
        p = g["params"][0]
        p.grad = (torch.randn(p.shape, generator=gen) * 10.0 ** float(torch.randint(-4, 1, (1,), generator=gen))).cuda()


def _dump(opt):
    out = []
    for g in opt.param_groups:
        p = g["params"][0]
        st = opt.state[p]
        out += [p.detach().clone(), st["exp_avg"].clone(), st["exp_avg_sq"].clone(), torch.tensor(float(st["step"])).cuda()]
    return out


@pytest.mark.parametrize("N", [1, 2, 63, 1000, 1365, 4099])
@pytest.mark.parametrize("sparse", [None, 0.0, 0.3, 1.0])
@pytest.mark.parametrize("ceiling", [0.01, 1e9])
def test_clipped_step_is_clip_then_step_bit_for_bit(N, sparse, ceiling):
    import gsplat_optim as G
    a, b = (_optimizer(N, G.FusedGaussianAdam, extra=True) for _ in range(2))
    vis = None if sparse is None else torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N)) < sparse
    for norm_type in (2.0, 1.0, math.inf):
        raw = [g["params"][0].grad.clone() for g in a.param_groups]
        n1 = G.clip_grad_norm_([g["params"][0] for g in b.param_groups], ceiling, norm_type)
        b.step(vis, None if vis is None else N)
        n2 = a.clipped_step(ceiling, vis, None if vis is None else N, norm_type=norm_type)
        assert torch.equal(n1, n2)
        assert all(torch.equal(g["params"][0].grad, r) for g, r in zip(a.param_groups, raw))
        for x, y in zip(_dump(a), _dump(b)):
            assert torch.equal(x, y)
        for ga, gb in zip(a.param_groups, b.param_groups):
            gb["params"][0].grad = ga["params"][0].grad.clone()


def test_clipped_step_against_the_formula_in_64_bits():
    """Every rounding of the update counted (u = 2^-24): the gradient 2u, the first moment 3u of its step and u of
    itself plus what the gradient brings, the second 8u, the denominator 8u, the update 12u more, the parameter u."""
    import gsplat_optim as G
    for cls in (torch.optim.Adam, G.FusedGaussianAdam):
        opt = _optimizer(777, cls)
        old = [x.double().cpu().numpy() for x in _dump(opt)]
        grads = [g["params"][0].grad for g in opt.param_groups]
        ref = _norm64(grads, 2.0)
        c = 0.05 / (ref + 1e-6)
        n = G.clipped_adam_step(opt, 0.05)
        assert abs(float(n) - ref) <= ref * (U + 1e-11)
        new = [x.double().cpu().numpy() for x in _dump(opt)]
        for k, group in enumerate(opt.param_groups):
            p, m, v, t = old[4 * k:4 * k + 4]
            p1, m1, v1, t1 = new[4 * k:4 * k + 4]
            t = float(t) + 1
            assert float(t1) == t
            g = grads[k].double().cpu().numpy() * c
            rm = m + 0.1 * (g - m)
            em = 1.01 * U * (0.1 * (3 * np.abs(g - m) + 2 * np.abs(g)) + np.abs(rm))
            rv = 0.999 * v + 0.001 * g * g
            b1, b2 = 1 - 0.9 ** t, 1 - 0.999 ** t
            den = np.sqrt(rv / b2) + 1e-15
            step = group["lr"] / b1
            upd = step * rm / den
            assert np.all(np.abs(m1 - rm) <= em + 1e-45)
            assert np.all(np.abs(v1 - rv) <= 8.1 * U * rv + 1e-45)
            assert np.all(np.abs(p1 - (p - upd)) <= step * em / den * 1.01 + 20 * U * np.abs(upd) + 1.01 * U * np.abs(p - upd))


def test_first_step_creates_the_state_and_a_failure_leaves_none():
    import gsplat_optim as G
    p = torch.nn.Parameter(torch.ones(100, 3, device="cuda"))
    opt = G.FusedGaussianAdam([{"params": [p], "lr": 0.1, "name": "xyz"}], eps=1e-15)
    assert float(opt.clipped_step(1.0)) == 0.0 and len(opt.state) == 0      # no gradient at all: nothing happens
    p.grad = torch.full((100, 3), math.nan, device="cuda")
    with pytest.raises(RuntimeError, match="nothing was changed"):
        opt.clipped_step(1.0, error_if_nonfinite=True)
    assert len(opt.state) == 0 and torch.equal(p.detach(), torch.ones(100, 3, device="cuda"))
    p.grad = torch.full((100, 3), 0.5, device="cuda")
    opt.clipped_step(1.0, error_if_nonfinite=True)
    assert float(opt.state[p]["step"]) == 1.0
    assert torch.allclose(p.detach(), torch.full((100, 3), 0.9, device="cuda"), rtol=1e-6)   # 1 - lr * sign(g)


def test_clipped_step_refusals():
    import gsplat_optim as G
    p = torch.nn.Parameter(torch.ones(10, 3, device="cuda"))
    p.grad = torch.ones_like(p)
    for kw in (dict(weight_decay=0.1), dict(amsgrad=True), dict(maximize=True), dict(capturable=True)):
        with pytest.raises(RuntimeError, match="not supported"):
            G.clipped_adam_step(torch.optim.Adam([p], lr=1e-3, **kw), 1.0)
    with pytest.raises(RuntimeError, match="torch.optim.Adam"):
        G.clipped_adam_step(torch.optim.SGD([p], lr=1e-3), 1.0)
    opt = G.FusedGaussianAdam([p], lr=1e-3)
    with pytest.raises(RuntimeError, match="one entry per Gaussian"):
        opt.clipped_step(1.0, torch.ones(9, dtype=torch.bool, device="cuda"))
    with pytest.raises(RuntimeError, match="visibility must be on"):
        opt.clipped_step(1.0, torch.ones(10, dtype=torch.bool))
    for bad in (-1.0, math.nan):
        with pytest.raises(RuntimeError, match="max_norm"):
            opt.clipped_step(bad)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.clipped_step(1.0)
    assert len(opt.state) == 0 and torch.equal(p.detach(), torch.ones(10, 3, device="cuda"))


def test_the_norm_is_the_same_bits_in_every_run():
    import gsplat_optim as G
    grads = _make([3_000_001, 77, 500_000], [torch.float32, torch.bfloat16, torch.float16], seed=4)
    params = _params(grads)
    first = G.grad_norm(params)
    for _ in range(20):
        assert torch.equal(first, G.grad_norm(params))


def test_in_place_changes_are_seen_by_autograd():
    import gsplat_optim as G
    p = torch.nn.Parameter(torch.ones(100, 3, device="cuda"))
    opt = G.FusedGaussianAdam([p], lr=0.1)
    p.grad = torch.ones_like(p)
    g0, p0 = p.grad._version, p._version
    G.clip_grad_norm_(p, 0.1)
    assert p.grad._version > g0
    y = (p * p).sum()                 # keeps p for its backward
    opt.clipped_step(1.0)
    assert p._version > p0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    w, c = torch.zeros(5, device="cuda"), torch.ones(5, device="cuda")
    w0 = w._version
    G.accumulate_weights(w, c)
    assert w._version > w0
    with torch.inference_mode():
        G.accumulate_weights(torch.zeros(5, device="cuda"), c)


def test_step_counts_of_a_checkpoint_loaded_to_the_gpu():
    import gsplat_optim as G
    a, b = _optimizer(50, G.FusedGaussianAdam), _optimizer(50, G.FusedGaussianAdam)
    for st in a.state.values():
        st["step"] = st["step"].cuda()
    a.clipped_step(0.01)
    b.clipped_step(0.01)
    for x, y in zip(_dump(a), _dump(b)):
        assert torch.equal(x, y)
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="not supported"):
        G.clipped_adam_step(torch.optim.Adam([p], fused=True), 1.0)


@pytest.mark.parametrize("width", [1, 2, 3, 7, 45, 1000, 4097, 8191, 8192, 9001])
@pytest.mark.parametrize("sparse", [False, True])
def test_rows_of_any_width_and_parameters_at_any_address(width, sparse):
    """Against clip_grad_norm_ and FusedGaussianAdam.step, which share no kernel with it; NaN around the tensors shows
    an access beyond them."""
    import gsplat_optim as G
    N = max(3, 30000 // width)
    gen = torch.Generator(device="cuda").manual_seed(width)
    vis = torch.rand(N, device="cuda", generator=gen) < 0.4 if sparse else None

    def make(off):
        bufs = [torch.full((N * width + 16,), math.nan, device="cuda") for _ in range(4)]
        views = [b[off:off + N * width].view(N, width) for b in bufs]
        g2 = torch.Generator(device="cuda").manual_seed(7)
        for v in views:
            v.copy_(torch.randn(N, width, device="cuda", generator=g2))
        views[3].square_()
        p = torch.nn.Parameter(views[0])
        p.grad = views[1]
        opt = G.FusedGaussianAdam([{"params": [p], "lr": 0.1, "name": "xyz"}], eps=1e-15)
        opt.state[p] = {"step": torch.tensor(4.0), "exp_avg": views[2], "exp_avg_sq": views[3]}
        return bufs, p, opt
    ref = None
    for off in (0, 1, 2, 3, 4):
        bufs, p, opt = make(off)
        opt.clipped_step(0.5, vis, N if sparse else None)
        got = [p.detach().clone(), opt.state[p]["exp_avg"].clone(), opt.state[p]["exp_avg_sq"].clone()]
        for b in bufs:
            assert bool(b[:off].isnan().all()) and bool(b[off + N * width:].isnan().all())
            assert not bool(b[off:off + N * width].isnan().any())
        if off == 0:
            _, q, two = make(0)
            G.clip_grad_norm_(q, 0.5)
            two.step(vis, N if sparse else None)
            assert all(torch.equal(x, y) for x, y in zip(got, (q.detach(), two.state[q]["exp_avg"], two.state[q]["exp_avg_sq"])))
            ref = got
        else:    # another address: the norm's sum runs in another order, one rounding of the coefficient apart at most
            for x, y in zip(got, ref):
                assert torch.allclose(x, y, rtol=1e-5, atol=1e-6)


def test_two_calls_at_once_on_two_streams():
    import gsplat_optim as G
    sets = [_make([1 << 20, 333, 70001], [torch.float32, torch.bfloat16], seed=k) for k in range(2)]
    want = [[g.clone() for g in s] for s in sets]
    norms = [G.clip_grad_norm_(_params(w), 1.0) for w in want]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(G.clip_grad_norm_(_params(s), 1.0))
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(got[k], norms[k]) and all(torch.equal(a, b) for a, b in zip(sets[k], want[k]))


def test_tensors_of_a_step_must_not_share_memory():
    import gsplat_optim as G
    flat = torch.ones(300, device="cuda")
    p, q = torch.nn.Parameter(flat[:200].view(100, 2)), torch.nn.Parameter(flat[150:250].view(50, 2))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt = G.FusedGaussianAdam([p, q], lr=0.1)
    with pytest.raises(RuntimeError, match="shares memory"):
        opt.clipped_step(1.0)
    assert len(opt.state) == 0 and bool((flat == 1).all())
    a, b = torch.nn.Parameter(torch.ones(10, device="cuda")), torch.nn.Parameter(torch.ones(10, device="cuda"))
    a.grad = b.grad = torch.ones(10, device="cuda")          # read by both: allowed
    G.FusedGaussianAdam([a, b], lr=0.1).clipped_step(1e9)
    assert torch.equal(a, b) and float(a[0]) < 1
    with pytest.raises(RuntimeError, match="shares memory"):
        a.grad = b.data
        G.FusedGaussianAdam([a, b], lr=0.1).clipped_step(1e9)


def test_lazy_negatives_count_as_what_they_stand_for():
    import gsplat_optim as G
    z = torch.complex(torch.randn(50, device="cuda"), torch.rand(50, device="cuda") + 1)
    g = z.conj().imag
    assert g.is_neg()
    p = torch.nn.Parameter(torch.ones(50, device="cuda"))
    p.grad = g.clone()
    want = torch.nn.Parameter(torch.ones(50, device="cuda"))
    want.grad = p.grad
    lazy = torch.nn.Parameter(torch.ones(50, device="cuda"))
    lazy.grad = g
    a, b = G.FusedGaussianAdam([want], lr=0.1), G.FusedGaussianAdam([lazy], lr=0.1)
    assert torch.equal(a.clipped_step(1.0), b.clipped_step(1.0)) and torch.equal(want, lazy)
    n = float(G.clip_grad_norm_(lazy, 0.5))
    assert torch.allclose(g, want.grad * (0.5 / (n + 1e-6)), rtol=1e-6)


@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
def test_gradients_of_many_chunks(norm_type):
    """Several chunks a workgroup, and a tensor's border inside a round."""
    import gsplat_optim as G
    gen = torch.Generator(device="cuda").manual_seed(3)
    grads = [torch.randn(n, device="cuda", generator=gen).to(t) for n, t in
             ((20_000_003, torch.float32), (5, torch.float16), (9_000_001, torch.bfloat16), (1, torch.float32))]
    wide = [g.double() for g in grads]
    ref = float(torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g, norm_type) for g in wide]), norm_type))
    n = sum(g.numel() for g in grads)
    params = _params(grads)
    got = G.grad_norm(params, norm_type)
    assert abs(float(got) - ref) <= ref * (U + 8 * n * 2.0 ** -53)
    assert torch.equal(G.clip_grad_norm_(params, 0.4 * ref, norm_type), got)
    c = 0.4 * ref / (ref + 1e-6)
    for g, w in zip(grads, wide):
        want = w * c
        assert bool(((g.double() - want).abs() <= want.abs() * (HALF_STEP[g.dtype] + 3 * U) + SUBNORMAL[g.dtype]).all())


@pytest.mark.parametrize("N", [9000, 60_000, 125_000])
@pytest.mark.parametrize("sparse", [None, 0.2])
def test_clipped_step_of_many_chunks_is_clip_then_step(N, sparse):
    """Sums joined by the update itself (up to 2048 of them in a sparse step), and by a launch of their own."""
    import gsplat_optim as G
    a, b = (_optimizer(N, G.FusedGaussianAdam, steps=1) for _ in range(2))
    vis = None if sparse is None else torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N)) < sparse
    n1 = G.clip_grad_norm_([g["params"][0] for g in b.param_groups], 0.01)
    b.step(vis, None if vis is None else N)
    n2 = a.clipped_step(0.01, vis, None if vis is None else N)
    assert torch.equal(n1, n2)
    for x, y in zip(_dump(a), _dump(b)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("n", [10, 40_000, 1_000_000])
def test_a_step_that_no_group_takes_still_returns_the_norm(n):
    """A sparse step whose N no group has: the norm counts all gradients, and nothing moves."""
    import gsplat_optim as G
    p = torch.nn.Parameter(torch.ones(n, 3, device="cuda"))
    p.grad = torch.full((n, 3), 2.0, device="cuda")
    opt = G.FusedGaussianAdam([p], lr=0.1)
    vis = torch.ones(7, dtype=torch.bool, device="cuda")
    poison = torch.full((1 << 20,), math.nan, device="cuda")     # what a fresh allocation may hold
    del poison
    for _ in range(2):
        assert float(opt.clipped_step(1.0, vis, 7)) == pytest.approx(2.0 * math.sqrt(3 * n), rel=1e-6)
    assert bool((p == 1).all())
    empty = torch.nn.Parameter(torch.ones(0, 3, device="cuda"))
    empty.grad = torch.ones(0, 3, device="cuda")
    assert float(G.FusedGaussianAdam([empty], lr=0.1).clipped_step(1.0)) == 0.0


def test_a_gradient_of_another_shape_is_refused():
    """`parameter.data = other` leaves the old gradient behind; the update would read past its end."""
    import gsplat_optim as G
    p = torch.nn.Parameter(torch.ones(100, 3, device="cuda"))
    q = torch.nn.Parameter(torch.ones(50, device="cuda"))
    opt = G.FusedGaussianAdam([{"params": [p]}, {"params": [q]}], lr=0.1)
    for t in (p, q):
        t.grad = torch.full_like(t, 0.5)
    opt.clipped_step(1.0)
    state = {k: {n: x.clone() for n, x in opt.state[k].items()} for k in (p, q)}
    for shape in ((200, 3), (99, 3), (300,), (100, 3, 1)):
        p.data = torch.ones(shape, device="cuda")
        for k in ("exp_avg", "exp_avg_sq"):
            opt.state[p][k] = torch.ones(shape, device="cuda")
        before = q.detach().clone()
        for kw in ({}, dict(error_if_nonfinite=True)):
            with pytest.raises(RuntimeError, match="does not have its parameter's shape"):
                opt.clipped_step(1.0, **kw)
        assert torch.equal(p.detach(), torch.ones(shape, device="cuda")) and torch.equal(q.detach(), before)
        assert all(torch.equal(opt.state[q][n], x) for n, x in state[q].items()) and float(opt.state[p]["step"]) == 1.0
        assert all(bool((opt.state[p][n] == 1).all()) for n in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("make", [
    lambda on: on.to(torch.int32) * 256, lambda on: on.to(torch.int64) << 40, lambda on: on.float() * 0.5, lambda on: on.half() * -0.25,
    lambda on: on.to(torch.int16) * -512, lambda on: on.to(torch.int8) * -128, lambda on: on.to(torch.uint8) * 200, lambda on: on,
    lambda on: on.double()[:, None] * 1e-300, lambda on: torch.stack((on, ~on), 1)[:, 0]])
def test_a_row_is_visible_where_the_mask_is_not_zero(make):
    """In both steps, whatever the mask's type: radii and weights serve as masks as they are."""
    N = 3001
    on = torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.4
    import gsplat_optim as G
    a, b, c = (_optimizer(N, G.FusedGaussianAdam) for _ in range(3))
    before = _dump(a)
    mask = make(on)
    a.step(on, N)
    b.step(mask, N)
    c.clipped_step(1e30, mask, N)
    for x, y, z, was in zip(_dump(a), _dump(b), _dump(c), before):
        assert torch.equal(x, y) and torch.equal(x, z)
        if x.dim() > 0:
            assert torch.equal(x[~on], was[~on])


def test_strided_gradients_that_share_memory_are_refused():
    """They are scaled in packed copies; their own memory is what must not be shared."""
    import gsplat_optim as G
    wide = torch.randn(50, 8, device="cuda")
    keep = wide.clone()
    for grads in ((wide[:, 2:5], wide[:, 4:6]), (wide[:, 1], wide), (wide, wide[::2, ::2]), (wide[:, :3], wide[:, :3])):
        with pytest.raises(RuntimeError, match="share memory"):
            G.clip_grad_norm_(_params(grads), 1.0)
    with pytest.raises(RuntimeError, match="several elements in one place"):
        G.clip_grad_norm_(_params([wide.view(-1).as_strided((5, 3), (1, 1))]), 1.0)
    assert torch.equal(wide, keep)
    columns = [wide[:, :3], wide[:, 3:5], wide[:, 5], wide[:, 6:].t()]      # one buffer, every element once
    norm = G.clip_grad_norm_(_params(columns), 0.1)
    ref = _norm64([keep], 2.0)
    assert abs(float(norm) - ref) <= ref * (U + 1e-11)
    c = 0.1 / (ref + 1e-6)
    assert bool(((wide.double() - keep.double() * c).abs() <= keep.double().abs() * c * 3 * U + SUBNORMAL[torch.float32]).all())


def _busy():
    """Some hundred milliseconds of work in front of whatever the current stream gets next."""
    a = torch.ones(8192, 8192, device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    for _ in range(300):
        torch.mm(a, a, out=b)


@pytest.mark.parametrize("call", ["clip", "step", "count"])
def test_other_python_threads_run_while_the_host_waits(call):
    """clip and step: for the norm; count: for a step count on the GPU.  What a thread does to `.grad` meanwhile does not
    reach the call."""
    import threading
    import time

    import gsplat_optim as G
    p, q = (torch.nn.Parameter(torch.ones(5000, 3, device="cuda")) for _ in range(2))
    opt = G.FusedGaussianAdam([p, q], lr=0.1)
    for t in (p, q):
        t.grad = torch.ones_like(t)
    opt.step()
    twin = [torch.nn.Parameter(t.detach().clone()) for t in (p, q)]
    other = G.FusedGaussianAdam(twin, lr=0.1)
    for t, u in zip((p, q), twin):
        other.state[u] = {k: v.clone() for k, v in opt.state[t].items()}
        u.grad = torch.full_like(u, 2.0)
    if call == "count":
        for t in (p, q):
            opt.state[t]["step"] = opt.state[t]["step"].cuda()
    grads = [torch.full_like(t, 2.0) for t in (p, q)]
    for t, g in zip((p, q), grads):
        t.grad = g
    torch.cuda.synchronize()
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.is_set():
            time.sleep(0.001)
            ticks.append(time.perf_counter())
            if len(ticks) > 40:
                p.grad = q.grad = None

    thread = threading.Thread(target=tick)
    _busy()
    thread.start()
    begin = time.perf_counter()
    if call == "clip":
        norm = G.clip_grad_norm_([p, q], 1.0, error_if_nonfinite=True)
    else:
        norm = opt.clipped_step(1.0, error_if_nonfinite=call == "step")
    end = time.perf_counter()
    stop.set()
    thread.join()
    want = G.clip_grad_norm_(twin, 1.0) if call == "clip" else other.clipped_step(1.0)
    torch.cuda.synchronize()
    assert end - begin > 0.05, "the call had nothing to wait for"
    assert sum(begin < t < end for t in ticks) >= 20
    assert p.grad is None and q.grad is None
    assert torch.equal(norm, want)
    if call == "clip":
        assert all(torch.equal(g, u.grad) for g, u in zip(grads, twin))
    else:
        assert all(torch.equal(t, u) for t, u in zip((p, q), twin))
        assert all(float(opt.state[t]["step"]) == 2.0 for t in (p, q))


@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("sizes", [[1000, 3, (20, 7)], [16 * 4096, 1], [16 * 4096 + 1], [300_001, 77, 5000], [9_000_001]],
                         ids=["small", "17 chunks", "16 chunks and 4 bytes", "joined", "finished"])
@pytest.mark.parametrize("over", [True, False])
def test_a_norm_that_was_looked_at_first_clips_to_the_same_bits(sizes, norm_type, over):
    """The coefficient is 0.3 * norm / (norm + 1e-6), which is 0.3 to 5e-7 for norms of 2 and more; it and the product
    are rounded to float32 (2 u = 1.2e-7 together), the product once more to the tensor's type."""
    import gsplat_optim as G
    one, two = (_make(sizes, [torch.float32, torch.bfloat16, torch.float16], seed=4) for _ in range(2))
    raw = [g.clone() for g in one]
    ceiling = _norm64(one, norm_type) * (0.3 if over else 3.0)
    a = G.clip_grad_norm_(_params(one), ceiling, norm_type)
    b = G.clip_grad_norm_(_params(two), ceiling, norm_type, error_if_nonfinite=True)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(one, two))
    if over:
        assert not any(torch.equal(x, y) for x, y in zip(two, raw))
        for x, y in zip(two, raw):
            c = 0.3   # off by less than 1e-6 in all
            assert bool(((x.double() - y.double() * c).abs() <= (y.double().abs() * c) * (HALF_STEP[x.dtype] + 1e-6) + SUBNORMAL[x.dtype]).all())
    else:
        assert all(torch.equal(x, y) for x, y in zip(two, raw))


@pytest.mark.parametrize("N", [300, 4099, 60_000])
@pytest.mark.parametrize("sparse", [None, 0.3])
@pytest.mark.parametrize("ceiling", [0.01, 1e9])
def test_a_norm_that_was_looked_at_first_steps_to_the_same_bits(N, sparse, ceiling):
    """Moments that are not zero: a first step would be the same for any coefficient."""
    import gsplat_optim as G
    a, b, c = (_optimizer(N, G.FusedGaussianAdam, extra=True) for _ in range(3))
    vis = None if sparse is None else torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N)) < sparse
    rows = None if vis is None else N
    n1 = a.clipped_step(ceiling, vis, rows)
    n2 = b.clipped_step(ceiling, vis, rows, error_if_nonfinite=True)
    n3 = G.clip_grad_norm_([g["params"][0] for g in c.param_groups], ceiling, error_if_nonfinite=True)
    c.step(vis, rows)
    assert torch.equal(n1, n2) and torch.equal(n1, n3)
    for x, y, z in zip(_dump(a), _dump(b), _dump(c)):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("tensors", [40, 41, 90])
@pytest.mark.parametrize("sparse", [None, 0.0, 0.3])
@pytest.mark.parametrize("ceiling", [0.01, 1e9])
def test_a_step_of_more_tensors_than_a_launch_takes(tensors, sparse, ceiling):
    import gsplat_optim as G
    N = 700

    def make():
        gen = torch.Generator().manual_seed(tensors)
        shapes = [(N, 1 + 5 * k % 23) if sparse is not None else ((k * 977) % 5003 + 1,) if k % 3 else (N, 1 + k) for k in range(tensors)]
        opt = G.FusedGaussianAdam([{"params": [torch.nn.Parameter(torch.randn(*s, generator=gen).cuda())], "lr": 10.0 ** -(1 + k % 4),
                                    "betas": (0.8 + 0.002 * k, 0.99)} for k, s in enumerate(shapes)], eps=1e-15)
        for _ in range(2):
            _fill(opt, gen)
            opt.step()
        _fill(opt, gen)
        return opt

    a, b = make(), make()
    before = _dump(a)
    vis = None if sparse is None else torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N)) < sparse
    rows = None if vis is None else N
    for known in (False, True):
        n1 = G.clip_grad_norm_([g["params"][0] for g in b.param_groups], ceiling)
        b.step(vis, rows)
        n2 = a.clipped_step(ceiling, vis, rows, error_if_nonfinite=known)
        assert torch.equal(n1, n2)
        assert all(torch.equal(x, y) for x, y in zip(_dump(a), _dump(b)))
        for ga, gb in zip(a.param_groups, b.param_groups):
            gb["params"][0].grad = ga["params"][0].grad.clone()
    for x, y, k in zip(_dump(a)[::4], before[::4], range(tensors)):
        assert torch.equal(x, y) == (sparse == 0.0), k
