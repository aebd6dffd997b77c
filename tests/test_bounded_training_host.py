"""No-GPU checks of the gradient norm, clipping, the Adam step under a ceiling and the eviction: what is refused, in
Python and at the C ABI, and the sum of the weights over the ranks."""
import ctypes as C
import math
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_gsdp_gloo import _free_port


def _param():
    p = torch.nn.Parameter(torch.ones(4, 3))
    p.grad = torch.ones(4, 3)
    return p


def test_there_is_no_cpu_path():
    import gsplat_optim as G
    p = _param()
    for call in (lambda: G.grad_norm(p), lambda: G.clip_grad_norm_([p], 1.0),
                 lambda: G.clipped_adam_step(torch.optim.Adam([p]), 1.0), lambda: G.FusedGaussianAdam([p]).clipped_step(1.0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        G.evict_rows(torch.ones(4), 2)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        G.accumulate_weights(torch.ones(4), [torch.ones(4)])
    with pytest.raises(RuntimeError, match="no CPU path"):
        G.evict_optimizer(torch.optim.Adam([{"params": [p], "name": "xyz"}]), torch.ones(4), 2)
    assert torch.equal(p.grad, torch.ones(4, 3)) and torch.equal(p.detach(), torch.ones(4, 3))


def test_blending_weights_need_a_gpu():
    from diff_gaussian_rasterization import GaussianRasterizationSettings, GaussianRasterizer
    z = torch.zeros
    rs = GaussianRasterizationSettings(8, 8, 1.0, 1.0, z(3), 1.0, torch.eye(4), torch.eye(4), 0, z(3), False, False, False)
    with pytest.raises(RuntimeError, match="no CPU path"):
        GaussianRasterizer(rs).blending_weights(z(4, 3), z(4, 1), z(4, 3), z(4, 4))


def test_arguments_are_checked_before_anything_runs():
    import gsplat_optim as G
    p = _param()
    with pytest.raises(RuntimeError, match="norm_type"):
        G.grad_norm(p, 0.5)
    for bad in (-1.0, math.nan):
        with pytest.raises(RuntimeError, match="max_norm"):
            G.clip_grad_norm_(p, bad)
        with pytest.raises(RuntimeError, match="max_norm"):
            G.clipped_adam_step(torch.optim.Adam([p]), bad)
    with pytest.raises(RuntimeError, match="torch.optim.Adam"):
        G.clipped_adam_step(torch.optim.SGD([p], lr=0.1), 1.0)
    with pytest.raises(RuntimeError, match="not supported"):
        G.clipped_adam_step(torch.optim.AdamW([p]), 1.0)
    sparse = torch.nn.Parameter(torch.ones(4, 3))
    sparse.grad = torch.ones(4, 3).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        G.grad_norm(sparse)
    for groups in ([{"params": [_param(), _param()], "name": "a"}], [{"params": [_param()]}]):
        with pytest.raises(RuntimeError, match="every group"):
            G.evict_optimizer(torch.optim.Adam(groups), torch.ones(4), 2)
    with pytest.raises(RuntimeError, match="'xyz'"):
        G.evict_optimizer(torch.optim.Adam([{"params": [_param()], "name": "xyz"}]), torch.ones(5), 2)
    assert float(G.grad_norm([])) == 0.0 and float(G.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0


def _stale(device="cpu", rows=8):
    """A parameter that was given more rows while its gradient kept the old ones."""
    p = torch.nn.Parameter(torch.ones(4, 3, device=device))
    p.grad = torch.ones(4, 3, device=device)
    p.data = torch.ones(rows, 3, device=device)
    assert p.grad.shape == (4, 3)
    return p


def test_a_gradient_of_another_shape_is_refused_by_the_clipped_step():
    import gsplat_optim as G
    for rows in (8, 3, 0):
        p = _stale(rows=rows)
        opt = torch.optim.Adam([p])
        with pytest.raises(RuntimeError, match="does not have its parameter's shape"):
            G.clipped_adam_step(opt, 1.0)
        assert len(opt.state) == 0 and torch.equal(p.detach(), torch.ones(rows, 3))


def test_a_gradient_of_another_shape_is_refused_by_the_step():
    import gsplat_optim as G
    for rows in (8, 3, 0):
        p = _stale(rows=rows)
        opt = G.FusedGaussianAdam([p])
        with pytest.raises(RuntimeError, match="does not have its parameter's shape"):
            opt.step()
        assert len(opt.state) == 0 and torch.equal(p.detach(), torch.ones(rows, 3))


def test_visibility_of_another_device_is_refused_by_the_step():
    import gsplat_optim as G
    p = _param()
    opt = G.FusedGaussianAdam([p])
    with pytest.raises(RuntimeError, match="visibility must be on cpu, got meta"):
        opt.step(torch.ones(4, dtype=torch.bool, device="meta"), 4)
    assert len(opt.state) == 0 and torch.equal(p.detach(), torch.ones(4, 3))


def _with_grads(*grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype))
        p.grad = g
        out.append(p)
    return out


def test_strided_gradients_that_share_memory_are_refused():
    import gsplat_optim as G
    wide = torch.zeros(50, 8)
    other = wide.view(torch.bfloat16)
    for grads in ((wide[:, 2:5], wide[:, 4:6]), (wide[:, 1], wide), (wide, wide[::2, ::2]), (wide[::2], wide[4]), (wide[:, :3], wide[:, :3]),
                  (wide[:, 0], other[:, 1]), (wide[:, 0], wide[:, 1], other[:, 3]), (wide.t()[3:5], wide[:, 4:])):
        with pytest.raises(RuntimeError, match="share memory"):
            G.clip_grad_norm_(_with_grads(*grads), 1.0)
    for grads in ((wide[:, :3], wide[:, 3:5], wide[:, 5:]), (wide[::2], wide[1::2]), (wide[:, ::2], wide[:, 1::2]), (wide[:, 0], other[:, 2::3]),
                  (wide[:25, 1:].t(), wide[25:]), tuple(wide[:, k] for k in range(8))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            G.clip_grad_norm_(_with_grads(*grads), 1.0)
    line = torch.zeros(100)
    for size, stride in (((5, 3), (1, 1)), ((4, 2), (2, 4)), ((5,), (0,)), ((3, 3, 3), (9, 2, 4))):
        with pytest.raises(RuntimeError, match="several elements in one place"):
            G.clip_grad_norm_(_with_grads(line.as_strided(size, stride)), 1.0)
    for size, stride in (((3, 2), (2, 3)), ((5, 1), (2, 0)), ((4, 4), (10, 2))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            G.clip_grad_norm_(_with_grads(line.as_strided(size, stride)), 1.0)


def test_shared_memory_is_found_as_by_listing_every_byte():
    import random

    import gsplat_optim as G
    rng = random.Random(11)
    memory = torch.zeros(4096, dtype=torch.uint8)
    verdicts = []
    for _ in range(4000):
        grads, places = [], []
        for _ in range(2):
            dtype = rng.choice([torch.float32, torch.bfloat16, torch.float16])
            size = [rng.randint(1, 5) for _ in range(rng.randint(1, 3))]
            stride = [rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 20]) for _ in size]
            base = memory.view(dtype)
            t = base.as_strided(size, stride, rng.randint(0, 60))
            e = t.element_size()
            places.append([b for i in torch.cartesian_prod(*[torch.arange(n) for n in size]).view(-1, len(size)).tolist()
                           for b in range(e * (t.storage_offset() + sum(x * s for x, s in zip(i, stride))),
                                          e * (t.storage_offset() + sum(x * s for x, s in zip(i, stride))) + e)])
            grads.append(t)
        alone = any(len(set(p)) < len(p) for p in places)
        want = "several elements" if alone else "share memory" if set(places[0]) & set(places[1]) else "no CPU path"
        with pytest.raises(RuntimeError, match=want):
            G.clip_grad_norm_(_with_grads(*grads), 1.0)
        verdicts.append(want)
    assert min(verdicts.count(v) for v in set(verdicts)) > 300 and len(set(verdicts)) == 3


@pytest.mark.parametrize("key", ["exp_avg", "exp_avg_sq", "max_exp_avg_sq"])
def test_eviction_refuses_moments_of_other_rows(key):
    """They would stay behind, and no longer belong to the rows of their parameter."""
    import gsplat_optim as G
    p = _param()
    opt = torch.optim.Adam([{"params": [p], "name": "xyz"}], amsgrad=True)
    opt.step()
    opt.state[p][key] = torch.zeros(5, 3)
    state = dict(opt.state[p])
    for budget in (2, 4):
        with pytest.raises(RuntimeError, match=f"{key} of group 'xyz'"):
            G.evict_optimizer(opt, torch.ones(4), budget)
    assert opt.param_groups[0]["params"][0] is p and all(opt.state[p][k] is t for k, t in state.items())


def test_c_abi_refuses_bad_arguments():
    from _gsplat_lib import lib
    L = lib()
    ARG, OVERFLOW, BUFFER = -1, -3, -4
    one, big = (C.c_int64 * 1)(10), (C.c_int64 * 1)(1 << 50)
    neg = (C.c_int64 * 1)(-1)
    t0, t9 = (C.c_int * 1)(0), (C.c_int * 1)(9)
    good, odd, null = (C.c_void_p * 1)(4096), (C.c_void_p * 1)(4097), (C.c_void_p * 1)(None)
    size = L.gso_norm_temp_bytes(1)
    assert size > 0 and L.gso_norm_temp_bytes(-1) == 0 and L.gso_norm_temp_bytes(0) > 0

    def norm(n=1, g=good, k=one, t=t0, kind=2, temp=4096, bytes_=size, out=4096):
        return L.gso_grad_norm(n, g, k, t, kind, temp, bytes_, out, None)
    assert norm(n=-1) == ARG and norm(g=null) == ARG and norm(g=odd) == ARG and norm(k=neg) == ARG and norm(t=t9) == ARG
    assert norm(kind=3) == ARG and norm(kind=-1) == ARG and norm(temp=None) == ARG and norm(temp=4100) == ARG
    assert norm(out=None) == ARG and norm(g=None) == ARG and norm(bytes_=8) == BUFFER
    assert norm(k=big) == OVERFLOW

    def clip(max_norm=1.0, g=good, out=4096, n=1, bytes_=size):
        return L.gso_clip_grads(n, g, one, t0, 2, max_norm, 0, 4096, bytes_, out, None)
    assert clip(-1.0) == ARG and clip(math.nan) == ARG and clip(g=odd) == ARG and clip(out=None) == ARG and clip(n=-1) == ARG
    assert clip(bytes_=size - 1) == BUFFER

    class Adam(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("param", "grad", "m", "v")] + [("rows", C.c_int64), ("width", C.c_int64)] + \
                   [(n, C.c_double) for n in ("lr", "b1", "b2", "eps", "bc1", "bc2")]

    def adam(max_norm=1.0, n=1, out=4096, **kw):
        f = dict(param=4096, grad=4096, m=4096, v=4096, rows=10, width=3, lr=0.1, b1=0.9, b2=0.99, eps=1e-8, bc1=1.0, bc2=1.0)
        f.update(kw)
        return L.gso_adam_clipped(1, good, one, t0, n, C.byref(Adam(**f)), None, 2, max_norm, 0, 4096, size, out, None)
    assert adam(-1.0) == ARG and adam(n=-1) == ARG and adam(param=None) == ARG and adam(grad=4097) == ARG
    assert adam(rows=-1) == ARG and adam(width=0) == ARG and adam(bc1=0.0) == ARG and adam(bc2=math.nan) == ARG and adam(out=None) == ARG
    assert adam(rows=1 << 31) == OVERFLOW and adam(rows=1 << 30, width=1 << 12) == OVERFLOW

    assert L.gso_accumulate_weights(-1, 4096, 0, None, None, 1.0, None) == ARG
    assert L.gso_accumulate_weights(5, None, 0, None, None, 1.0, None) == ARG
    assert L.gso_accumulate_weights(5, 4096, 1, null, None, 1.0, None) == ARG
    assert L.gso_accumulate_weights(5, 4096, 1, None, None, 1.0, None) == ARG
    assert L.gso_accumulate_weights(1 << 31, 4096, 0, None, None, 1.0, None) == OVERFLOW
    assert L.gso_accumulate_weights(0, None, 0, None, None, 1.0, None) == 0

    need = L.gso_evict_temp_bytes(1000)
    assert 0 < need <= L.gso_evict_temp_bytes(1_000_000)

    def select(N=1000, w=4096, budget=10, recent=0, rows=4096, temp=4096, bytes_=need):
        return L.gso_evict_select(N, w, budget, recent, rows, temp, bytes_, None)
    assert select(N=-1) == ARG and select(budget=-1) == ARG and select(recent=-1) == ARG and select(recent=11) == ARG
    assert select(w=None) == ARG and select(rows=None) == ARG and select(temp=None) == ARG and select(bytes_=need - 1) == BUFFER
    assert select(N=1 << 31, bytes_=1 << 40) == OVERFLOW and select(N=0) == 0 and select(budget=0, rows=None) == 0

    class Rows(C.Structure):
        _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("row_bytes", C.c_int64), ("pitch", C.c_int64)]

    def gather(n=1, K=5, rows=4096, **kw):
        f = dict(src=4096, dst=4096, row_bytes=12, pitch=12)
        f.update(kw)
        return L.gso_gather_rows_multi(n, C.byref(Rows(**f)), rows, K, None)
    assert gather(n=-1) == ARG and gather(K=-1) == ARG and gather(rows=None) == ARG and gather(src=None) == ARG
    assert gather(dst=None) == ARG and gather(row_bytes=-4) == ARG and gather(pitch=-4) == ARG
    assert gather(row_bytes=1 << 31) == OVERFLOW and gather(K=1 << 31) == OVERFLOW and gather(K=1 << 30, row_bytes=1 << 13) == OVERFLOW
    assert gather(K=0) == 0 and gather(n=0) == 0 and gather(row_bytes=0, src=None, dst=None) == 0


def _worker(rank, world, port, out_dir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    import gsdp
    own = torch.arange(5.0) * (rank + 1)
    total = gsdp.reduce_weights(own)
    torch.save(dict(own=own, total=total), os.path.join(out_dir, f"r{rank}.pt"))
    dist.destroy_process_group()


def test_weights_are_summed_over_the_ranks(tmp_path):
    import gsdp
    w = torch.arange(4.0)
    alone = gsdp.reduce_weights(w)
    assert torch.equal(alone, w) and alone.data_ptr() != w.data_ptr()
    mp.spawn(_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    for r in range(2):
        d = torch.load(os.path.join(str(tmp_path), f"r{r}.pt"), weights_only=True)
        assert torch.equal(d["own"], torch.arange(5.0) * (r + 1))      # a rank's own sums stay its own
        assert torch.equal(d["total"], torch.arange(5.0) * 3)
