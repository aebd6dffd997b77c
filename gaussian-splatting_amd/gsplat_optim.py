"""Fused Adam for the Gaussian parameter groups (one HIP kernel per tensor:
parameter, gradient and both moments are read once, 28 bytes per element).

`FusedGaussianAdam` subclasses torch.optim.Adam, keeps its param_groups and
state layout ({"step", "exp_avg", "exp_avg_sq"}), so the densification code
that edits the optimizer state (scene/gaussian_model.py:325-458) and
state_dict()/load_state_dict() work unchanged:

    self.optimizer = FusedGaussianAdam(l, lr=0.0, eps=1e-15)      # scene/gaussian_model.py:113
    ...
    gaussians.optimizer.step()                                     # dense: torch.optim.Adam's update
    gaussians.optimizer.step(radii > 0, radii.shape[0])            # sparse: train.py:339-343

The sparse step is the update of SparseGaussianAdam (graphdeco-inria/
diff-gaussian-rasterization, branch 3dgs_accel, which the reference tries to
import but does not vendor): Adam without bias correction, applied to the rows
flagged visible only.  The class is deliberately not exported from
diff_gaussian_rasterization: the reference switches its renderer to a branch
that does not work with the fork's rasterizer as soon as that import succeeds
(train.py:38-42, gaussian_renderer/__init__.py:138-150).
"""
import contextlib
import ctypes as C
import math

import torch
import torch.nn as nn

from _gsplat_lib import check, lib, stream_of


class FusedGaussianAdam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        super().__init__(params, lr=lr, betas=betas, eps=eps)

    @torch.no_grad()
    def step(self, visibility=None, N=None, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        L = lib()
        vis = None
        if visibility is not None:
            # a row is visible where the mask is not zero, whatever its type (radii, weights)
            vis = visibility if visibility.dtype in (torch.bool, torch.uint8) else visibility != 0
            vis = vis.contiguous().view(torch.uint8)
        current = None   # the device whose context is entered: once for all tensors where they are on one
        with contextlib.ExitStack() as contexts:
            for group in self.param_groups:
                beta1, beta2 = group["betas"]
                lr, eps = float(group["lr"]), float(group["eps"])
                for p in group["params"]:
                    g = p.grad
                    if g is None:
                        continue
                    shape, dev = p.shape, p.device
                    rows = shape[0] if shape else 1
                    # a group that is not per-Gaussian takes no sparse step
                    idle = vis is not None and N is not None and rows != N
                    if not idle and g.shape != shape:   # a gradient outlives `p.data = other`
                        raise RuntimeError(f"FusedGaussianAdam: a gradient of shape {tuple(g.shape)} does not have its "
                                           f"parameter's shape {tuple(shape)}")
                    if not idle and vis is not None and vis.device != dev:
                        raise RuntimeError(f"FusedGaussianAdam: visibility must be on {dev}, got {vis.device}")
                    if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                        raise RuntimeError("FusedGaussianAdam needs contiguous float32 GPU parameters (there is no CPU path)")
                    st = self.state[p]
                    if len(st) == 0:
                        st["step"] = torch.tensor(0.0, dtype=torch.float32)
                        st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                        st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    if idle:
                        continue
                    g = g if g.is_contiguous() else g.contiguous()
                    m, v = st["exp_avg"], st["exp_avg_sq"]
                    for t in (g, m, v):
                        if t.dtype is not torch.float32 or t.device != dev or t.shape != shape or not t.is_contiguous():
                            raise RuntimeError("FusedGaussianAdam: gradient and moments must be contiguous float32 tensors of "
                                               f"the parameter's shape {tuple(shape)} on {dev}, got {tuple(t.shape)} "
                                               f"{t.dtype} on {t.device}")
                    width = p.numel() // max(rows, 1)
                    if vis is not None:
                        if vis.numel() != rows:
                            raise RuntimeError("visibility must have one entry per Gaussian")
                        bc1, bc2s = 1.0, 1.0
                    else:
                        st["step"] += 1
                        t = float(st["step"])
                        bc1, bc2s = 1.0 - beta1 ** t, math.sqrt(1.0 - beta2 ** t)
                    if dev != current:
                        contexts.enter_context(torch.cuda.device(dev))
                        current = dev
                    check(L.gso_adam_update(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(),
                                            None if vis is None else vis.data_ptr(), rows, width, lr, beta1, beta2, eps, bc1,
                                            bc2s, stream_of(dev)),
                          "adam update")
        return loss

    def clipped_step(self, max_norm, visibility=None, N=None, norm_type=2.0, error_if_nonfinite=False):
        """`clip_grad_norm_` over all of this optimizer's gradients followed by `step(visibility, N)`, in two passes
        over the data: see `clipped_adam_step`.  Returns the norm before clipping."""
        return clipped_adam_step(self, max_norm, visibility, N, norm_type, error_if_nonfinite)


# ---------------------------------------------------------------- gradient norm and clipping
_host_layer = None


def _host():
    """The compiled host layer (csrc/torch/optim_ext.cpp)."""
    global _host_layer
    if _host_layer is None:
        from diff_gaussian_rasterization import _C
        if _C._hip_ext is None:
            raise ImportError("the PyTorch host extension is missing or was replaced by a library override: build it with "
                              "`python gaussian-splatting_amd/csrc/torch/build_ext.py` (there is no CPU fallback)")
        _host_layer = _C._hip_ext
    return _host_layer


def _tensors(parameters):
    return [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)


def grad_norm(parameters, norm_type=2.0):
    """The norm of all the gradients of `parameters` (an iterable of tensors, or one) together, as if they were one
    vector: norm_type 2, 1 or inf.  A 0-d float32 tensor on the gradients' device; the host does not wait for it.

    Parameters without a gradient are left out (without any: a CPU zero, as torch.nn.utils.clip_grad_norm_ gives).
    Gradients are float32, bfloat16 or float16 GPU tensors of one device, of mixed types and any sizes.  Sums are held
    in 64 bits and added in an order that the tensors' sizes and their addresses modulo 16 fix, so the result does not
    depend on the run, and replicas with the same gradients in the same layout (a `ParamGradSink` each, after
    `gsdp.GradReducer`) get the same bits.  A NaN makes the norm NaN; one beyond float32 is infinite."""
    return _host().grad_norm(_tensors(parameters), float(norm_type))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_: scales the gradients in place by min(1, max_norm / (norm + 1e-6)) and returns
    the norm they had (`grad_norm`).  Under the ceiling the gradients are read once and not written.  As there, a
    norm that is NaN makes every gradient NaN, and an infinite one makes them zero (NaN where they were infinite);
    with error_if_nonfinite=True the host waits for the norm and a RuntimeError leaves the gradients as they were (not
    under stream capture).  Two gradients must not share memory.

    With `ParamGradSink(keep_zero_rows=True)`: scaling leaves zero rows zero, so nothing has to be marked, unless the
    norm is not finite; a caller that goes on after that calls `sink.mark_rows_dirty()`.
    When an Adam step follows, `clipped_adam_step` does both with fewer bytes."""
    return _host().clip_grad_norm(_tensors(parameters), float(max_norm), float(norm_type), bool(error_if_nonfinite))


def clipped_adam_step(optimizer, max_norm, visibility=None, N=None, norm_type=2.0, error_if_nonfinite=False):
    """`clip_grad_norm_(all parameters of the optimizer, max_norm)` followed by `FusedGaussianAdam.step(visibility, N)`
    for a torch.optim.Adam (or FusedGaussianAdam): one pass that sums and one that updates every tensor, which
    applies the coefficient on the fly.  Parameters and moments get the same bits as from the two calls; the `.grad`
    tensors keep their unclipped values.  Returns the norm before clipping (0-d tensor, not waited for).

    The norm counts every gradient of the optimizer, also those of groups that take no sparse step because their rows
    are not N.  Needs contiguous float32 GPU parameters and plain Adam groups (no weight decay, amsgrad, maximize,
    capturable, fused); cannot be captured into a graph (the bias correction is a number of the host).  Hooks that were
    registered on `step` do not run.  error_if_nonfinite: the host waits for the norm and a RuntimeError leaves
    parameters, moments and step counts as they were."""
    what = "clipped_adam_step"
    if not isinstance(optimizer, torch.optim.Adam):
        raise RuntimeError(f"{what} needs a torch.optim.Adam, got {type(optimizer).__name__}")
    if not float(max_norm) >= 0.0:
        raise RuntimeError(f"{what}: max_norm must not be negative or NaN, got {max_norm}")
    for group in optimizer.param_groups:
        if group["weight_decay"] or group["amsgrad"] or group["maximize"] or group["capturable"] or \
                group["differentiable"] or group["fused"]:
            raise RuntimeError(f"{what}: weight_decay, amsgrad, maximize, capturable, differentiable and fused are not supported")
    by_rows = visibility is not None and N is not None   # then a group that is not per-Gaussian takes no step
    params, m, v, steps, scalars, idle, fresh = [], [], [], [], [], [], []
    try:
        for group in optimizer.param_groups:
            beta1, beta2 = group["betas"]
            numbers = (float(group["lr"]), float(beta1), float(beta2), float(group["eps"]))
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = optimizer.state[p]
                if len(st) == 0:
                    fresh.append(p)
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                params.append(p)
                m.append(st["exp_avg"])
                v.append(st["exp_avg_sq"])
                steps.append(st["step"])
                scalars += numbers
                idle.append(by_rows and (p.shape[0] if p.dim() > 0 else 1) != N)
        return _host().clipped_adam(params, m, v, steps, scalars, idle, visibility, float(max_norm), float(norm_type),
                                    bool(error_if_nonfinite))
    except Exception:
        for p in fresh:
            del optimizer.state[p]
        raise


@torch.no_grad()
def add_densification_stats(radii, viewspace_grad, xyz_gradient_accum, denom, max_radii2D):
    """One fused pass for what train.py:298-312 and GaussianModel.add_densification_stats
    (scene/gaussian_model.py:202-214) do after every iteration, without the host-blocking
    `nonzero()` of the visibility mask: for Gaussians with radii > 0,
    max_radii2D = max(max_radii2D, radii), xyz_gradient_accum += |viewspace_grad[:, :2]|, denom += 1.
    All tensors are updated in place; `viewspace_grad` is `viewspace_point_tensor.grad` ([P,3])."""
    P = radii.shape[0]
    for t, shape in ((viewspace_grad, (P, 3)), (xyz_gradient_accum, (P, 1)), (denom, (P, 1)), (max_radii2D, (P,))):
        if tuple(t.shape) != shape or t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
            raise RuntimeError(f"expected a contiguous float32 GPU tensor of shape {shape}, got {tuple(t.shape)} {t.dtype}")
    if radii.dtype != torch.int32 or not radii.is_contiguous():
        raise RuntimeError("radii must be the contiguous int32 tensor the rasterizer returned")
    with torch.cuda.device(radii.device):
        check(lib().gso_densify_stats(P, radii.data_ptr(), viewspace_grad.data_ptr(), xyz_gradient_accum.data_ptr(),
                                      denom.data_ptr(), max_radii2D.data_ptr(), stream_of(radii.device)),
              "densify stats")


class RowCompactor:
    """The kept rows of a boolean mask, computed once and applied to any number of tensors:
    `RowCompactor(mask)(t)` equals `t[mask]` for tensors whose first dimension is the mask's
    length.  One host block (to learn how many rows are kept) instead of one per tensor."""

    def __init__(self, mask):
        if mask.dim() != 1 or not mask.is_cuda:
            raise RuntimeError("mask must be a 1-D GPU tensor (there is no CPU path)")
        L = lib()
        self.N = mask.shape[0]
        self.device = mask.device
        keep = (mask != 0).to(torch.uint8).contiguous() if mask.dtype not in (torch.uint8, torch.bool) else \
            mask.contiguous().view(torch.uint8)
        self.index = torch.empty((max(self.N, 1),), dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            temp = torch.empty((L.gso_compact_temp_bytes(self.N),), dtype=torch.uint8, device=self.device)
            kept = C.c_int64(0)
            check(L.gso_compact_map(self.N, keep.data_ptr() if self.N else None, self.index.data_ptr(), temp.data_ptr(),
                                    temp.numel(), C.byref(kept), stream_of(self.device)), "compact map")
        self.kept = int(kept.value)

    def __call__(self, t):
        if t.shape[0] != self.N or t.device != self.device:
            raise RuntimeError("tensor does not match the mask")
        if t.element_size() != 4 or not t.is_contiguous():
            return t[self.index[:self.kept].long()]   # other layouts: plain indexing with the same list
        out = torch.empty((self.kept,) + tuple(t.shape[1:]), dtype=t.dtype, device=t.device)
        M = t.numel() // max(self.N, 1)
        if self.kept and M:
            with torch.cuda.device(self.device):
                check(lib().gso_gather_rows(t.data_ptr(), out.data_ptr(), self.index.data_ptr(), self.kept, M,
                                            stream_of(self.device)), "gather rows")
        return out


@torch.no_grad()
def prune_optimizer(optimizer, mask):
    """GaussianModel._prune_optimizer (scene/gaussian_model.py:427-441) with the mask resolved once:
    keeps the rows of `mask` in every group's parameter and in its Adam moments, re-registers the
    state under the new nn.Parameter and returns {group name: new parameter}.  Also returns the
    compactor as the second value, for the per-Gaussian statistics tensors that prune_points
    filters next (scene/gaussian_model.py:419-424)."""
    comp = RowCompactor(mask)
    optimizable = {}
    for group in optimizer.param_groups:
        p = group["params"][0]
        stored = optimizer.state.get(p, None)
        new_p = nn.Parameter(comp(p.data).requires_grad_(True))
        if stored is not None:
            stored["exp_avg"] = comp(stored["exp_avg"])
            stored["exp_avg_sq"] = comp(stored["exp_avg_sq"])
            del optimizer.state[p]
            optimizer.state[new_p] = stored
        group["params"][0] = new_p
        optimizable[group["name"]] = new_p
    return optimizable, comp


@torch.no_grad()
def cat_tensors_to_optimizer(optimizer, tensors_dict):
    """GaussianModel.cat_tensors_to_optimizer (scene/gaussian_model.py:325-346): appends the new
    rows to every group's parameter, zero moments for them, returns {group name: new parameter}."""
    optimizable = {}
    for group in optimizer.param_groups:
        assert len(group["params"]) == 1
        ext = tensors_dict[group["name"]]
        p = group["params"][0]
        stored = optimizer.state.get(p, None)
        new_p = nn.Parameter(torch.cat((p.data, ext), dim=0).requires_grad_(True))
        if stored is not None:
            stored["exp_avg"] = torch.cat((stored["exp_avg"], torch.zeros_like(ext)), dim=0)
            stored["exp_avg_sq"] = torch.cat((stored["exp_avg_sq"], torch.zeros_like(ext)), dim=0)
            del optimizer.state[p]
            optimizer.state[new_p] = stored
        group["params"][0] = new_p
        optimizable[group["name"]] = new_p
    return optimizable


# ---------------------------------------------------------------- densification (clone / split / prune)
def _f32(t, shape, what):
    if tuple(t.shape) != tuple(shape) or t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
        raise RuntimeError(f"{what}: expected a contiguous float32 GPU tensor of shape {tuple(shape)}, "
                           f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t


@torch.no_grad()
def densify_select(xyz_gradient_accum, denom, scaling, grad_threshold, size_threshold, split, n_grads=None):
    """The clone (split=False, scene/gaussian_model.py:263-270) or split (split=True, :356-364) selection as a
    bool mask over the N rows of `scaling` (raw log-scales), in one kernel: gradient = accum / denom with
    NaN -> 0 for the first `n_grads` rows (default: all), 0 for the rest; size_threshold = percent_dense * extent."""
    N = scaling.shape[0]
    n_grads = N if n_grads is None else int(n_grads)
    _f32(scaling, (N, 3), "scaling")
    sel = torch.empty((N,), dtype=torch.uint8, device=scaling.device)
    with torch.cuda.device(scaling.device):
        check(lib().gso_densify_select(N, n_grads, xyz_gradient_accum.data_ptr() if n_grads else None,
                                       denom.data_ptr() if n_grads else None, scaling.data_ptr(), float(grad_threshold),
                                       float(size_threshold), int(bool(split)), sel.data_ptr(), stream_of(scaling.device)),
              "densify select")
    return sel.view(torch.bool)


@torch.no_grad()
def prune_mask(opacity, max_radii2D, scaling, min_opacity, max_screen_size, extent, also=None):
    """The prune decision of scene/gaussian_model.py:237-244 (+ the rows of `also`) as a bool mask, one kernel."""
    N = opacity.shape[0]
    m = torch.empty((N,), dtype=torch.uint8, device=opacity.device)
    al = None if also is None else also.contiguous().view(torch.uint8)
    with torch.cuda.device(opacity.device):
        check(lib().gso_prune_mask(N, opacity.contiguous().data_ptr(), max_radii2D.data_ptr(), scaling.data_ptr(),
                                   float(min_opacity), float(max_screen_size) if max_screen_size else 0.0,
                                   0.1 * float(extent), None if al is None else al.data_ptr(), m.data_ptr(),
                                   stream_of(opacity.device)), "prune mask")
    return m.view(torch.bool)


@torch.no_grad()
def split_children(parents, n, xyz, scaling, rotation, normals):
    """Positions and log-scales of the K * n children of the K parents (row indices, int32, ascending)
    as scene/gaussian_model.py:367-377 forms them, `normals` = the [K*n, 3] standard normal samples;
    also returns parent_of_child [K*n] (int32) for copying the other tensors' rows."""
    K = parents.shape[0]
    dev = xyz.device
    new_xyz = torch.empty((K * n, 3), dtype=torch.float32, device=dev)
    new_scaling = torch.empty((K * n, 3), dtype=torch.float32, device=dev)
    poc = torch.empty((K * n,), dtype=torch.int32, device=dev)
    if K:
        _f32(normals, (K * n, 3), "normals")
        with torch.cuda.device(dev):
            check(lib().gso_split_children(K, int(n), parents.data_ptr(), xyz.data_ptr(), scaling.data_ptr(),
                                           rotation.data_ptr(), normals.data_ptr(), new_xyz.data_ptr(),
                                           new_scaling.data_ptr(), poc.data_ptr(), stream_of(dev)), "split children")
    return new_xyz, new_scaling, poc


def _take_rows(t, rows):
    """t[rows] for an int32 row list through the row-gather kernel."""
    K = rows.shape[0]
    out = torch.empty((K,) + tuple(t.shape[1:]), dtype=t.dtype, device=t.device)
    M = t.numel() // max(t.shape[0], 1)
    if K and M:
        if t.element_size() != 4 or not t.is_contiguous():
            return t[rows.long()]
        with torch.cuda.device(t.device):
            check(lib().gso_gather_rows(t.data_ptr(), out.data_ptr(), rows.data_ptr(), K, M, stream_of(t.device)),
                  "gather rows")
    return out


@torch.no_grad()
def densify_and_prune(optimizer, stats, max_grad, min_opacity, extent, max_screen_size, radii, percent_dense=0.01,
                      n_split=2, normals=None):
    """GaussianModel.densify_and_prune (scene/gaussian_model.py:216-252) on an optimizer whose param groups carry
    the reference's names ("xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation", "reps"; one tensor each):
    clone the small Gaussians with a large view-space gradient, split the large ones into `n_split` children,
    prune the transparent and the oversized, with the Adam moments following every row.  `stats` is a dict with
    xyz_gradient_accum [N,1], denom [N,1], max_radii2D [N]; `radii` the last forward's radii (the reference's
    tmp_radii).  `normals`: the standard normal samples for the split, [n_split * (number split), 3] or a
    callable (rows) -> tensor; default torch.randn.  The selections, the split and the prune mask are one
    kernel each, every row list is resolved once (one host block per stage) and applied to all tensors.
    Returns ({group name: new parameter}, new stats dict, radii of the surviving rows)."""
    by_name = {g["name"]: g for g in optimizer.param_groups}
    P = lambda name: by_name[name]["params"][0]
    accum, den = stats["xyz_gradient_accum"], stats["denom"]
    N0 = P("xyz").shape[0]
    size_thr = percent_dense * extent
    tmp_radii = radii

    def append(rows_src, overrides):
        ext = {}
        for name in by_name:
            ext[name] = overrides[name] if name in overrides else _take_rows(P(name).data, rows_src)
        return cat_tensors_to_optimizer(optimizer, ext)

    # clone (:254-283)
    sel = densify_select(accum, den, P("scaling").data, max_grad, size_thr, split=False)
    comp = RowCompactor(sel)
    rows = comp.index[:comp.kept]
    if comp.kept:
        append(rows, {})
        tmp_radii = torch.cat((tmp_radii, _take_rows(tmp_radii, rows)))
    # split (:347-392): decided on the grown model, gradients padded with zeros for the clones
    sel = densify_select(accum, den, P("scaling").data, max_grad, size_thr, split=True, n_grads=N0)
    comp = RowCompactor(sel)
    rows = comp.index[:comp.kept]
    also = None
    if comp.kept:
        K = comp.kept
        z = normals(K * n_split) if callable(normals) else normals
        if z is None:
            z = torch.randn((K * n_split, 3), device=sel.device)
        new_xyz, new_scaling, poc = split_children(rows, n_split, P("xyz").data, P("scaling").data, P("rotation").data,
                                                   z.contiguous())
        append(poc, {"xyz": new_xyz, "scaling": new_scaling})
        tmp_radii = torch.cat((tmp_radii, _take_rows(tmp_radii, poc)))
        also = torch.cat((sel, torch.zeros(K * n_split, dtype=torch.bool, device=sel.device)))
    # densification_postfix restarts the statistics at the new size whether or not rows were appended
    # (:318-320), max_radii2D included: the screen-size test below therefore reads zeros, as it does in the
    # reference, and the returned statistics are zeros of the final size.
    N2 = P("xyz").shape[0]
    dev = P("xyz").device
    max_radii2D = torch.zeros((N2,), device=dev)
    # prune: the parents a split replaced (:388-392) and the transparent / oversized (:237-247), decided per
    # row, so one compaction serves both (the reference prunes twice; the surviving rows and their order are
    # the same)
    mask = prune_mask(P("opacity").data.view(-1), max_radii2D, P("scaling").data, min_opacity, max_screen_size, extent,
                      also=also)
    optimizable, comp = prune_optimizer(optimizer, ~mask)
    n = comp.kept
    new_stats = dict(xyz_gradient_accum=torch.zeros((n, 1), device=dev), denom=torch.zeros((n, 1), device=dev),
                     max_radii2D=torch.zeros((n,), device=dev))
    return optimizable, new_stats, comp(tmp_radii)


# ---------------------------------------------------------------- a model within a row budget
def accumulate_weights(weights, contributions, opacity=None, decay=1.0):
    """Adds what some views say about how much each Gaussian matters, in place and in one pass:

        weights = decay * weights + sigmoid(opacity) * (contributions[0] + contributions[1] + ...)

    `contributions`: a list of [N] tensors, or one.  With opacity=None they are weights as they are: the views'
    `GaussianRasterizer.blending_weights`, what each Gaussian contributed to the images, as attention weights summed over
    queries are what a cache entry gave.  With the raw opacities ([N] or [N, 1], logits) they are what is to be
    multiplied by the activated ones: the `gauss_sum` of each rendered view, which costs no rendering of its own, but
    counts the transmittance of every pixel that tests the Gaussian, whatever its alpha there.  The product is an
    upper bound of the blending weight (in free space some six times it for round splats much larger than a tile, whose
    bounding square is tested, and a hundred times and more for those below a pixel), so it ranks Gaussians of
    different sizes differently.  decay < 1 forgets old views.  All float32 on one GPU.  With several ranks each
    accumulates its own views: see `gsdp.reduce_weights`."""
    contributions = [contributions] if isinstance(contributions, torch.Tensor) else list(contributions)
    _host().accumulate_weights(weights, contributions, opacity, float(decay))
    return weights


def evict_rows(weights, budget, recent=0, tensors=()):
    """Which rows stay when a model of N rows may have only `budget`, and those rows of `tensors`.

    Kept are the last `recent` rows (densification appends new Gaussians at the end: they have had no time to gather
    weight) and, of the others, the budget - recent of largest weight; of equal weights the lower row index stays, and a
    NaN goes first.  Returns (rows, kept): `rows` [min(N, budget)] int32, ascending, and `kept[k] = tensors[k][rows]`
    as new contiguous tensors, for any number of tensors of any type with N rows.  The number of rows is known
    beforehand, so unlike `RowCompactor` the host never waits.  `weights`: [N] or [N, 1], float32, on the GPU."""
    host = _host()
    rows = host.evict_select(weights, int(budget), int(recent))
    return rows, host.take_rows(_tensors(tensors), rows, weights.numel())


@torch.no_grad()
def evict_optimizer(optimizer, weights, budget, recent=0, stats=None):
    """`evict_rows` for the whole model: every group's parameter, its optimizer state and the per-Gaussian tensors
    of the dict `stats` keep the chosen rows, and the state moves to the new nn.Parameter as `prune_optimizer` moves
    it.  Returns ({group name: new parameter}, rows, new stats).  Nothing is changed if a tensor does not have one row
    per weight.  A `ParamGradSink` has to be built anew afterwards, as after densification.

    A model that has no more rows than the budget stays as it is: the same parameters with their gradients, the same
    state and the tensors of `stats` come back, and a sink stays valid (`optimizable[name] is old` tells).  Otherwise
    the old and the new tensors are alive together until the call returns, so that a failure leaves the old ones: the
    kept rows of all of them have to fit beside the model."""
    N = weights.numel()
    stats = {} if stats is None else dict(stats)
    moved = []   # (group, [state keys])
    tensors = []
    for group in optimizer.param_groups:
        if len(group["params"]) != 1 or "name" not in group:
            raise RuntimeError("evict_optimizer: every group must have a name and hold one per-Gaussian tensor")
        p = group["params"][0]
        if p.dim() == 0 or p.shape[0] != N:
            raise RuntimeError(f"evict_optimizer: group {group.get('name')!r} has shape {tuple(p.shape)}, the weights "
                               f"have {N} rows")
        st = optimizer.state.get(p, None)
        for k in ("exp_avg", "exp_avg_sq", "max_exp_avg_sq"):
            if st and k in st and st[k].shape != p.shape:
                raise RuntimeError(f"evict_optimizer: {k} of group {group['name']!r} has shape {tuple(st[k].shape)}, its "
                                   f"parameter {tuple(p.shape)}")
        keys = [k for k, t in st.items() if torch.is_tensor(t) and t.shape == p.shape] if st else []
        moved.append((group, keys))
        tensors.append(p.data)
        tensors += [st[k] for k in keys]
    tensors += list(stats.values())
    if int(budget) >= N:
        host = _host()
        rows = host.evict_select(weights, int(budget), int(recent))
        host.take_rows(tensors, rows[:0], N)   # refuses what an eviction would refuse
        return {group["name"]: group["params"][0] for group, _ in moved}, rows, stats
    rows, kept = evict_rows(weights, budget, recent, tensors)
    kept = iter(kept)
    optimizable = {}
    for group, keys in moved:
        p = group["params"][0]
        new_p = nn.Parameter(next(kept).requires_grad_(True))
        st = optimizer.state.pop(p, None)
        for k in keys:
            st[k] = next(kept)
        if st is not None:
            optimizer.state[new_p] = st
        group["params"][0] = new_p
        optimizable[group["name"]] = new_p
    return optimizable, rows, {k: next(kept) for k in stats}
