"""The expert router against its formulas in 64 bits.

1. The choice: indices are exact (ties to the lowest index), weights agree with
   the float64 scores; rows that a mask or -inf logits leave without experts.
2. The balance loss and the counts, over ragged segments.
3. Gradients against the formula's (float64 autograd of the same definition)
   and against differences of the kernel's own forward.
4. Refusals.

Tolerances, from float32's rounding 2^-24: a score is exp(z - c) over a sum.
z - c carries 2^-24 |z - c| into the exponent; where a score matters
|z - c| < 24, so scores agree within 32 * 2^-24 = 2e-6 of themselves, products
of two within 4e-6. The loss adds at most a few hundred positive terms in a
row before a join: 1e-5 of itself. A gradient is a difference of such
products, each at most the row's largest entry's size in play: 2e-5 of the
largest gradient. 16-bit gradients add one rounding (2^-9 or 2^-12 of the
value, and float16's smallest step).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_iqk_b200 import balance_loss, route, route_balanced
from mlx_iqk_b200 import kernels as K

W_TOL, LOSS_TOL, GRAD_TOL = 4e-6, 1e-5, 2e-5
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# ------------------------------------------------------- definition, 64 bits


def ref_choice(z, k, scoring, renormalize, scale, mask=None):
    """float64 CPU: indices by repeated first-maximum, weights from the scores."""
    z = z.detach().double().cpu() if not z.requires_grad else z
    t, e = z.shape
    zv = z.detach().numpy()
    idx = np.full((t, k), -1, dtype=np.int64)
    for r in range(t):
        if mask is not None and not bool(mask[r]):
            continue
        order = sorted(range(e), key=lambda i: (-zv[r, i], i))
        keep = [i for i in order if zv[r, i] > -np.inf][:k]
        idx[r, :len(keep)] = keep
    idx = torch.from_numpy(idx)
    here = idx >= 0
    picked = z.gather(1, idx.clamp(min=0))
    logs = picked if scoring == "softmax" else torch.nn.functional.logsigmoid(picked)
    logs = torch.where(here, logs, torch.tensor(-1e300, dtype=torch.float64))
    if renormalize:
        w = torch.exp(logs - logs.amax(1, keepdim=True).detach())
        w = w / w.sum(1, keepdim=True)
    elif scoring == "softmax":
        w = torch.softmax(torch.where(z == -torch.inf, -1e300, z), 1)
        w = w.gather(1, idx.clamp(min=0))
    else:
        w = torch.exp(logs)
    return idx, torch.where(here, w, 0.0) * scale


def ref_balance(z, idx, scoring, mask=None, offsets=None):
    t, e = z.shape
    k = idx.shape[1]
    ok = torch.ones(t, dtype=torch.bool) if mask is None else mask.cpu().clone()
    ok &= (z > -torch.inf).any(1)
    zs = torch.where(z == -torch.inf, -1e300, z)
    logs = zs if scoring == "softmax" else torch.nn.functional.logsigmoid(zs)
    s = torch.softmax(logs, 1)
    offs = [0, t] if offsets is None else offsets.tolist()
    counts = torch.zeros((len(offs) - 1, e), dtype=torch.int32)
    losses = []
    for g, (a, b) in enumerate(zip(offs[:-1], offs[1:])):
        sel = idx[a:b][ok[a:b]]
        n = sel.shape[0]
        if n == 0:
            continue
        sel = sel[(sel >= 0) & (sel < e)]
        counts[g] = torch.bincount(sel, minlength=e).int()
        losses.append((counts[g].double() * e / (k * n) * s[a:b][ok[a:b]].mean(0)).sum())
    loss = torch.stack(losses).mean() if losses else torch.zeros((), dtype=torch.float64)
    return loss, counts


def make(t, e, dtype, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((t, e), generator=g) * 1.5 + 0.5 * torch.randn(e, generator=g)
    return z.to(dtype).to(device)


def ragged(t, segments, seed):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, t + 1, (segments - 1,), generator=g)
    return torch.cat([torch.tensor([0, t]), cuts]).sort().values.to(torch.int32)


def close(got, want, tol, scale=None):
    got, want = got.detach().double().cpu(), want.detach().double()
    ref = want.abs() if scale is None else torch.full_like(want, scale)
    bad = (got - want).abs() > tol * ref + 1e-30
    assert not bad.any(), ((got - want).abs() / (ref + 1e-30)).max()


# --------------------------------------------------------------- the choice


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring,renormalize",
                         [("softmax", True), ("softmax", False), ("sigmoid", True),
                          ("sigmoid", False)])
@pytest.mark.parametrize("t,e,k", [(1, 256, 6), (5, 1, 1), (33, 7, 7), (64, 60, 4), (9, 129, 8),
                                   (130, 256, 8), (3, 512, 1), (4, 1000, 32), (17, 33, 2)])
def test_choice_and_weights(cuda, dtype, scoring, renormalize, t, e, k):
    z = make(t, e, dtype, seed=t * e + k)
    idx, w = route(z, k, scoring=scoring, renormalize=renormalize, scale=1.5)
    want_idx, want_w = ref_choice(z, k, scoring, renormalize, 1.5)
    assert torch.equal(idx.cpu().long(), want_idx)
    close(w, want_w, W_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("e", [8, 40, 256, 300])
def test_ties_go_to_the_lowest_index(cuda, e):
    g = torch.Generator().manual_seed(e)
    z = torch.randint(-2, 3, (50, e), generator=g).float().cuda()
    z[0] = 0.0
    z[1, ::2] = -0.0
    z[1, 1::2] = 0.0  # -0 and +0 are equal
    k = min(8, e)
    idx, _ = route(z, k)
    assert torch.equal(idx.cpu().long(), ref_choice(z, k, "softmax", True, 1.0)[0])
    assert idx[0].tolist() == list(range(k)) and idx[1].tolist() == list(range(k))


@pytest.mark.gpu
@pytest.mark.parametrize("scoring,renormalize",
                         [("softmax", True), ("softmax", False), ("sigmoid", True),
                          ("sigmoid", False)])
def test_masked_rows_and_experts(cuda, scoring, renormalize):
    z = make(40, 70, torch.float32, seed=3)
    mask = torch.ones(40, dtype=torch.bool)
    mask[::3] = False
    z[0] = float("nan")       # masked: not looked at
    z[3] = float("inf")       # masked
    z[1] = -torch.inf         # no expert at all
    z[2, 3:] = -torch.inf     # fewer experts than top_k
    z[4, 5] = -torch.inf
    z[5] = torch.finfo(torch.float32).min   # the type's lowest value is a number
    z[7, 1:] = torch.finfo(torch.float32).min
    z[8] = -200.0             # every sigmoid underflows
    z[8, 9] = -199.0
    z[10] = 3.0e38
    idx, w = route(z, 6, scoring=scoring, renormalize=renormalize, mask=mask.cuda())
    want_idx, want_w = ref_choice(z, 6, scoring, renormalize, 1.0, mask)
    assert torch.equal(idx.cpu().long(), want_idx)
    fine = torch.ones(40, dtype=torch.bool)
    if not renormalize and scoring == "sigmoid":
        fine[8] = False  # e^-200 is below float32: 0
        assert (w[8].abs() < 1e-37).all()
    close(w[fine.cuda()], want_w[fine], 2e-5)  # |z - c| near 100 in row 2 and 8
    assert (idx[0] == -1).all() and (w[0] == 0).all() and (idx[1] == -1).all()
    assert idx[2].tolist()[3:] == [-1] * 3


@pytest.mark.gpu
def test_nan_and_infinite_logits_reach_the_weights(cuda):
    z = make(3, 16, torch.float32, seed=1)
    z[0, 7] = float("nan")
    z[1, 9] = float("inf")
    idx, w = route(z, 4, renormalize=False)
    assert idx[0, 0] == 7 and torch.isnan(w[0]).all()
    assert idx[1, 0] == 9 and torch.isnan(w[1, 0])
    assert torch.isfinite(w[2]).all()


@pytest.mark.gpu
def test_empty_strided_and_leading_axes(cuda):
    idx, w = route(torch.empty((0, 8), device="cuda"), 2)
    assert idx.shape == (0, 2) and w.shape == (0, 2)
    wide = make(30, 100, torch.bfloat16, seed=9)
    cut = wide[::2, 3:67]                      # strided rows, odd start
    a = route(cut, 4)
    b = route(cut.contiguous(), 4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = route(cut.contiguous().view(3, 5, 64), 4)
    assert c[0].shape == (3, 5, 4) and torch.equal(c[0].view(15, 4), b[0])
    d = route(wide.t(), 4)                     # transposed: columns not adjacent
    e = route(wide.t().contiguous(), 4)
    assert torch.equal(d[0], e[0])


# --------------------------------------------------- balance loss and counts


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k,segments,masked",
                         [(1, 4, 1, 1, False), (37, 60, 4, 1, True), (1000, 256, 6, 9, True),
                          (1203, 17, 3, 40, False), (8, 1000, 8, 3, False), (2500, 64, 2, 1, True)])
def test_balance(cuda, dtype, scoring, t, e, k, segments, masked):
    z = make(t, e, dtype, seed=t + e)
    mask = torch.rand(t, generator=torch.Generator().manual_seed(t)) < 0.8 if masked else None
    offs = ragged(t, segments, t) if segments > 1 else None
    kw = dict(scoring=scoring, mask=None if mask is None else mask.cuda(),
              offsets=None if offs is None else offs.cuda())
    idx, w, loss, counts = route_balanced(z, k, renormalize=False, **kw)
    plain = route(z, k, renormalize=False, scoring=scoring, mask=kw["mask"])
    assert torch.equal(idx, plain[0]) and torch.equal(w, plain[1])
    want, want_counts = ref_balance(z.double().cpu(), idx.cpu().long(), scoring, mask, offs)
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want, LOSS_TOL)
    again = balance_loss(z, idx, **kw)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts)
    assert torch.equal(route_balanced(z, k, renormalize=False, **kw)[2], loss)  # repeats


@pytest.mark.gpu
def test_balance_without_any_row(cuda):
    z = make(6, 8, torch.float32, seed=2)
    off = torch.zeros(6, dtype=torch.bool, device="cuda")
    _, _, loss, counts = route_balanced(z, 2, mask=off)
    assert loss == 0 and (counts == 0).all()
    _, _, loss, counts = route_balanced(torch.empty((0, 8), device="cuda"), 2)
    assert loss == 0 and counts.shape == (1, 8) and (counts == 0).all()
    z[1] = -torch.inf
    offs = torch.tensor([0, 0, 1, 2, 6, 6], dtype=torch.int32, device="cuda")
    idx, _, loss, counts = route_balanced(z, 2, offsets=offs)
    want, want_counts = ref_balance(z.double().cpu(), idx.cpu().long(), "softmax", None,
                                    offs.cpu())
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want, LOSS_TOL)


@pytest.mark.gpu
def test_balance_of_a_choice_with_stray_indices(cuda):
    z = make(20, 10, torch.float32, seed=5)
    idx = torch.randint(-3, 14, (20, 3), generator=torch.Generator().manual_seed(1))
    loss, counts = balance_loss(z, idx.cuda())
    want, want_counts = ref_balance(z.double().cpu(), idx, "softmax")
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want, LOSS_TOL)


# --------------------------------------------------------------- gradients


def grads(z, k, scoring, renormalize, mask, offs, gw, gl):
    """The kernel's gradient and the definition's."""
    x = z.clone().requires_grad_()
    idx, w, loss, _ = route_balanced(x, k, scoring=scoring, renormalize=renormalize, scale=1.5,
                                     mask=None if mask is None else mask.cuda(),
                                     offsets=None if offs is None else offs.cuda())
    got, = torch.autograd.grad([w, loss], [x], [gw.cuda(), gl.cuda()])
    zr = z.double().cpu().requires_grad_()
    ridx, rw = ref_choice(zr, k, scoring, renormalize, 1.5, mask)
    rl, _ = ref_balance(zr, ridx, scoring, mask, offs)
    want, = torch.autograd.grad((rw * gw.double()).sum() + rl * gl.double(), [zr])
    return got, want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring,renormalize",
                         [("softmax", True), ("softmax", False), ("sigmoid", True),
                          ("sigmoid", False)])
@pytest.mark.parametrize("t,e,k,segments,masked", [(1, 8, 2, 1, False), (70, 60, 4, 5, True),
                                                   (33, 256, 6, 1, True), (6, 700, 9, 2, False)])
def test_gradient_against_the_formula(cuda, dtype, scoring, renormalize, t, e, k, segments,
                                      masked):
    z = make(t, e, dtype, seed=7 * t + e)
    g = torch.Generator().manual_seed(t)
    mask = torch.rand(t, generator=g) < 0.8 if masked else None
    offs = ragged(t, segments, t) if segments > 1 else None
    gw, gl = torch.randn((t, k), generator=g), torch.tensor(3.0)
    got, want = grads(z, k, scoring, renormalize, mask, offs, gw, gl)
    assert got.dtype == dtype
    step = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    err = (got.double().cpu() - want).abs()
    assert (err <= step * want.abs() + GRAD_TOL * want.abs().max() + 1e-7 * (step > 0)).all()


@pytest.mark.gpu
def test_gradient_of_rows_without_experts_is_zero(cuda):
    z = make(12, 40, torch.float32, seed=4)
    z[1] = -torch.inf
    z[2, 2:] = -torch.inf
    z[3] = float("nan")
    mask = torch.ones(12, dtype=torch.bool)
    mask[3] = mask[5] = False
    got, want = grads(z, 4, "softmax", False, mask, None, torch.randn(12, 4), torch.tensor(2.0))
    for r in (1, 3, 5):
        assert (got[r] == 0).all()
    keep = [r for r in range(12) if r not in (1, 3, 5)]
    close(got[keep], want[keep], GRAD_TOL, scale=float(want[keep].abs().max()))
    assert (got[2, 2:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False),
                                                 ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(cuda, scoring, renormalize):
    """Central differences of the kernel's forward along random directions.
    Logits sit 1/4 apart and h = 2^-6, so no choice changes. The objective is
    of size 1 in float32: 2^-24 * 10 / h = 4e-5 of noise; the cut-off term
    h^2 |f'''| / 6 is below 4e-5 |d|^3."""
    g = torch.Generator().manual_seed(11)
    t, e, k, h = 5, 24, 3, 2.0 ** -6
    z = torch.stack([torch.randperm(e, generator=g) for _ in range(t)]).float().cuda() / 4 - 3
    gw = (torch.randn((t, k), generator=g) / t).cuda()

    def value(x):
        _, w, loss, _ = route_balanced(x, k, scoring=scoring, renormalize=renormalize)
        return (w * gw).sum() + loss

    x = z.clone().requires_grad_()
    grad, = torch.autograd.grad(value(x), [x])
    for _ in range(6):
        d = torch.randn(z.shape, generator=g).cuda()
        d = d / d.abs().max()
        diff = (value(z + h * d) - value(z - h * d)) / (2 * h)
        assert abs(float(diff) - float((grad * d).sum())) < 5e-4


@pytest.mark.gpu
def test_one_gradient_alone_broadcast_gradients_and_no_second_derivative(cuda):
    z = make(9, 20, torch.float32, seed=8)
    x = z.clone().requires_grad_()
    idx, w = route(x, 3)
    got, = torch.autograd.grad(w[:, 0].sum(), [x], retain_graph=True)
    gw = torch.zeros(9, 3)
    gw[:, 0] = 1
    zr = z.double().cpu().requires_grad_()
    want, = torch.autograd.grad((ref_choice(zr, 3, "softmax", True, 1.0)[1] * gw).sum(), [zr])
    close(got, want, GRAD_TOL, scale=float(want.abs().max()))
    x = z.clone().requires_grad_()
    idx, w = route(x, 3, renormalize=False)
    got, = torch.autograd.grad(w, [x], torch.ones((), device="cuda").expand(9, 3))
    zr = z.double().cpu().requires_grad_()
    want, = torch.autograd.grad(ref_choice(zr, 3, "softmax", False, 1.0)[1].sum(), [zr])
    close(got, want, GRAD_TOL, scale=float(want.abs().max()))
    x = z.clone().requires_grad_()
    loss, _ = balance_loss(x, idx)
    got, = torch.autograd.grad(loss, [x])
    zr = z.double().cpu().requires_grad_()
    want, = torch.autograd.grad(ref_balance(zr, idx.cpu().long(), "softmax")[0], [zr])
    close(got, want, GRAD_TOL, scale=float(want.abs().max()))
    x = z.view(3, 3, 20).clone().requires_grad_()
    _, w, loss, _ = route_balanced(x, 3)
    (w.sum() + loss).backward()
    assert x.grad.shape == x.shape


@pytest.mark.gpu
def test_gradient_of_other_layouts_and_changed_logits(cuda):
    z = make(24, 16, torch.float32, seed=3)
    gw = torch.randn((24, 2), generator=torch.Generator().manual_seed(1)).cuda()

    def grad(x, view):
        idx, w = route(view(x), 2, renormalize=False)
        return torch.autograd.grad(w.reshape(24, 2), [x], gw)[0]

    want = grad(z.clone().requires_grad_(), lambda x: x)
    assert torch.equal(grad(z.clone().requires_grad_(), lambda x: x.view(2, 3, 4, 16)), want)
    t = z.t().contiguous().requires_grad_()    # columns not adjacent
    assert torch.equal(grad(t, lambda x: x.t()).t(), want)
    for shape in ((24, 16), (4, 6, 16)):       # logits written over before their gradient
        x = z.clone().view(shape)
        y = x.requires_grad_() * 1.0
        _, w = route(y, 2)
        y.add_(1.0)
        with pytest.raises(RuntimeError):
            w.sum().backward()


@pytest.mark.gpu
def test_on_a_side_stream(cuda):
    z = make(3000, 256, torch.bfloat16, seed=6)
    want = route_balanced(z, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = route_balanced(z, 6)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- refusals


def test_host_tensors_are_refused():
    with pytest.raises(K.IqkRuntimeError):
        route(torch.zeros(2, 8), 2)
    with pytest.raises(K.IqkRuntimeError):
        balance_loss(torch.zeros(2, 8), torch.zeros(3, 2, dtype=torch.int32))


def test_abi_refuses_before_any_device_call():
    lib = K.library()
    x = 0x10000

    def go(dtype=0, t=4, e=8, stride=8, k=2, scoring=0, idx=x, w=x, z=x):
        return lib.iqk_route(z, dtype, t, e, stride, None, k, scoring, 1, 1.0, idx, w, None)

    assert go(dtype=5) == 4 and go(scoring=2) == 4 and go(idx=None) == 4 and go(z=None) == 4
    assert go(e=0) == 3 and go(e=1025, stride=2000) == 3 and go(k=0) == 3 and go(k=9) == 3
    assert go(e=64, stride=64, k=33) == 3 and go(t=-1) == 3 and go(stride=7) == 3
    assert go(idx=x + 2) == 5 and go(z=x + 2) == 5
    assert go(t=0) == 0
    assert lib.iqk_balance_workspace_bytes(4, 8, 0) == 0
    need = lib.iqk_balance_workspace_bytes(4, 8, 1)
    assert need > 0

    def bal(ws=need, segments=1, offsets=None, loss=x):
        return lib.iqk_route_balanced(x, 0, 4, 8, 8, None, offsets, segments, 2, 0, 1, 1.0, x, x,
                                      loss, x, x, x, ws, None)

    assert bal(ws=need - 1) == 6 and bal(segments=0) == 3 and bal(segments=2) == 3
    assert bal(loss=None) == 4 and bal(offsets=x + 1) == 5

    def back(gw=x, slope=x, gl=x, out=x, idx=x):
        return lib.iqk_route_backward(x, 0, 4, 8, 8, None, None, 1, 2, 0, 1, 1.0, idx, gw, slope,
                                      gl, out, None)

    assert back(out=None) == 4 and back(gl=None) == 4 and back(idx=None) == 4
    assert back(gw=x + 1) == 5


@pytest.mark.gpu
def test_refusals(cuda):
    z = torch.zeros((4, 8), device="cuda")
    for bad in (dict(top_k=0), dict(top_k=9)):
        with pytest.raises(K.IqkKernelError):
            route(z, **bad)
    with pytest.raises(K.IqkKernelError):
        route(torch.zeros((2, 1025), device="cuda"), 2)
    with pytest.raises(K.IqkKernelError):
        route(torch.zeros((2, 0), device="cuda"), 1)
    with pytest.raises(K.IqkRuntimeError):
        route(z, 2, scoring="relu")
    with pytest.raises(K.IqkRuntimeError):
        route(z.double(), 2)
    with pytest.raises(K.IqkRuntimeError):
        route(z, 2, mask=torch.ones(3, dtype=torch.bool, device="cuda"))
    with pytest.raises(K.IqkRuntimeError):
        route(z, 2, mask=torch.ones(4, device="cuda"))
    with pytest.raises(K.IqkRuntimeError):
        route_balanced(z, 2, offsets=torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(K.IqkRuntimeError):
        route_balanced(z, 2, offsets=torch.zeros(2, device="cuda"))
    with pytest.raises(K.IqkRuntimeError):
        balance_loss(z, torch.zeros((3, 2), dtype=torch.int32, device="cuda"))
