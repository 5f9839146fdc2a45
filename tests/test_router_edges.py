"""The router at its edges: derivatives it does not have, indices and offsets out
of the common range, more tokens than the kernels take at once. Definitions and
tolerances are those of ``test_router``."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mlx_iqk_b200 import balance_loss, route, route_balanced
from mlx_iqk_b200 import kernels as K
from test_router import (GRAD_TOL, LOSS_TOL, W_TOL, close, grads, make, ref_balance,
                         ref_choice)


def test_a_tangent_is_seen():
    x = torch.ones(3)
    K.refuse_tangent(x, "x")
    with forward_ad.dual_level():
        K.refuse_tangent(x, "x")
        dual = forward_ad.make_dual(x, torch.ones(3))
        for t in (dual, dual.view(3, 1)):
            with pytest.raises(K.IqkRuntimeError, match="forward-mode"):
                K.refuse_tangent(t, "x")
            with torch.no_grad(), pytest.raises(K.IqkRuntimeError, match="forward-mode"):
                K.refuse_tangent(t, "x")


@pytest.mark.gpu
def test_forward_mode_is_refused(cuda):
    z = make(5, 12, torch.float32, seed=1)
    idx, _ = route(z, 3)
    with forward_ad.dual_level():
        for primal in (z, z.clone().requires_grad_()):
            dual = forward_ad.make_dual(primal, torch.ones_like(z))
            for call in (lambda: route(dual, 3), lambda: route_balanced(dual, 3),
                         lambda: balance_loss(dual, idx)):
                with pytest.raises(K.IqkRuntimeError, match="forward-mode"):
                    call()
        assert torch.equal(route(z, 3)[0], idx)  # others are served as ever


@pytest.mark.gpu
def test_balance_of_indices_beyond_32_bits(cuda):
    """Entries outside the experts count for none, whatever their lower 32 bits are."""
    z = make(9, 10, torch.float32, seed=5)
    idx = torch.arange(27).view(9, 3) % 10
    idx[:7, 1] = torch.tensor([2 ** 32 + 3, 2 ** 32 - 1, -2 ** 32, 2 ** 40 + 1, -2 ** 63,
                               2 ** 63 - 1, 2 ** 31])
    loss, counts = balance_loss(z, idx.cuda())
    want, want_counts = ref_balance(z.double().cpu(), idx, "softmax")
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want, LOSS_TOL)


@pytest.mark.gpu
def test_memory_kept_for_the_gradient(cuda):
    """Between forward and backward a call keeps its outputs and the slopes, not the
    records that its blocks joined (148 * 1024 * 8 bytes here)."""
    x = make(4800, 1024, torch.bfloat16, seed=1).requires_grad_()

    def step():
        out = route_balanced(x, 2)
        return out, torch.cuda.memory_allocated()

    (_, w, loss, _), _ = step()
    want, = torch.autograd.grad([w, loss], [x], [torch.ones_like(w), torch.ones_like(loss)])
    del w, loss
    before = torch.cuda.memory_allocated()
    (_, w, loss, _), held = step()
    assert held - before <= 2 * 4800 * 2 * 4 + 2 * 1024 * 4 + 4096
    got, = torch.autograd.grad([w, loss], [x], [torch.ones_like(w), torch.ones_like(loss)])
    assert torch.equal(got, want)


# ------------------------------------------- segments, and more rows than at once


@pytest.mark.gpu
@pytest.mark.parametrize("scoring,renormalize", [("softmax", False), ("sigmoid", True)])
@pytest.mark.parametrize("cuts", [[3, 40, 40, 71], [0, 1], [99, 100], [100, 100], [0, 50, 130],
                                  [20, 180]])
def test_rows_outside_every_segment(cuda, scoring, renormalize, cuts):
    """Offsets need not begin at 0 nor end at the token count: the rows outside are
    routed, and counted nowhere."""
    z = make(100, 40, torch.float32, seed=len(cuts))
    offs = torch.tensor(cuts, dtype=torch.int32)
    plain = route(z, 3, scoring=scoring, renormalize=renormalize)
    idx, w, loss, counts = route_balanced(z, 3, scoring=scoring, renormalize=renormalize,
                                          offsets=offs.cuda())
    assert torch.equal(idx, plain[0]) and torch.equal(w, plain[1])
    want, want_counts = ref_balance(z.double().cpu(), idx.cpu().long(), scoring, None, offs)
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want, LOSS_TOL)
    g = torch.Generator().manual_seed(1)
    got, ref = grads(z, 3, scoring, renormalize, None, offs, torch.randn((100, 3), generator=g),
                     torch.tensor(3.0))
    close(got, ref, GRAD_TOL, scale=float(ref.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("t,segments", [(900, 300), (150, 257), (5000, 1100)])
def test_many_segments(cuda, t, segments):
    """More segments than the joining kernel keeps the row counts of, some empty, some
    wholly masked."""
    z = make(t, 24, torch.float32, seed=t)
    g = torch.Generator().manual_seed(t)
    offs = torch.cat([torch.tensor([0, t]), torch.randint(0, t + 1, (segments - 1,), generator=g)])
    offs = offs.sort().values.to(torch.int32)
    mask = torch.rand(t, generator=g) < 0.6
    idx, _, loss, counts = route_balanced(z, 3, mask=mask.cuda(), offsets=offs.cuda())
    want, want_counts = ref_balance(z.double().cpu(), idx.cpu().long(), "softmax", mask, offs)
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want, LOSS_TOL)
    got, ref = grads(z, 3, "softmax", True, mask, offs, torch.randn((t, 3), generator=g),
                     torch.tensor(float(segments)))
    close(got, ref, GRAD_TOL, scale=float(ref.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,e,scoring,renormalize", [
    (torch.float32, 60, "softmax", True), (torch.bfloat16, 200, "softmax", False),
    (torch.float16, 256, "sigmoid", True), (torch.float32, 300, "sigmoid", False)])
def test_more_rows_than_the_warps_take_at_once(cuda, dtype, e, scoring, renormalize):
    """Several rows to a warp, forward and backward, with segments that end inside a
    warp's run and rows that the mask leaves out between them."""
    t, k = 12011, 4
    z = make(t, e, dtype, seed=e)
    g = torch.Generator().manual_seed(e)
    mask = torch.rand(t, generator=g) < 0.9
    offs = torch.cat([torch.tensor([0, t]), torch.randint(0, t + 1, (37,), generator=g)])
    offs = offs.sort().values.to(torch.int32)
    kw = dict(scoring=scoring, renormalize=renormalize, mask=mask.cuda())
    idx, w = route(z, k, scale=1.5, **kw)
    zr = z.double().cpu().requires_grad_()
    want_idx, want_w = ref_choice(zr, k, scoring, renormalize, 1.5, mask)
    assert torch.equal(idx.cpu().long(), want_idx)
    close(w, want_w, W_TOL)
    x = z.clone().requires_grad_()
    b_idx, b_w, loss, counts = route_balanced(x, k, scale=1.5, offsets=offs.cuda(), **kw)
    assert torch.equal(b_idx, idx) and torch.equal(b_w, w)
    want_loss, want_counts = ref_balance(zr, want_idx, scoring, mask, offs)
    assert torch.equal(counts.cpu(), want_counts)
    close(loss, want_loss, LOSS_TOL)
    gw, gl = torch.randn((t, k), generator=g) / t, torch.tensor(1.0)
    got, = torch.autograd.grad([b_w, loss], [x], [gw.cuda(), gl.cuda()])
    want, = torch.autograd.grad((want_w * gw.double()).sum() + want_loss, [zr])
    step = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    # float16's values below 2^-14 are 2^-24 apart
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    err = (got.double().cpu() - want).abs()
    assert (err <= step * want.abs() + GRAD_TOL * want.abs().max() + tiny).all()
