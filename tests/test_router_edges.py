"""The router at its edges: derivatives it does not have, indices and offsets out
of the common range, more tokens than the kernels take at once. Definitions and
tolerances are those of ``test_router``."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mlx_iqk_b200 import balance_loss, route, route_balanced
from mlx_iqk_b200 import kernels as K
from test_router import LOSS_TOL, close, make, ref_balance


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
