"""MXFP4 quantisation and products against their definition in 64 bits.

1. Quantisation and its inverse are exact: every value equals the definition's,
   over all codes, ties, powers of two, subnormal and non-finite blocks.
2. Products: both operands' values are exact, so a result differs from the
   float64 sum only by the float32 sum's rounding. 64 products are added at
   once and the sums of such groups in turn, with truncation at worst:
   (K / 64 + 8) 2^-23 sum |x w|, and one rounding to a 16-bit output.
3. Refusals.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_iqk_b200 import (MxSwitchGLU, mx_aligned_scales, mx_dequantize, mx_linear, mx_quantize,
                          mx_switch_linear, route)
from mlx_iqk_b200 import kernels as K

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


# ------------------------------------------------------- definition, 64 bits


def ref_quantize(x: np.ndarray):
    """float64 ``x [rows, width]`` (values of a float32 or narrower type):
    codes [rows, width] 0..15 and scale bytes [rows, width / 32]."""
    rows, width = x.shape
    v = x.reshape(rows, width // 32, 32)
    bad = ~np.isfinite(v).all(-1)
    m = np.where(bad, 1.0, np.abs(np.where(np.isfinite(v), v, 0)).max(-1))
    exp = np.where(m > 0, np.frexp(m)[1] - 1 - 2, -127)
    exp = np.maximum(exp, -127)
    size = np.abs(np.where(bad[..., None], 0, v)) / np.exp2(exp.astype(np.float64))[..., None]
    dist = np.abs(size[..., None] - SIZES)
    best = dist.min(-1, keepdims=True)
    near = dist == best  # one, or two neighbours of a tie: take the even code
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(near.sum(-1) > 1, even.argmax(-1), near.argmax(-1))
    code = np.where(size > 6, 7, code) + 8 * np.signbit(v)
    byte = np.where(bad, 255, exp + 127).astype(np.uint8)
    return code.reshape(rows, width), byte


def ref_values(code, byte):
    value = SIZES[code & 7] * np.where(code & 8, -1.0, 1.0)
    scale = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return value * np.repeat(scale, 32, -1)


def rounded(x: torch.Tensor) -> np.ndarray:
    return ref_values(*ref_quantize(x.double().cpu().numpy().reshape(-1, x.shape[-1]))
                      ).reshape(x.shape)


def make_matrix(shape, seed, device="cuda"):
    """Random codes and scales near 2^-5; the float64 values."""
    g = torch.Generator().manual_seed(seed)
    *lead, width = shape
    codes = torch.randint(0, 256, (*lead, width // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(118, 126, (*lead, width // 32), generator=g, dtype=torch.uint8)
    flat = codes.numpy()
    both = np.stack([flat & 15, flat >> 4], -1).reshape(*lead, width)
    values = ref_values(both.reshape(-1, width), scales.numpy().reshape(-1, width // 32))
    return (codes.to(device), mx_aligned_scales(scales.to(device)),
            values.reshape(*lead, width))


def make_x(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g))
    return x.to(dtype).cuda()


def check(got, x64, w64, dtype):
    """``got [rows, out]`` against ``x64 w64^T`` within the bound above."""
    want, room = x64 @ w64.T, np.abs(x64) @ np.abs(w64).T
    k = x64.shape[-1]
    step = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tol = (k / 64 + 8) * 2.0 ** -23 * room * (1 + step) + step * np.abs(want) + \
        (2.0 ** -25 if dtype == torch.float16 else 0)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err / (tol + 1e-300)).max()


# ------------------------------------------------------------- quantisation


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 32), (1, 4096), (3, 96), (77, 1056), (130, 2048),
                                        (5, 32 * 17), (1000, 64)])
def test_quantize_is_exact(cuda, dtype, rows, width):
    x = make_x((rows, width), dtype, seed=rows + width)
    codes, scales = mx_quantize(x)
    code, byte = ref_quantize(x.double().cpu().numpy())
    got = codes.cpu().numpy()
    got = np.stack([got & 15, got >> 4], -1).reshape(rows, width)
    assert np.array_equal(scales.cpu().numpy(), byte)
    assert np.array_equal(got, code)
    assert scales.stride(0) % 16 == 0 or rows == 1
    back = mx_dequantize(codes, scales)
    assert np.array_equal(back.double().cpu().numpy(), ref_values(code, byte))
    for out in (torch.float16, torch.bfloat16):
        assert torch.equal(mx_dequantize(codes, scales, out), back.to(out))


@pytest.mark.gpu
def test_quantize_ties_and_extremes(cuda):
    """Every half step between codes at every exponent, and its neighbours."""
    rows = []
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99], dtype=np.float32)
    around = np.concatenate([ties, np.nextafter(ties, 0), np.nextafter(ties, np.float32(9))])
    for e in list(range(-149, -100)) + list(range(-20, 21)) + list(range(100, 126)):
        block = np.zeros(32, dtype=np.float64)
        block[:30] = around * np.where(np.arange(30) % 3, 1, -1)
        block[30], block[31] = 4.0, -0.0
        with np.errstate(over="ignore", under="ignore"):
            rows.append((block * 2.0 ** e).astype(np.float32))
    x = np.stack(rows)
    x = x[np.isfinite(x).all(1)]
    extra = np.zeros((6, 32), dtype=np.float32)
    extra[1, 4] = np.float32(1e-45)                      # the smallest subnormal
    extra[2] = np.finfo(np.float32).max
    extra[3, 7], extra[3, 8] = np.nan, 5.0
    extra[4, 0] = -np.inf
    extra[5] = np.finfo(np.float32).tiny
    x = np.concatenate([x, extra])
    codes, scales = mx_quantize(torch.from_numpy(x).cuda())
    code, byte = ref_quantize(x.astype(np.float64))
    got = codes.cpu().numpy()
    got = np.stack([got & 15, got >> 4], -1).reshape(x.shape)
    assert np.array_equal(scales.cpu().numpy(), byte)
    finite = byte[:, 0] != 255
    assert np.array_equal(got[finite], code[finite])
    back = mx_dequantize(codes, scales).double().cpu().numpy()
    assert np.array_equal(back[finite], ref_values(code, byte)[finite])
    assert np.isnan(back[~finite]).all() and (~finite).sum() == 2


@pytest.mark.gpu
def test_dequantize_every_code_and_scale(cuda):
    codes = torch.arange(256, dtype=torch.uint8).view(16, 16).repeat(16, 1).cuda()
    scales = mx_aligned_scales(torch.arange(256, dtype=torch.uint8).view(256, 1).cuda())
    got = mx_dequantize(codes, scales).double().cpu().numpy()
    flat = codes.cpu().numpy()
    code = np.stack([flat & 15, flat >> 4], -1).reshape(256, 32)
    with np.errstate(over="ignore"):  # 2^128 and beyond are no float32
        want = ref_values(code, scales.cpu().numpy()).astype(np.float32).astype(np.float64)
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.gpu
def test_quantize_strides_and_empties(cuda):
    x = make_x((40, 300), torch.bfloat16, seed=4)
    cut = x[::2, 5:5 + 256]                    # rows not on 16-byte boundaries
    a, b = mx_quantize(cut), mx_quantize(cut.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = make_x((64, 40), torch.float32, seed=5).t()
    a, b = mx_quantize(t), mx_quantize(t.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    same = x[:1, :32].expand(7, 32)            # one row seen seven times
    a, b = mx_quantize(same), mx_quantize(same.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    codes, scales = mx_quantize(torch.empty((0, 64), device="cuda"))
    assert codes.shape == (0, 32) and scales.shape == (0, 2)
    assert mx_dequantize(codes, scales).shape == (0, 64)
    codes, scales = mx_quantize(make_x((2, 3, 64), torch.float16, seed=6))
    assert codes.shape == (2, 3, 32) and scales.shape == (2, 3, 2)
    assert mx_dequantize(codes, scales).shape == (2, 3, 64)


# ------------------------------------------------------------------ products


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,out", [
    (1, 32, 1), (1, 4096, 2048), (1, 2048, 130), (2, 96, 127), (3, 544, 128), (7, 1056, 1000),
    (8, 512, 129), (9, 480, 64), (16, 4096, 257), (17, 512, 300), (33, 1024, 96),
    (64, 2080, 140), (65, 512, 513), (127, 1056, 200), (128, 1024, 128), (129, 608, 384),
    (200, 4096, 136), (256, 512, 260), (300, 64, 500), (777, 1504, 200)])
def test_linear(cuda, dtype, rows, width, out):
    codes, scales, w = make_matrix((out, width), seed=rows + width + out)
    x = make_x((rows, width), dtype, seed=rows)
    y = mx_linear(x, codes, scales)
    assert y.shape == (rows, out) and y.dtype == dtype
    check(y, rounded(x), w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,out", [
    (1, 8192, 64), (3, 16384, 200), (16, 10016, 97), (20, 8224, 33), (40, 16384, 130),
    (64, 9984, 260), (70, 16384, 300), (129, 12320, 520), (300, 20480, 128), (1, 40000, 1)])
def test_linear_of_wide_rows(cuda, rows, width, out):
    """Wide enough that CTAs share an item and join its parts; twice, since the
    counters of the first call serve the second."""
    codes, scales, w = make_matrix((out, width), seed=rows + out)
    x = make_x((rows, width), torch.float32, seed=rows)
    y = mx_linear(x, codes, scales)
    check(y, rounded(x), w, torch.float32)
    assert torch.equal(y, mx_linear(x, codes, scales))
    check(mx_linear(x.half() / 64, codes, scales), rounded(x.half() / 64), w, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,experts", [(1, 3, 5), (20, 3, 6), (90, 2, 3)])
def test_switch_linear_of_wide_rows(cuda, t, k, experts):
    codes, scales, w, x, idx = routed_case(t, k, experts, False, torch.float32, 8224, 70, t)
    idx[t // 2, 0] = -1
    for _ in range(2):
        check_routed(mx_switch_linear(x, idx.cuda(), codes, scales), x, idx, w, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 150])
def test_linear_out_types_strides_axes_and_repeats(cuda, rows):
    codes, scales, w = make_matrix((200, 1024), seed=3)
    wide = make_x((rows, 2, 1100), torch.bfloat16, seed=rows)
    x = wide[:, :1, 3:1027]
    for out in DTYPES:
        y = mx_linear(x, codes, scales, out)
        assert y.shape == (rows, 1, 200) and y.dtype == out
        check(y.view(rows, 200), rounded(x).reshape(rows, 1024), w, out)
        assert torch.equal(y, mx_linear(x, codes, scales, out))
    assert mx_linear(x[:0], codes, scales).shape == (0, 1, 200)
    assert mx_linear(x, codes[:0], scales[:0]).shape == (rows, 1, 0)


@pytest.mark.gpu
def test_linear_scales_of_every_size(cuda):
    """Scales from 2^-60 to 2^60 in one row: the sum is the largest terms'."""
    g = torch.Generator().manual_seed(2)
    codes, scales, _ = make_matrix((140, 512), seed=5)
    raw = torch.randint(67, 188, (140, 16), generator=g, dtype=torch.uint8)
    scales.copy_(raw)
    flat = codes.cpu().numpy()
    w = ref_values(np.stack([flat & 15, flat >> 4], -1).reshape(140, 512), raw.numpy())
    x = make_x((20, 512), torch.float32, seed=8)
    check(mx_linear(x, codes, scales), rounded(x), w, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 40, 140])
def test_linear_keeps_nan_to_its_rows(cuda, rows):
    codes, scales, w = make_matrix((150, 544), seed=1)
    x = make_x((rows, 544), torch.float32, seed=2)
    x[1, 100] = float("nan")
    x[2, 0] = float("inf")
    y = mx_linear(x, codes, scales)
    assert torch.isnan(y[1:3]).all()
    keep = [r for r in range(rows) if r not in (1, 2)]
    check(y[keep], rounded(x[keep]), w, torch.float32)
    scales[77, 3] = 255
    y = mx_linear(x[keep], codes, scales)
    assert torch.isnan(y[:, 77]).all()
    cols = [c for c in range(150) if c != 77]
    check(y[:, cols], rounded(x[keep]), w[cols], torch.float32)


def routed_case(t, k, experts, paired, dtype, width, out, seed):
    codes, scales, w = make_matrix((experts, out, width), seed)
    x = make_x((t, k if paired else 1, 1, width), dtype, seed + 1)
    g = torch.Generator().manual_seed(seed + 2)
    idx = torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(t)])
    return codes, scales, w, x, idx


def check_routed(y, x, idx, w, dtype):
    t, k = idx.shape
    xv = rounded(x).reshape(t, -1, x.shape[-1])
    for e in range(w.shape[0]):
        tt, jj = (idx == e).nonzero(as_tuple=True)
        if tt.numel():
            check(y[tt, jj, 0], xv[tt, jj if xv.shape[1] > 1 else 0], w[e], dtype)
    none = (idx < 0) | (idx >= w.shape[0])
    assert (y[none.to(y.device)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("t,k,experts,width,out", [
    (1, 1, 1, 32, 1), (1, 6, 64, 2048, 256), (3, 2, 5, 96, 130), (8, 6, 40, 512, 129),
    (10, 6, 16, 1056, 100), (11, 6, 300, 544, 64), (70, 3, 7, 512, 300), (300, 2, 4, 480, 150),
    (513, 6, 8, 64, 136)])
def test_switch_linear(cuda, dtype, paired, t, k, experts, width, out):
    codes, scales, w, x, idx = routed_case(t, k, experts, paired, dtype, width, out, t + width)
    y = mx_switch_linear(x, idx.cuda(), codes, scales)
    assert y.shape == (t, k, 1, out) and y.dtype == dtype
    check_routed(y, x, idx, w, dtype)
    assert torch.equal(y, mx_switch_linear(x, idx.int().cuda(), codes, scales))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [4, 30, 400])
def test_switch_linear_without_experts_and_one_for_all(cuda, t):
    codes, scales, w, x, idx = routed_case(t, 3, 6, False, torch.float32, 512, 140, t)
    idx[::3] = -1
    idx[1, 1] = -1
    ws = torch.empty(K.mx_workspace_bytes(t * 3, 6, 512, 140), dtype=torch.uint8, device="cuda")
    y = mx_switch_linear(x, idx.cuda(), codes, scales, workspace=ws)
    check_routed(y, x, idx, w, torch.float32)
    assert K.mx_read_error(ws) == 0
    idx[2, 2], idx[2, 0] = 6, -7
    y = mx_switch_linear(x, idx.cuda(), codes, scales, workspace=ws)
    check_routed(y, x, idx, w, torch.float32)
    assert K.mx_read_error(ws) == K.DEVERR_EXPERT
    idx[:] = -1
    assert (mx_switch_linear(x, idx.cuda(), codes, scales) == 0).all()
    idx[:] = 5                                 # every pair on one expert
    check_routed(mx_switch_linear(x, idx.cuda(), codes, scales), x, idx, w, torch.float32)
    empty = mx_switch_linear(x[:0], idx[:0].cuda(), codes, scales)
    assert empty.shape == (0, 3, 1, 140)


@pytest.mark.gpu
def test_switch_linear_equals_linear_of_each_expert(cuda):
    """A pair's result does not depend on which pairs share the call's tiles."""
    codes, scales, w, x, idx = routed_case(50, 4, 9, False, torch.bfloat16, 1024, 200, 9)
    y = mx_switch_linear(x, idx.cuda(), codes, scales, torch.float32)
    rows = x.view(50, 1024)
    for e in range(9):
        tt, jj = (idx == e).nonzero(as_tuple=True)
        if tt.numel():
            z = mx_linear(rows[tt.cuda()], codes[e], scales[e], torch.float32)
            step = 72 * 2.0 ** -23 * float(np.abs(rounded(x)).max() * np.abs(w).max() * 1024)
            assert (z - y[tt.cuda(), jj.cuda(), 0]).abs().max() <= step


@pytest.mark.gpu
def test_products_on_a_side_stream(cuda):
    codes, scales, _, x, idx = routed_case(100, 4, 8, False, torch.bfloat16, 1024, 256, 3)
    sel = idx.cuda()
    want = mx_switch_linear(x, sel, codes, scales)
    small = mx_switch_linear(x[:2], sel[:2], codes, scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx_switch_linear(x, sel, codes, scales)
        got_small = mx_switch_linear(x[:2], sel[:2], codes, scales)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_small, small)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 40])
def test_products_in_a_cuda_graph(cuda, t):
    codes, scales, _, x, idx = routed_case(t, 4, 8, False, torch.bfloat16, 1024, 256, 5)
    sel = idx.cuda()
    mx_switch_linear(x, sel, codes, scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mx_switch_linear(x, sel, codes, scales)
    x.copy_(make_x(x.shape, torch.bfloat16, 77))
    sel.copy_(sel.flip(0).roll(1, 1))
    for _ in range(2):
        graph.replay()
        assert torch.equal(y, mx_switch_linear(x, sel, codes, scales))


@pytest.mark.gpu
def test_outputs_past_32_bit_offsets(cuda):
    """2.2e9 outputs: the last rows are the same as in a small call."""
    out, rows = 65600, 33000
    codes, scales, _ = make_matrix((out, 32), seed=1)
    x = make_x((rows, 32), torch.bfloat16, seed=2)
    y = mx_linear(x, codes, scales)
    assert y.numel() > 2 ** 31
    assert torch.equal(y[-200:], mx_linear(x[-200:].clone(), codes, scales))
    assert torch.equal(y[:130], mx_linear(x[:130].clone(), codes, scales))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 45])
def test_layer_behind_the_router(cuda, t):
    """Router and MXFP4 experts together: logits to the layer's output. The
    reference quantises the same h: where float32 and float64 round an h to
    different codes (a tie's neighbourhood, 2^-20 of the blocks' values) one
    step of at most m / 4 enters one product, so the whole is compared in the
    2-norm."""
    E, H, I, k = 16, 256, 160, 4
    g = torch.Generator().manual_seed(t)
    layer = MxSwitchGLU(E, H, I, device="cuda")
    weights = {}
    for name, shape in (("gate", (E, I, H)), ("up", (E, I, H)), ("down", (E, H, I))):
        w = torch.randn(shape, generator=g) * 0.1
        layer.load_weights(name, w.cuda())
        weights[name] = rounded(w)
    x = torch.randn((t, H), generator=g).to(torch.bfloat16).cuda()
    logits = torch.randn((t, E), generator=g).cuda()
    mask = torch.ones(t, dtype=torch.bool, device="cuda")
    mask[1::4] = False
    idx, scores = route(logits, k, mask=mask)
    got = layer(x, idx, scores).double().cpu().numpy()
    xq = rounded(x)
    want = np.zeros((t, H))
    for r in range(t):
        for e, s in zip(idx[r].tolist(), scores[r].tolist()):
            if e < 0:
                continue
            a, b = weights["gate"][e] @ xq[r], weights["up"][e] @ xq[r]
            h = torch.from_numpy(a / (1 + np.exp(-a)) * b * s).float().view(1, I)
            want[r] += weights["down"][e] @ rounded(h)[0]
    assert (got[~mask.cpu().numpy()] == 0).all()
    assert np.linalg.norm(got - want) <= 5e-3 * np.linalg.norm(want)


@pytest.mark.gpu
def test_layer_without_scores(cuda):
    g = torch.Generator().manual_seed(3)
    layer = MxSwitchGLU(6, 64, 96, device="cuda")
    for name, shape in (("gate", (6, 96, 64)), ("up", (6, 96, 64)), ("down", (6, 64, 96))):
        layer.load_weights(name, torch.randn(shape, generator=g).cuda())
    x = torch.randn((5, 2, 64), generator=g).cuda()
    idx = torch.randint(-1, 6, (5, 2, 3), generator=g).cuda()
    pairs = layer(x, idx)
    assert pairs.shape == (5, 2, 3, 64)
    assert (pairs[idx < 0] == 0).all()
    # scores of 1 are no factor: the sum of the pairs, in the combine's order
    whole = layer(x, idx, torch.ones(idx.shape, device="cuda"))
    assert torch.equal(whole, pairs[:, :, 0] + pairs[:, :, 1] + pairs[:, :, 2])
    assert layer(x[:0], idx[:0]).shape == (0, 2, 3, 64)
    assert layer(x[:0], idx[:0], torch.ones((0, 2, 3), device="cuda")).shape == (0, 2, 64)


@pytest.mark.gpu
def test_example_trains_and_serves(cuda):
    """The balance loss falls towards 1, and a decode step repeats the prefill's
    row: the same products, whose float32 sums may be cut elsewhere, so that an
    h near a tie can round to a neighbouring 4-bit value (as in the layer test)."""
    from mlx_iqk_b200 import moe_example
    seen = moe_example.run(experts=16, hidden=128, inter=64, tokens=200, top_k=2, steps=12)
    assert float(seen["balance"][-1]) < float(seen["balance"][0])
    got, want = seen["decode"], seen["prefill"][:4]
    assert float((got - want).norm()) <= 5e-3 * float(want.norm())


# ---------------------------------------------------------------- refusals


def test_abi_refuses_before_any_device_call():
    lib = K.library()
    x = 0x10000

    def q(dtype=0, rows=2, width=64, stride=64, sstride=16, p=x, c=x, s=x):
        return lib.iqk_mx_quantize(p, dtype, rows, width, stride, c, s, sstride, None)

    assert q(width=48) == 3 and q(width=0) == 3 and q(rows=-1) == 3 and q(stride=63) == 3
    assert q(sstride=8) == 5 and q(sstride=0) == 5 and q(c=x + 8) == 5 and q(s=x + 4) == 5
    assert q(p=x + 2) == 5 and q(dtype=3) == 4 and q(p=None) == 4 and q(c=None) == 4
    assert q(rows=0) == 0
    assert lib.iqk_mx_dequantize(x, x, 16, 2, 64, x + 8, 0, None) == 5
    assert lib.iqk_mx_dequantize(x, x, 16, 2, 64, None, 0, None) == 4
    assert lib.iqk_mx_workspace_bytes(8, 1, 48, 64) == 0
    need = lib.iqk_mx_workspace_bytes(8, 4, 64, 64)
    assert need > 0

    def linear(rows=8, out=64, ws=need, yd=0, y=x, w=x):
        return lib.iqk_mx_linear(x, 0, rows, 64, x, x, 16, out, 64, y, yd, w, ws, None)

    assert linear(out=0) == 3 and linear(ws=16) == 6 and linear(yd=7) == 4
    assert linear(y=None) == 4 and linear(y=x + 2) == 5 and linear(w=x + 16) == 5
    assert linear(rows=1 << 25) == 3 and linear(rows=0) == 0

    def routed(xrows=4, pairs=8, experts=4, out=64, ws=need, sel=x):
        return lib.iqk_mx_routed(x, 0, xrows, 64, sel, pairs, x, x, 16, experts, out, 64, x, 0, x,
                                 ws, None)

    assert routed(experts=0) == 3 and routed(experts=4097) == 3 and routed(xrows=3) == 3
    assert routed(sel=None) == 4 and routed(sel=x + 2) == 5 and routed(ws=need - 256) == 6
    assert routed(pairs=0) == 0


def test_host_tensors_are_refused():
    with pytest.raises(K.IqkRuntimeError):
        mx_quantize(torch.zeros(2, 64))
    with pytest.raises(K.IqkRuntimeError):
        mx_dequantize(torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((2, 2),
                                                                         dtype=torch.uint8))
    with pytest.raises(K.IqkKernelError):
        MxSwitchGLU(4, 100, 64, device="cpu")


@pytest.mark.gpu
def test_refusals(cuda):
    codes, scales, _ = make_matrix((64, 128), seed=1)
    x = torch.zeros((2, 128), device="cuda")
    with pytest.raises(K.IqkKernelError):
        mx_quantize(torch.zeros((2, 40), device="cuda"))
    with pytest.raises(K.IqkRuntimeError):
        mx_quantize(x.double())
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x.clone().requires_grad_(), codes, scales)
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x[:, :64], codes, scales)
    packed = scales.contiguous()
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x, codes, packed)          # rows of 4 bytes
    assert torch.equal(mx_linear(x, codes, mx_aligned_scales(packed)),
                       mx_linear(x, codes, scales))
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x, codes.t().contiguous().t(), scales)
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x, codes[:, :32], scales)
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x, codes.int(), scales)
    with pytest.raises(K.IqkRuntimeError):
        mx_linear(x, codes, scales, torch.int32)
    c3, s3 = codes.view(2, 32, 64), mx_aligned_scales(packed.view(2, 32, 4))
    idx = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    with pytest.raises(K.IqkRuntimeError):
        mx_switch_linear(torch.zeros((4, 1, 1, 128), device="cuda"), idx, c3, s3)
    with pytest.raises(K.IqkRuntimeError):
        mx_switch_linear(torch.zeros((3, 1, 1, 128), device="cuda"), idx.float(), c3, s3)
    with pytest.raises(K.IqkRuntimeError):
        mx_switch_linear(torch.zeros((3, 1, 1, 128), device="cuda"), idx, codes, scales)
    layer = MxSwitchGLU(2, 64, 32, device="cuda")
    with pytest.raises(K.IqkRuntimeError):
        layer.load("side", codes, scales)
    with pytest.raises(K.IqkRuntimeError):
        layer.load("gate", codes, scales)
