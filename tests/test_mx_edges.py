"""MXFP4 operators at their edges: where arguments live, how they are laid out,
what happens after an error. Definitions and bounds are those of ``test_mx``."""

from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

from mlx_iqk_b200 import (MxSwitchGLU, mx_dequantize, mx_linear, mx_quantize, mx_switch_linear,
                          route)
from mlx_iqk_b200 import kernels as K
from test_mx import check, check_routed, make_matrix, make_x, rounded


# ------------------------------------------------------ the layer's arguments


def small_layer(device):
    layer = MxSwitchGLU(4, 64, 32, device=device)
    x = torch.ones((3, 64), device=device)
    idx = torch.zeros((3, 2), dtype=torch.int32, device=device)
    return layer, x, idx


def test_layer_refuses_scores_elsewhere():
    layer, x, idx = small_layer("cpu")
    for scores in (torch.ones((3, 2), device="meta"), [[1.0, 1.0]] * 3):
        with pytest.raises(K.IqkRuntimeError, match="scores"):
            layer(x, idx, scores)


@pytest.mark.gpu
def test_layer_refuses_host_scores(cuda):
    layer, x, idx = small_layer("cuda")
    with pytest.raises(K.IqkRuntimeError, match="scores"):
        layer(x, idx, torch.ones((3, 2)))
    assert layer(x, idx, torch.ones((3, 2), device="cuda")).shape == (3, 64)


# ---------------------------------------------------------- caller's workspace


def test_host_workspaces_are_refused():
    x, y = torch.zeros((2, 64)), torch.zeros((2, 32))
    sel = torch.zeros(2, dtype=torch.int32)
    codes, scales = (torch.zeros((4, 32, n), dtype=torch.uint8) for n in (32, 16))
    with pytest.raises(K.IqkRuntimeError, match="workspace"):
        K.mx_routed(x, 2, 64, sel, codes, scales, 16, y,
                    torch.zeros(1 << 20, dtype=torch.uint8))
    with pytest.raises(K.IqkRuntimeError, match="workspace"):
        K.mx_read_error(torch.zeros(1 << 20, dtype=torch.uint8))


@pytest.mark.gpu
def test_workspaces_of_another_kind_are_refused(cuda):
    codes, scales, _ = make_matrix((4, 32, 64), seed=1)
    x = make_x((3, 1, 1, 64), torch.float32, seed=2)
    idx = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    need = K.mx_workspace_bytes(6, 4, 64, 32)
    want = mx_switch_linear(x, idx, codes, scales)
    good = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert torch.equal(mx_switch_linear(x, idx, codes, scales, workspace=good), want)
    for bad in (torch.empty(need, dtype=torch.uint8),
                torch.empty(need, dtype=torch.uint8).pin_memory(),
                torch.empty(need, dtype=torch.int32, device="cuda"),
                torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2],
                good[:need - 256]):
        with pytest.raises(K.IqkRuntimeError):
            mx_switch_linear(x, idx, codes, scales, workspace=bad)
    with pytest.raises(K.IqkRuntimeError, match="workspace"):
        K.mx_read_error(good[:8])
    assert K.mx_read_error(good) == 0


def test_layer_refuses_scores_that_ask_for_a_gradient():
    layer, x, idx = small_layer("cpu")
    scores = torch.ones((3, 2), requires_grad=True)
    with pytest.raises(K.IqkRuntimeError, match="no gradient.*scores"):
        layer(x, idx, scores)
    with torch.no_grad(), pytest.raises(K.IqkRuntimeError, match="on the GPU"):
        layer(x, idx, scores)  # without a graph they are plain numbers


@pytest.mark.gpu
def test_layer_behind_a_router_under_training(cuda):
    """The router's weights as scores: refused while a graph is built, served without one."""
    layer, x, idx = small_layer("cuda")
    logits = torch.zeros((3, 4), device="cuda", requires_grad=True)
    indices, weights = route(logits, 2)
    with pytest.raises(K.IqkRuntimeError, match="no gradient.*scores"):
        layer(x, indices, weights)
    want = layer(x, indices, weights.detach())
    with torch.no_grad():
        assert torch.equal(layer(x, indices, weights), want)


def test_layer_refuses_scores_with_a_tangent():
    layer, x, idx = small_layer("cpu")
    with forward_ad.dual_level():
        scores = forward_ad.make_dual(torch.ones((3, 2)), torch.ones((3, 2)))
        with pytest.raises(K.IqkRuntimeError, match="forward-mode"):
            layer(x, idx, scores)


@pytest.mark.gpu
def test_forward_mode_is_refused(cuda):
    codes, scales, _ = make_matrix((32, 64), seed=1)
    idx = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    x = torch.ones((2, 64), device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for call in (lambda: mx_quantize(dual), lambda: mx_linear(dual, codes, scales),
                     lambda: mx_switch_linear(dual.view(2, 1, 1, 64), idx, codes[None],
                                              scales[None])):
            with pytest.raises(K.IqkRuntimeError, match="forward-mode"):
                call()


# ------------------------------------------------------------- expert indices

# int64 values whose lower 32 bits name an expert, or -1
BEYOND = [2 ** 32 + 3, 2 ** 32 - 1, -2 ** 32, 2 ** 40 + 1, -2 ** 63, 2 ** 63 - 1, 2 ** 31]


def test_narrowing_refuses_before_any_device_call():
    lib = K.library()
    x = 0x10000
    assert lib.iqk_narrow_indices(x, -1, x, None) == 3
    assert lib.iqk_narrow_indices(None, 0, None, None) == 0
    assert lib.iqk_narrow_indices(None, 4, x, None) == 4
    assert lib.iqk_narrow_indices(x, 4, None, None) == 4
    assert lib.iqk_narrow_indices(x + 4, 4, x, None) == 5
    assert lib.iqk_narrow_indices(x, 4, x + 2, None) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("t", [7, 300])
def test_indices_beyond_32_bits_are_no_expert(cuda, t):
    codes, scales, w = make_matrix((5, 40, 96), seed=t)
    x = make_x((t, 1, 1, 96), torch.float32, seed=t)
    idx = torch.arange(2 * t).view(t, 2) % 5
    idx[:7, 1] = torch.tensor(BEYOND)
    ws = torch.empty(K.mx_workspace_bytes(2 * t, 5, 96, 40), dtype=torch.uint8, device="cuda")
    y = mx_switch_linear(x, idx.cuda(), codes, scales, workspace=ws)
    assert K.mx_read_error(ws) == K.DEVERR_EXPERT
    for got in (y, mx_switch_linear(x, idx.cuda(), codes, scales),
                mx_switch_linear(x, idx.t().contiguous().cuda().t(), codes, scales)):
        assert (got[:7, 1] == 0).all()
        check_routed(got, x, idx, w, torch.float32)


@pytest.mark.gpu
def test_layer_takes_indices_beyond_32_bits_for_no_expert(cuda):
    layer = MxSwitchGLU(4, 64, 32, device="cuda")
    g = torch.Generator().manual_seed(1)
    for name, shape in (("gate", (4, 32, 64)), ("up", (4, 32, 64)), ("down", (4, 64, 32))):
        layer.load_weights(name, torch.randn(shape, generator=g).cuda())
    x = torch.randn((7, 64), generator=g).cuda()
    idx = torch.zeros((7, 2), dtype=torch.int64)
    idx[:, 1] = torch.tensor(BEYOND)
    none = torch.where(idx > 0, -1, idx).clamp(min=-1)
    pairs = layer(x, idx.cuda())
    assert (pairs[:, 1] == 0).all() and torch.equal(pairs, layer(x, none.cuda()))
    ones = torch.ones((7, 2), device="cuda")
    assert torch.equal(layer(x, idx.cuda(), ones), layer(x, none.cuda(), ones))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [0, 1, 255, 1000, 148 * 8 * 256 * 2 + 5])
def test_narrowed_indices(cuda, count):
    g = torch.Generator().manual_seed(count)
    wide = torch.randint(-2 ** 62, 2 ** 62, (count,), generator=g) >> \
        torch.randint(0, 62, (count,), generator=g)
    got = K.expert_indices(wide.cuda())
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu().long(), wide.clamp(-2 ** 31, 2 ** 31 - 1))


# ------------------------------------------------------------- workspace sizes


def test_workspace_of_an_empty_call():
    """A call of no pairs has a workspace size, and it serves one."""
    lib = K.library()
    assert 0 < lib.iqk_mx_workspace_bytes(0, 4, 64, 64) <= lib.iqk_mx_workspace_bytes(1, 4, 64, 64)
    assert lib.iqk_mx_workspace_bytes(0, 1, 64, 64) > 0
    x = 0x10000
    assert lib.iqk_mx_routed(x, 0, 4, 64, x, 0, x, x, 16, 4, 64, 64, x, 0, x, 0, None) == 0


# --------------------------------------------------------- a layer that moves


def scale_buffers(layer):
    return [layer.gate_scales, layer.up_scales, layer.down_scales]


def aligned_rows(layer):
    return all(s.stride(-1) == 1 and s.stride(1) % 16 == 0 and s.stride(1) >= s.shape[2] and
               s.stride(0) == s.shape[1] * s.stride(1) for s in scale_buffers(layer))


def test_scale_rows_keep_their_boundaries_when_a_layer_moves(tmp_path):
    layer = MxSwitchGLU(2, 2880, 768)  # 90 and 24 scales a row, 96 and 32 bytes apart
    assert aligned_rows(layer) and layer.gate_scales.stride(1) == 96
    for scales in scale_buffers(layer):
        scales.copy_(torch.randint(100, 130, scales.shape, dtype=torch.uint8))
    want = [s.clone() for s in scale_buffers(layer)]

    def same(other):
        assert aligned_rows(other)
        for s, w in zip(scale_buffers(other), want):
            assert s.shape == w.shape and torch.equal(s, w)

    assert aligned_rows(copy.deepcopy(layer).to("meta"))
    moved = copy.deepcopy(layer).to("meta").to_empty(device="cpu")
    assert aligned_rows(moved)
    moved.load_state_dict(layer.state_dict())
    same(moved)
    packed = {k: v.contiguous().clone() for k, v in layer.state_dict().items()}
    for assign in (False, True):
        other = MxSwitchGLU(2, 2880, 768)
        other.load_state_dict(packed, assign=assign)
        same(other)
    parent = torch.nn.Sequential(copy.deepcopy(layer)).half().to(torch.bfloat16)
    same(parent[0])
    same(pickle.loads(pickle.dumps(layer)))
    torch.save(layer.state_dict(), tmp_path / "layer.pt")
    other = MxSwitchGLU(2, 2880, 768)
    other.load_state_dict(torch.load(tmp_path / "layer.pt"), assign=True)
    same(other)


@pytest.mark.gpu
def test_a_layer_made_on_the_host_serves_after_cuda(cuda):
    g = torch.Generator().manual_seed(4)
    there, here = MxSwitchGLU(3, 96, 160, device="cuda"), MxSwitchGLU(3, 96, 160)
    for name, shape in (("gate", (3, 160, 96)), ("up", (3, 160, 96)), ("down", (3, 96, 160))):
        there.load_weights(name, torch.randn(shape, generator=g).cuda())
        here.load(name, getattr(there, f"{name}_codes").cpu(), getattr(there, f"{name}_scales").cpu())
    x = torch.randn((5, 96), generator=g).cuda()
    idx = torch.tensor([[0, 2], [1, 0], [-1, 1], [2, 2], [1, 2]], device="cuda")
    scores = torch.rand((5, 2), generator=g).cuda()
    assert torch.equal(here.cuda()(x, idx, scores), there(x, idx, scores))


# ------------------------------------------------------- after an expired wait


def poison(tickets):
    """The state of the current stream's one-launch calls as a call leaves it whose
    wait ran out: the error word set, parts of shared items counted that never came."""
    stream = K.stream_handle(torch.device("cuda", torch.cuda.current_device()))
    state = K._FEW_STATES[torch.cuda.current_device(), stream]
    words = state[:8192].view(torch.int32)
    words[3] = K.DEVERR_TIMEOUT
    words[64:64 + 8 * 148] = tickets
    return words


@pytest.mark.gpu
@pytest.mark.parametrize("tickets", [1, 20, -1])
def test_one_launch_calls_recover_from_an_expired_wait(cuda, tickets):
    """Rows wide enough that CTAs join parts of an item behind the counters."""
    codes, scales, w = make_matrix((200, 16384), seed=1)
    x = make_x((3, 16384), torch.float32, seed=2)
    mats = make_matrix((5, 70, 8224), seed=3)
    rows = make_x((4, 1, 1, 8224), torch.float32, seed=4)
    idx = torch.tensor([[0, 4], [1, 0], [3, -1], [4, 4]])
    check(mx_linear(x, codes, scales), rounded(x), w, torch.float32)
    words = poison(tickets)
    for seed in range(5, 8):  # other inputs: the parts of the call before do not serve
        x = make_x((3, 16384), torch.float32, seed)
        rows = make_x((4, 1, 1, 8224), torch.float32, seed)
        check(mx_linear(x, codes, scales), rounded(x), w, torch.float32)
        check_routed(mx_switch_linear(rows, idx.cuda(), *mats[:2]), rows, idx, mats[2],
                     torch.float32)
    assert int(words[3]) == K.DEVERR_TIMEOUT  # until it is read
    words.zero_()
    check(mx_linear(x, codes, scales), rounded(x), w, torch.float32)


def test_error_entries_refuse_before_any_device_call():
    lib = K.library()
    assert lib.iqk_mx_take_errors(None, None) == 4
    assert lib.iqk_mx_error_word(None) == 4


@pytest.mark.gpu
def test_an_expired_wait_can_be_read_without_a_workspace(cuda):
    """A wait that nothing satisfies leaves its bit in the device's word, as one inside
    a product does; reading clears it and drops the states that it may have spoiled."""
    device = torch.device("cuda", torch.cuda.current_device())
    codes, scales, w = make_matrix((200, 16384), seed=1)
    x = make_x((3, 16384), torch.float32, seed=2)
    want = mx_linear(x, codes, scales)
    assert K.mx_take_errors(device) == 0
    assert torch.equal(mx_linear(x, codes, scales), want)  # the state was kept
    words, stream = poison(20), K.stream_handle(device)
    word = ctypes.c_void_p()
    assert K.library().iqk_mx_error_word(ctypes.byref(word)) == 0
    assert K.library().iqk_check_bounded_wait(1_000_000, word, stream) == 0
    assert K.mx_take_errors(device) == K.DEVERR_TIMEOUT
    assert K.mx_take_errors(torch.device("cuda")) == 0
    assert torch.equal(mx_linear(x, codes, scales), want)
    fresh = K._FEW_STATES[device.index, stream]
    assert fresh.data_ptr() != words.data_ptr() and int(fresh[:8192].view(torch.int32)[3]) == 0
    with pytest.raises(K.IqkRuntimeError):
        K.mx_take_errors(torch.device("cpu"))


# ---------------------------------------------------------- results that repeat


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,experts,width,out", [(1280, 4, 4, 16384, 64), (600, 2, 3, 16384, 300),
                                                   (700, 3, 5, 12320, 130), (45, 2, 2, 8224, 33)])
def test_wide_routed_calls_repeat_bit_for_bit(cuda, t, k, experts, width, out):
    """An expert has several tiles whose sums are cut at different columns. Blocks of
    sizes from 2^-20 to 2^20 make every f32 sum depend on where it is cut."""
    g = torch.Generator(device="cuda").manual_seed(t)
    codes, scales = mx_quantize(torch.randn((experts, out, width), generator=g, device="cuda"))
    size = torch.randint(-20, 21, (t, 1, 1, width // 32), generator=g, device="cuda")
    x = torch.randn((t, 1, 1, width), generator=g, device="cuda") * \
        torch.exp2(size.float()).repeat_interleave(32, -1)
    idx = torch.stack([torch.randperm(experts, generator=g, device="cuda")[:k]
                       for _ in range(t)]).int()
    idx[::7, 0] = -1
    idx[5, 0] = experts + 3
    y = mx_switch_linear(x, idx, codes, scales)
    for _ in range(12):
        assert torch.equal(mx_switch_linear(x, idx, codes, scales), y)
    # each pair against its own row through its own matrix, in 64 bits
    xq, w = mx_dequantize(*mx_quantize(x)).double().view(t, width), mx_dequantize(codes, scales)
    for e in range(experts):
        tt, jj = (idx == e).nonzero(as_tuple=True)
        want = xq[tt] @ w[e].double().t()
        room = xq[tt].abs() @ w[e].double().abs().t()
        err = (y[tt, jj, 0].double() - want).abs()
        assert (err <= (width / 64 + 8) * 2.0 ** -23 * room * (1 + 2.0 ** -24) +
                2.0 ** -24 * want.abs()).all()
    assert (y[(idx < 0) | (idx >= experts)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t,experts", [(33, 4096), (1030, 4096), (5000, 3), (257, 1)])
def test_wide_routed_sort(cuda, t, experts):
    """Counting in the pairs' order: many experts, few, stray indices, odd counts; the
    indices begin off 16-byte boundaries."""
    width = 8192
    codes = torch.randint(0, 256, (experts, 1, width // 2), dtype=torch.uint8, device="cuda")
    scales = torch.full((experts, 1, width // 32), 122, dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(t)
    flat = torch.randint(-2, experts + 2, (3 * t + 1,), generator=g).int().cuda()
    idx = flat[1:].view(t, 3)
    x = make_x((1, 1, 1, width), torch.bfloat16, seed=t)
    ws = torch.empty(K.mx_workspace_bytes(3 * t, experts, width, 1), dtype=torch.uint8,
                     device="cuda")
    y = mx_switch_linear(x, idx, codes, scales, torch.float32, workspace=ws)
    assert K.mx_read_error(ws) == (K.DEVERR_EXPERT if ((idx < -1) | (idx >= experts)).any() else 0)
    xq = mx_dequantize(*mx_quantize(x)).double().view(width)
    w = mx_dequantize(codes, scales).double().view(experts, width)
    want, room = w @ xq, w.abs() @ xq.abs()
    here = (idx >= 0) & (idx < experts)
    assert (y.view(t, 3)[~here] == 0).all()
    pick = idx[here].long()
    err = (y.view(t, 3)[here].double() - want[pick]).abs()
    assert (err <= (width / 64 + 8) * 2.0 ** -23 * room[pick] * 1.001).all()


# ------------------------------------------------------------------ memory held


@pytest.mark.parametrize("pairs,experts,width,out", [(128, 1, 4096, 512), (4096, 1, 4096, 8192),
                                                     (12288, 256, 4096, 2048), (70, 4, 7168, 64)])
def test_workspace_holds_what_the_call_uses(pairs, experts, width, out):
    """Codes and scales of the rows, four words a pair, tiles and counters: no parts of
    shared items for rows that are never shared (up to 7168 columns)."""
    need = K.mx_workspace_bytes(pairs, experts, width, out)
    rows = pairs * (width // 2 + (width // 32 + 15) // 16 * 16)
    tiles = 16 * (min(experts, pairs) + pairs // 16 + 1)
    assert need <= rows + 16 * pairs + tiles + (16 << 10)
    wide = K.mx_workspace_bytes(pairs, experts, 7200, out)
    assert wide > pairs * (3600 + 240) + 4 * 2 * 148 * 128 * 16


def test_state_of_one_launch_calls():
    lib = K.library()
    full = lib.iqk_mx_few_state_bytes()
    assert lib.iqk_mx_few_state_bytes_for(7168) == 256
    assert lib.iqk_mx_few_state_bytes_for(7200) == full > 8192
    x = 0x10000

    def few(width, state_bytes):
        return lib.iqk_mx_few(x, 0, 2, width, None, 2, x, x, 1024, 1, 64, width, x, 0, x,
                              state_bytes, None)

    assert few(7168, 255) == 6 and few(7200, full - 1) == 6 and few(7200, 256) == 6


@pytest.mark.gpu
@pytest.mark.parametrize("width,cleared", [(1024, 0), (8224, 1)])
def test_captured_one_launch_calls_allocate_and_clear_no_more_than_they_use(cuda, width, cleared):
    codes, scales, w = make_matrix((3, 64, width), seed=1)
    x = make_x((2, 1, 1, width), torch.bfloat16, seed=2)
    idx = torch.tensor([[0, 2], [1, 0]], dtype=torch.int32, device="cuda")

    def step():
        return mx_switch_linear(x, idx, codes, scales), mx_linear(x, codes[1], scales[1])

    step()
    seen = []

    class Ops(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            seen.append((func.overloadpacket.__name__,
                         out.numel() if isinstance(out, torch.Tensor) else 0))
            return out

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), Ops():
        y, z = step()
    names = [n for n, _ in seen]
    assert names.count("zero_") + names.count("fill_") == 2 * cleared
    if not cleared:
        assert all(n <= 1024 for name, n in seen if "empty" in name)
    x.copy_(make_x(x.shape, torch.bfloat16, seed=3))
    for _ in range(2):
        graph.replay()
        check_routed(y, x, idx.cpu(), w, torch.bfloat16)
        check(z.view(2, 64), rounded(x).reshape(2, width), w[1], torch.bfloat16)


# ------------------------------------- layouts, and more items than run at once


@pytest.mark.gpu
@pytest.mark.parametrize("t", [9, 40, 700])
def test_indices_off_16_byte_boundaries(cuda, t):
    codes, scales, w = make_matrix((6, 70, 96), seed=t)
    x = make_x((t, 1, 1, 96), torch.float32, seed=t)
    flat = torch.randint(-1, 6, (3 * t + 3,), generator=torch.Generator().manual_seed(t)).int()
    for start in (1, 2, 3):
        idx = flat.cuda()[start:start + 3 * t].view(t, 3)
        assert idx.is_contiguous() and idx.data_ptr() % 16
        check_routed(mx_switch_linear(x, idx, codes, scales), x, idx.cpu(), w, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 40, 300])
def test_products_of_one_row_seen_many_times(cuda, dtype, rows):
    codes, scales, w = make_matrix((3, 130, 544), seed=rows)
    one = make_x((1, 544), dtype, seed=rows)
    x = one.expand(rows, 544)
    assert x.stride(0) == 0
    y = mx_linear(x, codes[1], scales[1])
    check(y, rounded(x), w[1], dtype)
    idx = torch.arange(2 * rows).view(rows, 2) % 3
    many = x.view(rows, 1, 1, 544)
    check_routed(mx_switch_linear(many, idx.cuda(), codes, scales), many, idx, w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width", [(torch.bfloat16, 1013, 10016), (torch.float16, 997, 12000),
                                              (torch.float32, 1501, 4128)])
def test_streams_of_many_items(cuda, dtype, rows, width):
    """Each thread takes several items, at rows and columns that its step does not
    divide: the same codes, scales and values as in calls of a few rows."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, width), generator=g, device="cuda") * \
        torch.exp(torch.randn((rows, 1), generator=g, device="cuda"))
    x = x.to(dtype)
    codes, scales = mx_quantize(x)
    back = {out: mx_dequantize(codes, scales, out) for out in (torch.float32, torch.bfloat16)}
    for at in range(0, rows, 100):
        c, s = mx_quantize(x[at:at + 100])
        assert torch.equal(codes[at:at + 100], c) and torch.equal(scales[at:at + 100], s)
        for out, values in back.items():
            assert torch.equal(values[at:at + 100], mx_dequantize(c, s, out))


@pytest.mark.gpu
def test_streams_past_32_bit_items(cuda):
    """2^31 items and more: one row seen 8.4 million times, each the same codes."""
    width, rows = 4096, (1 << 31) // 256 + 3
    if torch.cuda.mem_get_info()[1] < 120 << 30:
        pytest.skip("90 GB of device memory")
    one = make_x((1, width), torch.bfloat16, seed=1)
    want_codes, want_scales = mx_quantize(one)
    codes, scales = mx_quantize(one.expand(rows, width))
    back = mx_dequantize(codes, scales, torch.bfloat16)
    want = mx_dequantize(want_codes, want_scales, torch.bfloat16)
    for at in range(0, rows, 1 << 20):
        cut = slice(at, at + (1 << 20))
        assert (codes[cut] == want_codes).all() and (scales[cut] == want_scales).all()
        assert (back[cut].view(torch.int16) == want.view(torch.int16)).all()
    del codes, scales, back
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,experts,width,out", [(1280, 4, 4, 4096, 64), (600, 2, 3, 7168, 300),
                                                   (3000, 3, 5, 2080, 130)])
def test_routed_calls_repeat_bit_for_bit(cuda, t, k, experts, width, out):
    """Which of an expert's tiles a pair is in may differ from call to call, and changes
    no result: every item of such widths is summed whole."""
    g = torch.Generator(device="cuda").manual_seed(t)
    codes, scales = mx_quantize(torch.randn((experts, out, width), generator=g, device="cuda"))
    size = torch.randint(-20, 21, (t, 1, 1, width // 32), generator=g, device="cuda")
    x = torch.randn((t, 1, 1, width), generator=g, device="cuda") * \
        torch.exp2(size.float()).repeat_interleave(32, -1)
    idx = torch.stack([torch.randperm(experts, generator=g, device="cuda")[:k]
                       for _ in range(t)]).int()
    y = mx_switch_linear(x, idx, codes, scales)
    for _ in range(12):
        assert torch.equal(mx_switch_linear(x, idx, codes, scales), y)


@pytest.mark.gpu
def test_matrices_without_outputs(cuda):
    """No rows have no layout to refuse, whatever strides the empty tensor has."""
    codes, scales, _ = make_matrix((3, 32, 64), seed=2)
    x = make_x((2, 1, 1, 64), torch.float32, seed=1)
    idx = torch.tensor([[0, 2], [2, -1]], device="cuda")
    for c, s in ((codes[:, :0], scales[:, :0]),
                 (codes[:, :0].contiguous(), scales[:, :0].contiguous())):
        assert mx_switch_linear(x, idx, c, s).shape == (2, 2, 1, 0)
        assert mx_dequantize(c, s).shape == (3, 0, 64)


@pytest.mark.gpu
def test_error_word_of_calls_without_a_product(cuda):
    """Calls that launch no product leave an error word all the same, of their own
    indices and not of what the workspace held."""
    x = make_x((2, 1, 1, 64), torch.float32, seed=1)
    codes, scales, _ = make_matrix((3, 32, 64), seed=2)
    stray = torch.tensor([[0, 7], [2, -1]], dtype=torch.int32, device="cuda")
    none = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    cases = [(x[:0], stray[:0], codes, scales, 0), (x, stray, codes[:, :0], scales[:, :0], 1),
             (x, stray.clamp(max=2), codes[:, :0], scales[:, :0], 0),
             (x, stray, codes[:0], scales[:0], 1), (x, none, codes[:0], scales[:0], 0)]
    for rows, idx, c, s, want in cases:
        ws = torch.full((K.mx_workspace_bytes(4, 3, 64, 32),), 255, dtype=torch.uint8,
                        device="cuda")
        y = mx_switch_linear(rows, idx, c, s, workspace=ws)
        assert y.shape == (*idx.shape, 1, c.shape[1]) and (y == 0).all()
        assert K.mx_read_error(ws) == want * K.DEVERR_EXPERT
    with pytest.raises(K.IqkRuntimeError, match="workspace"):
        mx_switch_linear(x[:0], none[:0], codes, scales,
                         workspace=torch.empty(1 << 20, dtype=torch.uint8))
