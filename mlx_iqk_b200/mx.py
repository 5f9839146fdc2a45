"""MXFP4: microscaled 4-bit floating point, quantisation and products.

The OCP Microscaling format beside the IQ_K members: 32 consecutive values of
a row share one power-of-two scale (E8M0, a byte), each value a 4-bit E2M1
code. A matrix ``[..., rows, width]`` is two tensors that the caller holds, as
the dense members' streams are:

- ``codes  uint8 [..., rows, width / 2]``, two codes a byte, the even column in
  the low nibble, contiguous;
- ``scales uint8 [..., rows, width / 32]``, each row on a 16-byte boundary
  (:func:`mx_quantize` returns it as a view of such rows;
  :func:`mx_aligned_scales` makes one of packed scales, once, at load time).

Functions:

- :func:`mx_quantize`, :func:`mx_dequantize`  to the format and back;
- :func:`mx_linear`         ``q(x) W^T`` through one matrix;
- :func:`mx_switch_linear`  the same through the experts that a router picked,
  on the seam of ``IqkSwitchLinear`` (``src/mlx_iqk/nn.py:105-333``);
- :class:`MxSwitchGLU`      one SwitchGLU layer of MXFP4 experts.

Activations are quantised inside the product, so that both operands are 4-bit
on the tensor cores; products and sums are float32, rounded once to
``out_dtype`` (the activations' type unless given). These are serving
operators: they carry no gradient and refuse an input that asks for one.

Every wait inside the products is bounded. One that expires leaves the call's
output incomplete and ``DEVERR_TIMEOUT`` for ``kernels.mx_take_errors(device)``.
"""

from __future__ import annotations

import torch
from torch import nn

from . import kernels as K
from .kernels import IqkKernelError, IqkRuntimeError

MX_BLOCK = 32


def _check_no_gradient(t, what):
    if t.requires_grad and torch.is_grad_enabled():
        raise IqkRuntimeError(f"the MXFP4 operators carry no gradient: detach {what}")
    K.refuse_tangent(t, what)


def _rows(x, what="x"):
    """``(x, rows, row_stride)`` of float rows whose columns are adjacent: ``x``
    itself, or a copy where its layout is not one of evenly spaced rows."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise IqkRuntimeError(f"{what} must be a tensor on the GPU")
    if x.dtype not in K.DTYPE_IDS:
        raise IqkRuntimeError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    _check_no_gradient(x, what)
    width = x.shape[-1] if x.dim() else 0
    if width <= 0 or width % MX_BLOCK:
        raise IqkKernelError(
            f"{what} must have a width that is a positive multiple of {MX_BLOCK}, "
            f"got shape {tuple(x.shape)}")
    K.check_current(x.device)
    count = x.numel() // width
    if x.is_contiguous():
        return x, count, width
    rows = x.reshape(-1, width)
    step, inner = rows.stride()
    if inner != 1 or (count > 1 and 0 != step < width):
        return rows.contiguous(), count, width
    return rows, count, step


def _matrix(codes, scales, dims, x=None):
    """The byte stride of a matrix's scale rows; refuses what the kernels do not take."""
    try:
        shape, steps = scales.shape, scales.stride()
        if codes.dtype is scales.dtype is torch.uint8 and len(shape) == dims \
                and codes.get_device() == scales.get_device() >= 0 \
                and (x is None or x.get_device() == codes.get_device()) \
                and codes.is_contiguous() \
                and codes.shape == shape[:-1] + (shape[-1] * (MX_BLOCK // 2),) \
                and steps[-1] == 1 and shape[-2] > 1 and steps[-2] >= shape[-1] > 0 \
                and (dims == 2 or steps[0] == steps[1] * shape[1]) \
                and not (steps[-2] | codes.data_ptr() | scales.data_ptr()) % 16:
            return steps[-2]
    except (AttributeError, IndexError):
        pass
    return _check_matrix(codes, scales, dims, None if x is None else x.device)


def _check_matrix(codes, scales, dims, device):
    """Every check of :func:`_matrix` with its message, and the layouts off its fast path."""
    for t, name in ((codes, "codes"), (scales, "scales")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise IqkRuntimeError(f"{name} must be a tensor on the GPU")
        if t.dtype != torch.uint8:
            raise IqkRuntimeError(f"{name} must be uint8, got {t.dtype}")
    if codes.device != scales.device or (device is not None and codes.device != device):
        raise IqkRuntimeError("codes, scales and activations must be on one device")
    shape, lead = codes.shape, scales.shape
    if not shape or (dims and len(shape) != dims):
        raise IqkRuntimeError(f"codes must have {dims or 'at least 1'} axes, got {len(shape)}")
    blocks = lead[-1] if lead else 0
    if lead[:-1] != shape[:-1] or shape[-1] != blocks * MX_BLOCK // 2 or blocks == 0:
        raise IqkRuntimeError(
            f"codes {tuple(shape)} and scales {tuple(lead)} do not belong "
            f"together: {MX_BLOCK // 2} code bytes to a scale")
    if not codes.is_contiguous() or codes.data_ptr() % 16:
        raise IqkRuntimeError("codes must be contiguous and 16-byte aligned")
    steps = scales.stride()
    stride, step, packed = (blocks + 15) // 16 * 16, None, blocks == 1 or steps[-1] == 1
    for axis in range(len(lead) - 2, -1, -1):  # one row or none: any stride
        if lead[axis] == 1 or scales.numel() == 0:
            continue
        if step is None:
            stride = step = steps[axis]
        packed = packed and steps[axis] == step
        step *= lead[axis]
    if not packed or stride % 16 or stride < blocks or scales.data_ptr() % 16:
        raise IqkRuntimeError(
            "scale rows must be evenly spaced and start on 16-byte boundaries "
            "(mx_aligned_scales lays packed scales out so)")
    return stride


def mx_aligned_scales(scales: torch.Tensor) -> torch.Tensor:
    """A copy of ``scales [..., rows, blocks]`` whose rows start on 16-byte boundaries."""
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.uint8 or scales.dim() < 1:
        raise IqkRuntimeError("scales must be a uint8 tensor")
    out = _scale_rows(scales.shape[:-1], scales.shape[-1], scales)
    out.copy_(scales)
    return out


def _scale_rows(lead, blocks, like) -> torch.Tensor:
    pitch = (blocks + 15) // 16 * 16
    t = like.new_empty((*lead, pitch), dtype=torch.uint8)
    return t if pitch == blocks else t.narrow(-1, 0, blocks)


def mx_quantize(x):
    """``(codes, scales)`` of ``x [..., width]`` (float32, float16 or bfloat16).

    Each block's scale is ``2^(floor(log2 m) - 2)``, ``m`` its largest magnitude
    (``2^-127`` at least); values round to the nearest code, ties to the even
    one, and hold at 6 beyond it. A block with a NaN or an infinity gets scale
    byte 255: all of it reads NaN."""
    rows, count, step = _rows(x)
    *lead, width = x.shape
    codes = x.new_empty((*lead, width // 2), dtype=torch.uint8)
    scales = _scale_rows(lead, width // MX_BLOCK, x)
    K.mx_quantize(rows, count, step, codes, scales, (width // MX_BLOCK + 15) // 16 * 16)
    return codes, scales


def mx_dequantize(codes, scales, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values ``[..., width]`` of an MXFP4 tensor: exact in float32, rounded once
    to float16 or bfloat16."""
    two = isinstance(codes, torch.Tensor) and codes.dim() == 2
    stride = _matrix(codes, scales, 2) if two else _check_matrix(codes, scales, 0, None)
    if dtype not in K.DTYPE_IDS:
        raise IqkRuntimeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    K.check_current(codes.device)
    *lead, half = codes.shape
    out = codes.new_empty((*lead, half * 2), dtype=dtype)
    K.mx_dequantize(codes, scales, stride, out)
    return out


def _out_dtype(x, out_dtype):
    dtype = x.dtype if out_dtype is None else out_dtype
    if dtype not in K.DTYPE_IDS:
        raise IqkRuntimeError(f"out_dtype must be float32, float16 or bfloat16, got {dtype}")
    return dtype


def mx_linear(x, codes, scales, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``q(x) W^T`` ``[..., out]`` for ``x [..., width]`` and ``W`` = ``codes [out,
    width / 2]``, ``scales [out, width / 32]``; ``q`` is :func:`mx_quantize`."""
    rows, count, step = _rows(x)
    stride = _matrix(codes, scales, 2, x)
    out, half = codes.shape
    *lead, width = x.shape
    if half * 2 != width:
        raise IqkRuntimeError(f"x of width {width} meets a matrix of {half * 2}")
    y = x.new_empty((*lead, out), dtype=_out_dtype(x, out_dtype))
    if count and out:
        K.mx_linear(rows, count, step, codes, scales, stride, y)
    return y


def mx_switch_linear(x, indices, codes, scales, out_dtype: torch.dtype | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``q(x) W_e^T`` through the experts that ``indices [..., top_k]`` names:
    ``[..., top_k, 1, out]``.

    ``x`` is ``[..., 1, 1, width]`` (one row per token, shared by its experts) or
    ``[..., top_k, 1, width]`` (one row per pair); the matrices are ``codes
    [experts, out, width / 2]`` and ``scales [experts, out, width / 32]``. Each
    picked expert's matrix is read once for all its pairs. Index -1 (a token
    that the router left out) gives a zero row. So does an index beyond the
    experts, which also sets ``DEVERR_EXPERT`` in a caller's ``workspace``
    (uint8, ``kernels.mx_workspace_bytes``), read by
    ``kernels.mx_read_error``."""
    rows, count, step = _rows(x)
    stride = _matrix(codes, scales, 3, x)
    if not isinstance(indices, torch.Tensor) or indices.device != x.device \
            or indices.dtype not in (torch.int32, torch.int64):
        raise IqkRuntimeError("indices must be an int32 or int64 tensor beside x")
    experts, out, half = codes.shape
    if half * 2 != x.shape[-1]:
        raise IqkRuntimeError(f"x of width {x.shape[-1]} meets matrices of {half * 2}")
    sel = K.expert_indices(indices)
    pairs = sel.numel()
    if pairs and (count == 0 or pairs % count):
        raise IqkRuntimeError(
            f"{pairs} token-expert pairs do not tile {count} activation "
            f"row(s); the operand and the routing disagree")
    y = x.new_empty((*indices.shape, 1, out), dtype=_out_dtype(x, out_dtype))
    if pairs and out and experts:
        K.mx_routed(rows, count, step, sel, codes, scales, stride, y, workspace)
        return y
    if workspace is not None:  # no product to leave the error word
        K.mx_set_error(workspace, y.device, ((sel < -1) | (sel >= experts)).any())
    return y.zero_()


class MxSwitchGLU(nn.Module):
    """One SwitchGLU layer of MXFP4 experts, ``(x, indices, scores)`` as
    ``IqkSwitchGLU``: gate and up ``[experts, inter, hidden]``, down ``[experts,
    hidden, inter]``, ``h = silu(gate) * up * score`` in float32, and each
    token's sum over its experts. The scores go in before the down projection's
    quantisation of ``h``, whose scales they move with it (a power of two
    exactly, another factor up to the rounding of a 4-bit value)."""

    def __init__(self, num_experts: int, hidden: int, inter: int, device=None):
        super().__init__()
        for what, value in (("hidden", hidden), ("inter", inter)):
            if value <= 0 or value % MX_BLOCK:
                raise IqkKernelError(f"{what} {value} is not a positive multiple of {MX_BLOCK}")
        if not 0 < num_experts <= 4096:
            raise IqkRuntimeError(f"num_experts {num_experts} is not in 1 to 4096")
        self.num_experts, self.hidden, self.inter = num_experts, hidden, inter
        for name, (rows, width) in self._shapes().items():
            codes = torch.zeros((num_experts, rows, width // 2), dtype=torch.uint8, device=device)
            self.register_buffer(f"{name}_codes", codes)
            self.register_buffer(f"{name}_scales", _scale_rows(
                (num_experts, rows), width // MX_BLOCK, codes).zero_())

    def _shapes(self):
        return {"gate": (self.inter, self.hidden), "up": (self.inter, self.hidden),
                "down": (self.hidden, self.inter)}

    def _lay_out_scales(self) -> None:
        """Scale rows back on 16-byte boundaries: a copy of a buffer that is a view of
        wider rows is packed."""
        for name in self._shapes():
            scales = self._buffers[f"{name}_scales"]
            experts, rows, _ = scales.shape
            outer, step, inner = scales.stride()
            if inner != 1 or step % 16 or outer != rows * step \
                    or scales.storage_offset() % 16:
                self._buffers[f"{name}_scales"] = mx_aligned_scales(scales)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._lay_out_scales()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._lay_out_scales()

    def load(self, name: str, codes: torch.Tensor, scales: torch.Tensor) -> None:
        """Install one projection's matrices (``gate``, ``up`` or ``down``)."""
        if name not in self._shapes():
            raise IqkRuntimeError(f"projection must be gate, up or down, got {name!r}")
        into = getattr(self, f"{name}_codes"), getattr(self, f"{name}_scales")
        for new, old, what in zip((codes, scales), into, ("codes", "scales")):
            if tuple(new.shape) != tuple(old.shape) or new.dtype != torch.uint8:
                raise IqkRuntimeError(f"{name} {what} must be uint8 {tuple(old.shape)}, got "
                                      f"{new.dtype} {tuple(new.shape)}")
        into[0].copy_(codes)
        into[1].copy_(scales)

    def load_weights(self, name: str, weights: torch.Tensor) -> None:
        """Quantise and install one projection's float matrices ``[experts, rows, width]``."""
        self.load(name, *mx_quantize(weights))

    def forward(self, x, indices, scores=None) -> torch.Tensor:
        """``x [..., hidden]``, ``indices`` and ``scores [..., top_k]`` ->
        ``[..., hidden]`` float32; with ``scores`` None each pair's own output,
        ``[..., top_k, hidden]``. Index -1 contributes nothing. Scores that ask
        for a gradient are refused: to train a router, leave them out and weight
        the pairs' outputs."""
        lead, k = tuple(indices.shape[:-1]), indices.shape[-1]
        if scores is not None:
            if not isinstance(scores, torch.Tensor) or scores.device != x.device:
                raise IqkRuntimeError("scores must be a tensor beside x")
            _check_no_gradient(scores, "scores")
        if tuple(x.shape) != lead + (self.hidden,) or \
                (scores is not None and scores.shape != indices.shape):
            raise IqkRuntimeError(
                f"x {tuple(x.shape)}, indices {tuple(indices.shape)} and scores "
                f"{None if scores is None else tuple(scores.shape)} do not belong together")
        sel = K.expert_indices(indices.reshape(-1, k))
        rows = x.reshape(-1, 1, 1, self.hidden)
        f32 = torch.float32
        if not sel.numel():
            shape = lead + ((self.hidden,) if scores is not None else (k, self.hidden))
            return torch.zeros(shape, dtype=f32, device=x.device)
        gate = mx_switch_linear(rows, sel, self.gate_codes, self.gate_scales, f32)
        up = mx_switch_linear(rows, sel, self.up_codes, self.up_scales, f32)
        w = None if scores is None else scores.reshape(-1).to(f32).contiguous()
        h = torch.empty((sel.numel(), self.inter), dtype=f32, device=x.device)
        K.swiglu_rows(gate.view(-1, self.inter), up.view(-1, self.inter), w, h)
        y = mx_switch_linear(h.view(-1, k, 1, self.inter), sel, self.down_codes,
                             self.down_scales, f32)
        if scores is None:
            return y.view(lead + (k, self.hidden))
        out = torch.empty((rows.shape[0], self.hidden), dtype=f32, device=x.device)
        K.pairs_combine(y, sel, k, self.num_experts, out)
        return out.view(lead + (self.hidden,))


__all__ = ["MX_BLOCK", "MxSwitchGLU", "mx_aligned_scales", "mx_dequantize", "mx_linear",
           "mx_quantize", "mx_switch_linear"]
