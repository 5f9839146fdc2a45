"""Workloads of the expert-routing and microscaled 4-bit (MXFP4) operators.

Five operators that a mixture-of-experts layer runs next to its experts:

* ``route``     top-k expert choice of each token with its router weights;
* ``train``     the same choice with the per-expert counts and the balance loss,
                forward and backward (the router's step in training);
* ``quantize``  a matrix to MXFP4 (32 consecutive E2M1 values share one E8M0
                power of two) and back to the values that the codes stand for;
* ``linear``    ``y = q(x) W^T`` for an MXFP4 matrix ``W``, ``q`` the MXFP4
                quantisation of the activations;
* ``switch``    the same product through the experts that a router picked.

``run`` computes each either in plain torch operations in 32 bits (``own``
false) or through the package's entry points (``own`` true). ``exact`` is the
definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32  # values under one scale


# ------------------------------------------------------------------- the cases


def listed():
    return [
        # one token of a decode step through the router of a 256-expert layer
        {"name": "route-decode-1", "op": "route", "tokens": 1, "experts": 256, "top_k": 6,
         "dtype": "f32", "scoring": "softmax", "renormalize": True, "masked": False},
        # the router of a prefill of 2048 tokens, some of them padding
        {"name": "route-prefill-2048", "op": "route", "tokens": 2048, "experts": 256, "top_k": 6,
         "dtype": "bf16", "scoring": "softmax", "renormalize": True, "masked": True},
        # a training step's router: packed sequences of ragged lengths, padding at random places
        {"name": "train-16384", "op": "train", "tokens": 16384, "experts": 256, "top_k": 6,
         "dtype": "bf16", "scoring": "softmax", "renormalize": True, "masked": True,
         "segments": 8},
        # a small layer with sigmoid scores that are not normalised; odd sizes
        {"name": "train-sigmoid-1021", "op": "train", "tokens": 1021, "experts": 60, "top_k": 4,
         "dtype": "f32", "scoring": "sigmoid", "renormalize": False, "masked": False,
         "segments": 1},
        # the activations of a 2048-token prefill
        {"name": "quantize-2048x4096", "op": "quantize", "rows": 2048, "width": 4096,
         "dtype": "bf16"},
        # a small odd matrix in f32
        {"name": "quantize-77x1056", "op": "quantize", "rows": 77, "width": 1056, "dtype": "f32"},
        # one decode token through a vocabulary head
        {"name": "linear-head-1", "op": "linear", "tokens": 1, "width": 4096, "out": 129280,
         "dtype": "bf16"},
        # a few rows of a small projection with odd sizes, f32 in and out
        {"name": "linear-37x1056x1000", "op": "linear", "tokens": 37, "width": 1056, "out": 1000,
         "dtype": "f32"},
        # a prefill through a dense projection
        {"name": "linear-4096x4096x8192", "op": "linear", "tokens": 4096, "width": 4096,
         "out": 8192, "dtype": "bf16"},
        # one decode token through the gate projection of its six experts
        {"name": "switch-decode-1", "op": "switch", "tokens": 1, "experts": 256, "top_k": 6,
         "width": 4096, "out": 2048, "paired": False, "masked": False, "dtype": "bf16"},
        # eight decode tokens through the down projection: one activation row per pair
        {"name": "switch-down-8", "op": "switch", "tokens": 8, "experts": 256, "top_k": 6,
         "width": 2048, "out": 4096, "paired": True, "masked": False, "dtype": "bf16"},
        # a 2048-token prefill through the gate projection, some of the tokens padding
        {"name": "switch-prefill-2048", "op": "switch", "tokens": 2048, "experts": 256,
         "top_k": 6, "width": 4096, "out": 2048, "paired": False, "masked": True,
         "dtype": "bf16"},
    ]


def draw(rng):
    def log_size(low, high):
        size = max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))
        return size - 1 if size in (3072, 3072 // BLOCK) else size  # 3072: in no case

    op = rng.choice(["route", "train", "quantize", "linear", "switch"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("route", "train"):
        experts = log_size(8, 512)
        case = {"op": op, "tokens": log_size(1, 8192) if op == "route" else log_size(16, 16384),
                "experts": experts, "top_k": rng.randint(1, 8), "dtype": dtype,
                "scoring": rng.choice(["softmax", "sigmoid"]),
                "renormalize": rng.random() < 0.6, "masked": rng.random() < 0.5}
        if op == "train":
            case["segments"] = rng.randint(1, 16)
            case["tokens"] = min(case["tokens"], 16384 * 256 // experts)
        return case
    if op == "quantize":
        return {"op": op, "rows": log_size(1, 4096), "width": BLOCK * log_size(1, 256),
                "dtype": dtype}
    if op == "linear":
        width, out = BLOCK * log_size(8, 256), log_size(16, 8192)
        most = 4096 * 4096 * 8192 // (width * out)
        return {"op": op, "tokens": log_size(1, min(4096, most)), "width": width, "out": out,
                "dtype": dtype}
    width, out = BLOCK * log_size(8, 128), log_size(16, 4096)
    experts = log_size(4, min(256, 256 * 4096 * 2048 // (width * out)))
    return {"op": op, "tokens": log_size(1, 2048), "experts": experts,
            "top_k": rng.randint(1, min(6, experts)), "width": width, "out": out,
            "paired": rng.random() < 0.4, "masked": rng.random() < 0.4, "dtype": dtype}


def work(case):
    op = case["op"]
    if op in ("route", "train"):
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        item = DTYPES[case["dtype"]].itemsize
        masks = t if case["masked"] else 0
        if op == "route":
            return {"bytes": t * e * item + t * k * 8 + masks, "flops": 4.0 * t * e}
        # logits in, their gradient out, choice and weights out, the weights' gradient in
        return {"bytes": 2 * t * e * item + t * k * 12 + masks + case["segments"] * e * 4,
                "flops": 12.0 * t * e}
    if op == "quantize":
        n = case["rows"] * case["width"]
        # the matrix in, the values that its codes stand for out (f32)
        return {"bytes": n * (DTYPES[case["dtype"]].itemsize + 4), "flops": 4.0 * n}
    item = DTYPES[case["dtype"]].itemsize
    k, n = case["width"], case["out"]
    matrix = n * (k // 2 + k // BLOCK)
    if op == "linear":
        t = case["tokens"]
        return {"bytes": t * k * item + matrix + t * n * item, "flops": 2.0 * t * k * n}
    t, e, top = case["tokens"], case["experts"], case["top_k"]
    pairs = t * top
    read = e * (1 - (1 - top / e) ** t)  # experts that some token picked
    return {"bytes": (pairs if case["paired"] else t) * k * item + read * matrix +
            pairs * (n * item + 4), "flops": 2.0 * pairs * k * n}


# ------------------------------------------------------------------ the inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    state = {"case": case}
    if op in ("route", "train"):
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        # some experts are liked more than others, as in a router half way through training
        liking = 0.5 * torch.randn(e, generator=g, device="cuda")
        state["logits"] = (torch.randn((t, e), generator=g, device="cuda") + liking).to(dtype)
        state["mask"] = None
        if case["masked"]:
            state["mask"] = torch.rand(t, generator=g, device="cuda") < 0.9
        if op == "train":
            cuts = torch.randint(0, t + 1, (case["segments"] - 1,), generator=g, device="cuda")
            ends = torch.tensor([0, t], device="cuda")
            state["offsets"] = torch.cat([ends, cuts]).sort().values.to(torch.int32)
            state["grad_weights"] = torch.randn((t, min(k, e)), generator=g, device="cuda") / t
            state["grad_loss"] = torch.full((), 0.01, device="cuda")
        return state
    if op == "quantize":
        state["x"] = _activations(case["rows"], case["width"], g).to(dtype)
        return state
    width, out = case["width"], case["out"]
    if op == "linear":
        state["x"] = _activations(case["tokens"], width, g).to(dtype)
        state["codes"], state["scales"] = _matrices(1, out, width, g)
        state["codes"], state["scales"] = state["codes"][0], state["scales"][0]
        return state
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    rows = t * k if case["paired"] else t
    state["x"] = _activations(rows, width, g).to(dtype).reshape(t, -1, 1, width)
    state["codes"], state["scales"] = _matrices(e, out, width, g)
    liking = 0.5 * torch.randn(e, generator=g, device="cuda")
    picked = (torch.randn((t, e), generator=g, device="cuda") + liking).topk(k).indices
    if case["masked"]:  # padding tokens have no expert: index -1
        pad = torch.rand(t, generator=g, device="cuda") >= 0.9
        picked = torch.where(pad[:, None], -1, picked)
    state["indices"] = picked.to(torch.int32)
    return state


def _activations(rows, width, g):
    """Normal activations whose channels differ in size, as a model's do."""
    channel = torch.exp(0.7 * torch.randn(width, generator=g, device="cuda"))
    return torch.randn((rows, width), generator=g, device="cuda") * channel


def _matrices(experts, out, width, g):
    """MXFP4 weights ``codes [experts, out, width / 2]`` (low nibble first) and
    ``scales [experts, out, width / 32]``. Rows of scales start on 16-byte
    boundaries, so ``scales`` may be a view of a wider buffer."""
    blocks = width // BLOCK
    pitch = (blocks + 15) // 16 * 16
    codes = torch.empty((experts, out, width // 2), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((experts, out, pitch), dtype=torch.uint8, device="cuda")
    rows = codes.view(experts * out, width // 2)
    row_scales = scales.view(experts * out, pitch)
    step = max(1, (1 << 27) // width)
    for at in range(0, experts * out, step):
        count = min(step, experts * out - at)
        w = 0.02 * torch.randn((count, blocks, BLOCK), generator=g, device="cuda")
        exponent = _shared_exponent(w.abs().amax(-1))
        size = _nearest_code(w.abs() / _power_of_two(exponent)[..., None])
        code = (size + 8 * (w < 0)).to(torch.uint8).view(count, width // 2, 2)
        rows[at:at + count] = code[..., 0] | (code[..., 1] << 4)
        row_scales[at:at + count, :blocks] = (exponent + 127).to(torch.uint8)
    return codes, scales[..., :blocks]


def _shared_exponent(amax):
    """floor(log2(amax)) - 2, at least -127: the largest value lands in [4, 8)."""
    return (torch.frexp(amax).exponent - 3).clamp(min=-127).where(amax > 0, -127)


def _power_of_two(exponent):
    return torch.exp2(exponent.double()).float()


def _nearest_code(size):
    """E2M1 code (0..7) of a magnitude: nearest, ties to the even code."""
    return ((size > 0.25).int() + (size >= 0.75) + (size > 1.25) + (size >= 1.75) +
            (size > 2.5) + (size >= 3.5) + (size > 5.0))


# --------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    return {"route": _route, "train": _train, "quantize": _quantize, "linear": _linear,
            "switch": _switch}[op](state)


def _route(state):
    case = state["case"]
    if own:
        from mlx_iqk_b200 import router
        return router.route(state["logits"], min(case["top_k"], case["experts"]),
                            scoring=case["scoring"], renormalize=case["renormalize"],
                            scale=2.5, mask=state["mask"])
    return _plain_choice(state["logits"].float(), case, state["mask"])


def _train(state):
    case = state["case"]
    logits = state["logits"].detach().requires_grad_()
    if own:
        from mlx_iqk_b200 import router
        indices, weights, loss, counts = router.route_balanced(
            logits, min(case["top_k"], case["experts"]), scoring=case["scoring"],
            renormalize=case["renormalize"], scale=2.5, mask=state["mask"],
            offsets=state["offsets"])
    else:
        z = logits.float()
        indices, weights = _plain_choice(z, case, state["mask"])
        loss, counts = _plain_balance(z, indices, case, state["mask"], state["offsets"])
    grad, = torch.autograd.grad([weights, loss], [logits],
                                [state["grad_weights"], state["grad_loss"]])
    return indices, weights.detach(), loss.detach(), counts, grad


def _quantize(state):
    if own:
        from mlx_iqk_b200 import mx
        return mx.mx_dequantize(*mx.mx_quantize(state["x"]), dtype=torch.float32)
    return _plain_rounded(state["x"])


def _linear(state):
    x = state["x"]
    if own:
        from mlx_iqk_b200 import mx
        return mx.mx_linear(x, state["codes"], state["scales"])
    w = _plain_values(state["codes"], state["scales"])
    return torch.matmul(_plain_rounded(x), w.t()).to(x.dtype)


def _switch(state):
    x, indices = state["x"], state["indices"]
    if own:
        from mlx_iqk_b200 import mx
        return mx.mx_switch_linear(x, indices, state["codes"], state["scales"])
    t, k = indices.shape
    rows = _plain_rounded(x).expand(t, k, 1, x.shape[-1]).reshape(t * k, -1)
    pick = indices.reshape(-1).long()
    codes, scales = state["codes"], state["scales"]
    here = pick >= 0
    if t * k <= 64:  # a matrix per pair
        w = _plain_values(codes[pick.clamp(min=0)], scales[pick.clamp(min=0)])
        y = torch.matmul(w, rows[..., None])[..., 0] * here[:, None]
    else:  # the pairs of each expert, in a table as long as the longest list
        e = codes.shape[0]
        order = torch.sort(pick, stable=True).indices
        owner = pick[order]
        counts = (pick[None, :] == torch.arange(e, device=pick.device)[:, None]).sum(1)
        first = counts.cumsum(0) - counts + (~here).sum()
        place = torch.arange(t * k, device=pick.device) - first[owner.clamp(min=0)]
        keep = owner >= 0
        owner, place, order = owner[keep], place[keep], order[keep]
        table = rows.new_zeros((e, max(1, int(counts.max())), rows.shape[1]))
        table[owner, place] = rows[order]
        y = rows.new_zeros((t * k, codes.shape[1]))
        y[order] = torch.matmul(table, _plain_values(codes, scales).transpose(1, 2))[owner, place]
    return y.to(x.dtype).reshape(t, k, 1, -1)


def _plain_choice(z, case, mask):
    """The top_k largest logits of each row (ties: the lowest index) and their
    weights; rows that the mask leaves out choose -1 with weight 0."""
    k = min(case["top_k"], case["experts"])
    if mask is not None:
        z = torch.where(mask[:, None], z, -math.inf)
    top, indices = (a[:, :k] for a in torch.sort(z, dim=-1, descending=True, stable=True))
    here = top > -math.inf
    indices = torch.where(here, indices, -1).to(torch.int32)
    if case["renormalize"]:
        score = top if case["scoring"] == "softmax" else torch.nn.functional.logsigmoid(top)
        weights = torch.exp(score - score.detach().amax(-1, keepdim=True).clamp(min=-1e30))
        weights = weights / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    elif case["scoring"] == "softmax":
        peak = top[:, :1].detach().clamp(min=-1e30)
        weights = torch.exp(top - peak) / torch.exp(z - peak).sum(-1, keepdim=True).clamp(min=1e-30)
    else:
        weights = torch.sigmoid(top)
    return indices, 2.5 * torch.where(here, weights, 0.0)


def _plain_balance(z, indices, case, mask, offsets):
    """Per segment: expert e's share f_e of the choices (1 when balanced) times
    its mean score P_e, summed; the mean over segments that hold a token."""
    t, e, k = z.shape[0], case["experts"], indices.shape[1]
    there = torch.ones(t, dtype=torch.bool, device=z.device) if mask is None else mask
    place = torch.arange(t, device=z.device)
    member = ((place >= offsets[:-1, None]) & (place < offsets[1:, None]) & there).float()
    chosen = (indices[..., None] == torch.arange(e, device=z.device)).sum(1).float()
    counts = torch.matmul(member, chosen)
    tokens = member.sum(1, keepdim=True)
    if case["scoring"] == "softmax":
        score = torch.softmax(z, -1)
    else:
        score = torch.sigmoid(z)
        score = score / score.sum(-1, keepdim=True)
    share = counts * e / (k * tokens).clamp(min=1.0)
    mean = torch.matmul(member, score) / tokens.clamp(min=1.0)
    loss = (share * mean).sum() / (tokens > 0).sum().clamp(min=1)
    return loss, counts.to(torch.int32)


def _plain_rounded(x):
    """Each 32 values of a row to MXFP4 and back, in f32."""
    v = x.float().reshape(*x.shape[:-1], -1, BLOCK)
    scale = _power_of_two(_shared_exponent(v.abs().amax(-1, keepdim=True)))
    size = (v / scale).abs()
    near = torch.where(size < 2, torch.round(size * 2) / 2,
                       torch.where(size < 4, torch.round(size), torch.round(size / 2) * 2))
    return (torch.copysign(near.clamp(max=6), v) * scale).reshape(x.shape)


def _plain_values(codes, scales):
    """The f32 values of MXFP4 codes."""
    sizes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([sizes, -sizes])
    pairs = torch.stack([table.repeat(16), table.repeat_interleave(16)], -1)
    values = pairs[codes.int()].reshape(*scales.shape, BLOCK)
    return (values * _power_of_two(scales.int() - 127)[..., None]).reshape(*codes.shape[:-1], -1)


# ------------------------------------------------------- the definition, 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_choice(state["logits"].double(), case, state["mask"])[:2]
    if op == "train":
        return _exact_train(state)
    if op == "quantize":
        return _exact_rounded(state["x"])
    if op == "linear":
        return _exact_rounded(state["x"]) @ _exact_values(state["codes"], state["scales"]).T
    x, indices = state["x"], state["indices"]
    t, k = indices.shape
    rows = _exact_rounded(x).reshape(t, -1, x.shape[-1])
    y = torch.zeros((t, k, 1, case["out"]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, slot = (indices == e).nonzero(as_tuple=True)
        if token.numel():
            w = _exact_values(state["codes"][e], state["scales"][e])
            y[token, slot, 0] = rows[token, slot if case["paired"] else 0] @ w.T
    return y


def _exact_choice(z, case, mask):
    t, e = z.shape
    k = min(case["top_k"], e)
    there = torch.ones(t, dtype=torch.bool, device=z.device) if mask is None else mask
    left = torch.where(there[:, None], z, -math.inf)
    indices = torch.full((t, k), -1, dtype=torch.int32, device=z.device)
    chosen = torch.full((t, k), -math.inf, dtype=torch.float64, device=z.device)
    for j in range(k):  # argmax of what is left; among equals the first
        best = left.amax(1)
        place = (left == best[:, None]).int().argmax(1)
        some = best > -math.inf
        indices[:, j] = torch.where(some, place, -1).int()
        chosen[:, j] = best
        left[torch.arange(t), place] = -math.inf
    some = indices >= 0
    if case["scoring"] == "softmax":
        score = torch.exp(z - z.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-z))
    weights = score.gather(1, indices.clamp(min=0).long()) * some
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True).where(some[:, :1], 1.0)
    return indices, 2.5 * weights, score, some


def _exact_train(state):
    case, mask, offsets = state["case"], state["mask"], state["offsets"].tolist()
    z = state["logits"].double()
    indices, weights, score, some = _exact_choice(z, case, mask)
    t, e = z.shape
    k = indices.shape[1]
    there = torch.ones(t, dtype=torch.bool, device=z.device) if mask is None else mask
    # the balance loss: its value, and a_te = dloss / d(normalised score)
    total = score.sum(1, keepdim=True)
    normal = score / total
    counts = torch.zeros((len(offsets) - 1, e), dtype=torch.int32, device=z.device)
    losses, slope = [], torch.zeros_like(z)
    for s, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        n = int(there[a:b].sum())
        if not n:
            continue
        picked = indices[a:b][there[a:b]]
        counts[s] = torch.bincount(picked[picked >= 0].long(), minlength=e).int()
        share = counts[s].double() * e / (k * n)
        losses.append((share * normal[a:b][there[a:b]].mean(0)).sum())
        slope[a:b] = share / n
    loss = torch.stack(losses).mean() if losses else torch.zeros((), dtype=torch.float64)
    slope = slope * there[:, None] * state["grad_loss"].double() / max(1, len(losses))
    # through the scores: softmax d s_e = s_e (dz_e - sum s dz), normalised sigmoid the
    # same with dz scaled by 1 - sigmoid
    fall = torch.ones_like(z) if case["scoring"] == "softmax" else 1 - score
    grad = normal * fall * (slope - (normal * slope).sum(1, keepdim=True))
    up = 2.5 * state["grad_weights"].double() * some
    at = indices.clamp(min=0).long()
    q = weights / 2.5
    if case["renormalize"]:
        part = q * (up - (q * up).sum(1, keepdim=True)) * fall.gather(1, at)
    elif case["scoring"] == "softmax":
        part = q * up
        grad = grad - score * part.sum(1, keepdim=True)
    else:
        part = q * (1 - q) * up
    grad = grad.scatter_add(1, at, part * some)
    return indices, weights, loss, counts, grad * there[:, None]


def _exact_rounded(x):
    v = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    # floor(log2) is the exponent field of a double; every f32 but 0 is a normal one
    exponent = ((amax.view(torch.int64) >> 52) - 1023).clamp(min=-125) - 2
    scale = _exact_power(exponent)
    sizes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (sizes[_nearest_code(v.abs() / scale).long()] * torch.sign(v) * scale).reshape(x.shape)


def _exact_values(codes, scales):
    sizes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    value = sizes[(code & 7).long()] * (1 - 2 * (code >> 3).double())
    scale = _exact_power(scales.long() - 127)
    return value * scale.repeat_interleave(BLOCK, -1)


def _exact_power(exponent):
    return ((exponent + 1023) << 52).view(torch.float64)
