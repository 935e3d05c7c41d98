"""What the operators around the fused experts are timed on: the norm that feeds a layer's products, the block-scaled FP8
product of dense layers, the SwiGLU between two of them and the router, from one decoded token to a prefill chunk."""
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "alpha-moe_amd")
_DEV = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_FP8_MAX = 448.0
_FLOOR = 1e-10
_EPS = 1e-6


def listed():
    return [
        # one user's decode step: the norm in front of an expert layer, which the router reads in bf16 too
        {"name": "norm_1", "op": "norm", "M": 1, "K": 7168, "dtype": "bf16", "residual": True, "keep_norm": True},
        # the first norm of a model on a ragged batch: no residual yet, activations still in fp32
        {"name": "norm_333_fp32", "op": "norm", "M": 333, "K": 2048, "dtype": "fp32", "residual": False, "keep_norm": False},
        # a prefill chunk
        {"name": "norm_8192", "op": "norm", "M": 8192, "K": 7168, "dtype": "bf16", "residual": True, "keep_norm": False},
        # one user's decode step through a dense layer's wide product
        {"name": "mm_1", "op": "mm", "M": 1, "N": 4096, "K": 7168},
        # an odd decode batch through a product whose rows end inside a block of weight scales
        {"name": "mm_61", "op": "mm", "M": 61, "N": 2112, "K": 7168},
        # the largest decode batches, back to the hidden size
        {"name": "mm_256", "op": "mm", "M": 256, "N": 7168, "K": 2048},
        # a prefill chunk
        {"name": "mm_8192", "op": "mm", "M": 8192, "N": 4096, "K": 7168},
        # an odd decode batch between the two products of a dense layer
        {"name": "swiglu_7", "op": "swiglu", "M": 7, "I": 768, "dtype": "bf16"},
        # a prefill chunk
        {"name": "swiglu_8192", "op": "swiglu", "M": 8192, "I": 2048, "dtype": "bf16"},
        # one token routed with a selection bias, limited to the best groups, and the fused shared expert behind the routed ones
        {"name": "route_1", "op": "route", "M": 1, "E": 256, "top_k": 8, "dtype": "fp32", "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalize": True, "shared": 1},
        # a ragged batch over many small experts, logits straight from a bf16 product: equal logits are common
        {"name": "route_1021_bf16", "op": "route", "M": 1021, "E": 512, "top_k": 10, "dtype": "bf16", "scoring": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "renormalize": True, "shared": 0},
        # a prefill chunk
        {"name": "route_8192", "op": "route", "M": 8192, "E": 256, "top_k": 8, "dtype": "fp32", "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renormalize": True, "shared": 1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "mm", "mm", "swiglu", "route"])
    M = _log_int(rng, 1, 8192)
    if op == "norm":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        K = 128 * rng.randint(1, 56 if dtype == "bf16" else 28)
        return {"op": op, "M": M, "K": K, "dtype": dtype, "residual": rng.random() < 0.75, "keep_norm": rng.random() < 0.4}
    if op == "mm":
        K = 128 * rng.randint(1, 56)
        N = _log_int(rng, 64, 8192)
        if rng.random() < 0.5:
            N = (N + 127) // 128 * 128
        return {"op": op, "M": min(M, 8192 * 4096 // N), "N": N, "K": K}
    if op == "swiglu":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        return {"op": op, "M": M, "I": 128 * rng.randint(1, 16 if dtype == "bf16" else 8), "dtype": dtype}
    E = rng.choice([8, 60, 64, 128, 160, 256])
    groups = rng.choice([1, 4]) if E < 256 else rng.choice([1, 8])
    top_groups = groups if groups == 1 else groups // 2
    scoring = rng.choice(["softmax", "sigmoid"])
    return {"op": op, "M": M, "E": E, "top_k": rng.randint(1, min(10, top_groups * (E // groups))),
            "dtype": rng.choice(["fp32", "bf16"]), "scoring": scoring, "bias": scoring == "sigmoid" and rng.random() < 0.7,
            "groups": groups, "top_groups": top_groups, "renormalize": rng.random() < 0.8, "shared": rng.choice([0, 1])}


def _activations(gen, M, K):
    """Rows of different sizes with a few loud channels, as hidden states are."""
    x = torch.randn((M, K), generator=gen, device=_DEV) * (0.5 + torch.rand((M, 1), generator=gen, device=_DEV))
    loud = torch.randint(0, K, (max(1, K // 512),), generator=gen, device=_DEV)
    x[:, loud] *= 8.0
    return x


def _quant_rows(y):
    """(codes, scales) of [M, K] fp32 in groups of 128 columns."""
    M, K = y.shape
    g = y.reshape(M, K // 128, 128)
    scale = g.abs().amax(-1, keepdim=True).clamp_min(_FLOOR) / _FP8_MAX
    q = (g / scale).clamp(-_FP8_MAX, _FP8_MAX).to(torch.float8_e4m3fn)
    return q.reshape(M, K), scale.reshape(M, K // 128)


def _quant_blocks(w):
    """(codes, scales) of [N, K] fp32 in blocks of 128 x 128; the last row of blocks may be short."""
    N, K = w.shape
    rows = (N + 127) // 128
    b = torch.nn.functional.pad(w, (0, 0, 0, rows * 128 - N)).reshape(rows, 128, K // 128, 128)
    scale = b.abs().amax((1, 3), keepdim=True).clamp_min(_FLOOR) / _FP8_MAX
    q = (b / scale).to(torch.float8_e4m3fn).reshape(rows * 128, K)[:N].contiguous()
    return q, scale.reshape(rows, K // 128).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    M, st = case["M"], {"case": case}
    if case["op"] == "norm":
        K, dtype = case["K"], _TYPES[case["dtype"]]
        st["x"] = _activations(gen, M, K).to(dtype)
        st["residual"] = (4.0 * _activations(gen, M, K)).to(dtype) if case["residual"] else None
        st["weight"] = (1.0 + 0.2 * torch.randn((K,), generator=gen, device=_DEV)).to(dtype)
    elif case["op"] == "mm":
        N, K = case["N"], case["K"]
        st["x"], st["x_scale"] = _quant_rows(_activations(gen, M, K))
        st["w"], st["w_scale"] = _quant_blocks(0.02 * torch.randn((N, K), generator=gen, device=_DEV))
    elif case["op"] == "swiglu":
        st["x"] = (1.5 * _activations(gen, M, 2 * case["I"])).to(_TYPES[case["dtype"]])
    else:
        # tokens agree on some experts more than on others
        mean = 0.5 * torch.randn((1, case["E"]), generator=gen, device=_DEV)
        st["logits"] = (mean + torch.randn((M, case["E"]), generator=gen, device=_DEV)).to(_TYPES[case["dtype"]])
        st["bias"] = 0.1 * torch.randn((case["E"],), generator=gen, device=_DEV) if case["bias"] else None
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------
def _plain_norm(st):
    case, x = st["case"], st["x"]
    h = x.float()
    if st["residual"] is not None:
        h = h + st["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS) * st["weight"].float()
    q, scale = _quant_rows(y)
    return {"q": q, "scale": scale, "residual": h.to(x.dtype) if case["residual"] else None,
            "norm": y.to(x.dtype) if case["keep_norm"] else None}


def _plain_mm(st):
    N, K = st["w"].shape
    x = (st["x"].float().reshape(-1, K // 128, 128) * st["x_scale"][:, :, None]).reshape(-1, K)
    scale = st["w_scale"].repeat_interleave(128, 0)[:N]
    w = (st["w"].float().reshape(N, K // 128, 128) * scale[:, :, None]).reshape(N, K)
    return (x @ w.t()).to(torch.bfloat16)


def _plain_swiglu(st):
    gate, up = st["x"].float().chunk(2, -1)
    q, scale = _quant_rows(gate / (1.0 + torch.exp(-gate)) * up)
    return {"q": q, "scale": scale}


def _plain_route(st):
    # the order of the experts is decided in 64 bits: sigmoid(logit) + bias of two experts may be nearer than 32 bits tell
    case, logits = st["case"], st["logits"].double()
    M, E = logits.shape
    if case["scoring"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-logits))
    choice = logits if st["bias"] is None else score + st["bias"].double()
    if case["groups"] > 1:
        parts = choice.reshape(M, case["groups"], -1)
        best = torch.sort(parts, dim=-1, descending=True)[0]
        value = best[..., 0] if st["bias"] is None else best[..., :2].sum(-1)
        stay = torch.sort(value, dim=-1, descending=True, stable=True)[1][:, :case["top_groups"]]
        gone = torch.ones_like(value, dtype=torch.bool).scatter_(1, stay, False)
        choice = parts.masked_fill(gone[..., None], -float("inf")).reshape(M, E)
    ids = torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :case["top_k"]]
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    if case["shared"]:
        more = torch.arange(E, E + case["shared"], device=ids.device).expand(M, -1)
        ids = torch.cat([ids, more], 1)
        weights = torch.cat([weights, torch.full_like(more, 0.4, dtype=weights.dtype)], 1)
    return {"weights": weights.float(), "ids": ids.to(torch.int32)}


# ---- the framework's operators -----------------------------------------------------------------------------
def _own(st):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from alpha_moe_python import layer_hip
    case = st["case"]
    if case["op"] == "norm":
        return layer_hip.rms_norm_quant_fp8(st["x"], st["weight"], _EPS, residual=st["residual"],
                                            keep_norm=case["keep_norm"])._asdict()
    if case["op"] == "mm":
        return layer_hip.block_scaled_mm(st["x"], st["x_scale"], st["w"], st["w_scale"])
    if case["op"] == "swiglu":
        q, scale = layer_hip.swiglu_quant_fp8(st["x"])
        return {"q": q, "scale": scale}
    weights, ids = layer_hip.route_topk(st["logits"], case["top_k"], scoring=case["scoring"], bias=st["bias"],
                                        num_groups=case["groups"], top_groups=case["top_groups"],
                                        renormalize=case["renormalize"], shared_experts=case["shared"], shared_weight=0.4)
    return {"weights": weights, "ids": ids}


_PLAIN = {"norm": _plain_norm, "mm": _plain_mm, "swiglu": _plain_swiglu, "route": _plain_route}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------
def _exact_groups(y):
    """What the codes stand for before their rounding, in units of the scale, and the scales."""
    M, K = y.shape
    amax = torch.linalg.vector_norm(y.view(M, K // 128, 128), ord=float("inf"), dim=2)
    scale = torch.maximum(amax, torch.full_like(amax, 1e-10)) / 448
    return y / torch.repeat_interleave(scale, 128, 1), scale


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        h = st["x"].to(torch.float64)
        if case["residual"]:
            h += st["residual"]
        length = torch.sqrt((h * h).sum(1) / case["K"] + 1e-6)
        y = st["weight"].to(torch.float64) * (h / length[:, None])
        q, scale = _exact_groups(y)
        return {"q": q, "scale": scale, "residual": h if case["residual"] else None, "norm": y if case["keep_norm"] else None}
    if case["op"] == "mm":
        # one block of the contraction after the other, its scales on its sums
        N, K = st["w"].shape
        out = torch.zeros((case["M"], N), dtype=torch.float64, device=_DEV)
        block_of = torch.arange(N, device=_DEV) // 128
        for kb in range(K // 128):
            cols = slice(128 * kb, 128 * kb + 128)
            part = torch.mm(st["x"][:, cols].to(torch.float64), st["w"][:, cols].to(torch.float64).t())
            out += part * torch.outer(st["x_scale"][:, kb].double(), st["w_scale"][block_of, kb].double())
        return out
    if case["op"] == "swiglu":
        x = st["x"].to(torch.float64)
        I = case["I"]
        q, scale = _exact_groups(x[:, :I] * (0.5 + 0.5 * torch.tanh(0.5 * x[:, :I])) * x[:, I:])
        return {"q": q, "scale": scale}
    l = st["logits"].to(torch.float64)
    M, E = l.shape
    if case["scoring"] == "softmax":
        score = torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    else:
        score = 0.5 + 0.5 * torch.tanh(0.5 * l)
    choice = l if st["bias"] is None else score + st["bias"]
    allowed = torch.ones((M, E), dtype=torch.bool, device=_DEV)
    if case["groups"] > 1:
        size = E // case["groups"]
        value = torch.stack([c.topk(1 if st["bias"] is None else min(2, size), dim=1)[0].sum(1)
                             for c in choice.split(size, 1)], 1)
        # a group stays when fewer than top_groups are ahead of it; of equal ones the first is ahead
        at = torch.arange(case["groups"], device=_DEV)
        ahead = (value[:, None, :] > value[:, :, None]) | ((value[:, None, :] == value[:, :, None]) & (at[None, :] < at[:, None]))
        allowed = torch.repeat_interleave(ahead.sum(2) < case["top_groups"], size, 1)
    left = torch.where(allowed, choice, torch.full_like(choice, -float("inf")))
    ids, place = [], torch.arange(E, device=_DEV).expand(M, E)
    for _ in range(case["top_k"]):
        best = left.max(1, keepdim=True)[0]
        pick = torch.where(left == best, place, torch.full_like(place, E)).min(1, keepdim=True)[0]
        ids.append(pick)
        left = left.scatter(1, pick, -float("inf"))
    ids = torch.cat(ids, 1)
    weights = torch.gather(score, 1, ids)
    if case["renormalize"]:
        weights /= weights.sum(1, keepdim=True)
    weights = torch.cat([weights, torch.full((M, case["shared"]), 0.4, dtype=torch.float64, device=_DEV)], 1)
    more = torch.arange(E, E + case["shared"], device=_DEV).expand(M, -1)
    return {"weights": weights, "ids": torch.cat([ids, more], 1).to(torch.int32)}


def work(case):
    M = case["M"]
    if case["op"] == "norm":
        size, n = 2 if case["dtype"] == "bf16" else 4, M * case["K"]
        moved = n * size * (1 + 2 * case["residual"] + case["keep_norm"]) + n + 4 * n // 128 + size * case["K"]
        return {"bytes": moved, "flops": 8 * n}
    if case["op"] == "mm":
        N, K = case["N"], case["K"]
        scales = 4 * (K // 128) * (M + (N + 127) // 128)
        return {"bytes": M * K + N * K + scales + 2 * M * N, "flops": 2.0 * M * N * K}
    if case["op"] == "swiglu":
        n = M * case["I"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4) + n + 4 * n // 128, "flops": 8 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    kept = case["top_k"] + case["shared"]
    return {"bytes": M * (case["E"] * size + 8 * kept) + (4 * case["E"] if case["bias"] else 0), "flops": 16.0 * M * case["E"]}
