"""What the operators that bring tokens to different weights are timed on: tokens sorted by expert and back, with their gradients, the
block-scaled FP8 product of sorted tokens with their experts' weights, and the low-rank adapters of many requests beside a shared
projection, from one decoded token to a prefill chunk."""
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "alpha-moe_amd")
_DEV = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp32": 4, "fp8": 1}
_FP8_MAX = 448.0
_FLOOR = 1e-10
_MOST_ROWS = 65536                       # of sorted tokens
_MOST_BYTES = 65536 * 7168               # of their values
_MOST_PRODUCT = 65536 * 1536 * 2048      # multiply-adds of one product
_MOST_ADAPTED = 8192 * 24 * 64 * (2048 + 7168)   # of all adapters on all tokens


def listed():
    return [
        # one user's decode step: the quantised token goes to its experts and the shared one
        {"name": "sort_1_fp8", "op": "sort", "M": 1, "K": 7168, "E": 257, "top_k": 9, "dtype": "fp8", "train": False, "padding": 0},
        # a training step on a ragged batch over many small experts: rows there, gradients back
        {"name": "sort_1021_train", "op": "sort", "M": 1021, "K": 2048, "E": 512, "top_k": 10, "dtype": "bf16", "train": True,
         "padding": 0},
        # a prefill chunk
        {"name": "sort_8192_fp8", "op": "sort", "M": 8192, "K": 7168, "E": 256, "top_k": 8, "dtype": "fp8", "train": False,
         "padding": 0},
        # an odd decode batch back from its experts
        {"name": "combine_61", "op": "combine", "M": 61, "K": 7168, "E": 257, "top_k": 9, "dtype": "bf16", "train": False,
         "padding": 0},
        # a batch that is padded to a captured size, in fp32
        {"name": "combine_333_fp32", "op": "combine", "M": 333, "K": 2048, "E": 128, "top_k": 8, "dtype": "fp32", "train": False,
         "padding": 45},
        # a training step: the weighted sums, and the gradients of the experts' results and of the router's weights
        {"name": "combine_4096_train", "op": "combine", "M": 4096, "K": 2048, "E": 128, "top_k": 8, "dtype": "bf16", "train": True,
         "padding": 0},
        # one user's decode step: eight experts, one row each
        {"name": "grouped_1", "op": "grouped", "M": 1, "E": 256, "top_k": 8, "N": 512, "K": 7168, "padding": 0},
        # an odd decode batch: nearly every expert has a row or two
        {"name": "grouped_61", "op": "grouped", "M": 61, "E": 256, "top_k": 8, "N": 512, "K": 7168, "padding": 0},
        # a prefill chunk through the wide products of its experts
        {"name": "grouped_8192", "op": "grouped", "M": 8192, "E": 128, "top_k": 8, "N": 1536, "K": 2048, "padding": 0},
        # one user with an adapter
        {"name": "adapters_1", "op": "adapters", "M": 1, "N": 4096, "K": 7168, "rank": 16, "adapters": 8, "requests": 1, "fp8": False},
        # an odd decode batch, an adapter for most requests, on the codes that the projection reads
        {"name": "adapters_61_fp8", "op": "adapters", "M": 61, "N": 2112, "K": 7168, "rank": 32, "adapters": 48, "requests": 61,
         "fp8": True},
        # a prefill chunk of many prompts
        {"name": "adapters_8192", "op": "adapters", "M": 8192, "N": 7168, "K": 2048, "rank": 64, "adapters": 24, "requests": 37,
         "fp8": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["sort", "combine", "grouped", "adapters"])
    M = _log_int(rng, 1, 8192)
    if op == "adapters":
        K, N = 128 * rng.randint(1, 56), _log_int(rng, 64, 8192)
        M = min(M, 8192 * 7168 // N)
        rank, requests = rng.choice([8, 16, 24, 32, 64, 128]), _log_int(rng, 1, min(M, 128))
        adapters = max(1, min(_log_int(rng, 1, 64), _MOST_ADAPTED // (M * rank * (N + K))))
        return {"op": op, "M": M, "N": N, "K": K, "rank": rank, "adapters": adapters, "requests": requests, "fp8": rng.random() < 0.4}
    E = rng.choice([8, 60, 64, 128, 160, 256, 512])
    top_k = rng.randint(1, min(10, E))
    M = min(M, _MOST_ROWS // top_k)
    padding = rng.randint(0, M // 4) if rng.random() < 0.3 else 0
    if op == "grouped":
        K, N = 128 * rng.randint(1, 56 if E <= 256 else 16), _log_int(rng, 64, 2112)
        return {"op": op, "M": max(1, min(M, _MOST_PRODUCT // (top_k * N * K))), "E": E, "top_k": top_k, "N": N, "K": K, "padding": 0}
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp8"] if op == "sort" else ["bf16", "bf16", "fp32"])
    # what is no code may have any number of columns
    K = 128 * rng.randint(1, 56) if dtype == "fp8" or rng.random() < 0.6 else _log_int(rng, 7, 7168)
    train = dtype != "fp8" and rng.random() < 0.5
    M = max(1, min(M, _MOST_BYTES // (top_k * K * _SIZES[dtype] * (2 if train else 1))))
    return {"op": op, "M": M, "K": K, "E": E, "top_k": top_k, "dtype": dtype, "train": train, "padding": min(padding, M - 1)}


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
    """(codes, scales) of [E, N, K] in blocks of 128 x 128; the last row of blocks of each may be short."""
    E, N, K = w.shape
    rows = (N + 127) // 128
    b = torch.nn.functional.pad(w, (0, 0, 0, rows * 128 - N)).reshape(E, rows, 128, K // 128, 128)
    scale = b.abs().amax((2, 4), keepdim=True).clamp_min(_FLOOR) / _FP8_MAX
    q = (b / scale).to(torch.float8_e4m3fn).reshape(E, rows * 128, K)[:, :N].contiguous()
    return q, scale.reshape(E, rows, K // 128).contiguous()


def _routing(gen, case):
    """Experts of the tokens, some more popular than others; the last tokens of a padded batch have none."""
    M, E = case["M"], case["E"]
    liking = 0.5 * torch.randn((1, E), generator=gen, device=_DEV) + torch.randn((M, E), generator=gen, device=_DEV)
    values, ids = torch.topk(liking, case["top_k"], dim=1)
    weights = torch.softmax(values, 1)
    if case["E"] % 2 == 1:               # the shared expert is the last one, and everybody's
        ids[:, -1] = E - 1
        ids[:, :-1] %= E - 1
    ids = ids.to(torch.int32)
    if case["padding"]:
        ids[M - case["padding"]:] = -1
    return ids.contiguous(), weights.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    M, K, st = case["M"], case["K"], {"case": case}
    if case["op"] == "adapters":
        N, L, rank, requests = case["N"], case["adapters"], case["rank"], case["requests"]
        x = _activations(gen, M, K)
        st["x"], st["x_scale"] = _quant_rows(x) if case["fp8"] else (x.to(torch.bfloat16), None)
        st["base"] = torch.randn((M, N), generator=gen, device=_DEV).to(torch.bfloat16)
        st["a"] = (torch.randn((L, rank, K), generator=gen, device=_DEV) / K ** 0.5).to(torch.bfloat16)
        st["b"] = (torch.randn((L, N, rank), generator=gen, device=_DEV) * 0.1).to(torch.bfloat16)
        st["scale"] = 0.5 + 1.5 * torch.rand((L,), generator=gen, device=_DEV)
        # requests one behind the other, of different lengths; about one in eight has no adapter
        of_request = torch.randint(0, L, (requests,), generator=gen, device=_DEV)
        if requests > 1:
            of_request[torch.rand((requests,), generator=gen, device=_DEV) < 0.125] = -1
        ends = torch.sort(torch.randperm(M - 1, generator=gen, device=_DEV)[:requests - 1] + 1)[0]
        which = torch.searchsorted(ends, torch.arange(M, device=_DEV), right=True)
        st["ids"] = of_request[which].to(torch.int32)
        return st
    ids, weights = _routing(gen, case)
    if case["op"] == "sort":
        x = _activations(gen, M, K)
        st["ids"] = ids
        if case["dtype"] == "fp8":
            st["x"], st["x_scale"] = _quant_rows(x)
        else:
            st["x"], st["x_scale"] = x.to(_TYPES[case["dtype"]]), None
        if case["train"]:
            st["x"].requires_grad_()
            st["grad"] = torch.randn((M * case["top_k"], K), generator=gen, device=_DEV).to(st["x"].dtype)
        return st
    order, row_of_slot, offsets = _order(ids, case["E"])
    if case["op"] == "combine":
        dtype = _TYPES[case["dtype"]]
        st["rows"] = _activations(gen, M * case["top_k"], K).to(dtype)
        st["row_of_slot"], st["weights"] = row_of_slot, weights
        if case["train"]:
            st["rows"].requires_grad_()
            st["weights"].requires_grad_()
            st["grad"] = torch.randn((M, K), generator=gen, device=_DEV).to(dtype)
        return st
    q, scale = _quant_rows(_activations(gen, M, K))
    token = order // case["top_k"]
    st["x"], st["x_scale"], st["offsets"] = q[token], scale[token], offsets
    st["w"], st["w_scale"] = _quant_blocks(0.02 * torch.randn((case["E"], case["N"], K), generator=gen, device=_DEV))
    st["most"] = int((offsets[1:] - offsets[:-1]).max())     # a batch's largest expert (the plain form's batches are that long)
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------
def _order(ids, E):
    """(slots in the order of their rows, row of each slot, first row of each expert): slots by ascending expert, a slot's row negative
    (~row) where the slot has no expert; those are behind the others."""
    expert = ids.flatten().long()
    expert = torch.where((expert >= 0) & (expert < E), expert, E)
    order = torch.sort(expert, stable=True)[1]
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=order.device)
    row = torch.where(expert < E, row, ~row)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).index_add_(0, expert, torch.ones_like(expert))
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts[:E], 0)])
    return order, row.to(torch.int32).reshape(ids.shape), offsets.to(torch.int32)


def _plain_sort(st):
    case = st["case"]
    x, ids = st["x"].detach(), st["ids"]
    order, row_of_slot, offsets = _order(ids, case["E"])
    token = order // case["top_k"]
    live = (torch.arange(order.numel(), device=order.device) < offsets[-1])[:, None]
    if case["dtype"] == "fp8":           # (bytes of 0 are codes of 0)
        rows = (x.view(torch.uint8)[token] * live).view(torch.float8_e4m3fn)
    else:
        rows = x[token] * live
    out = {"rows": rows, "scale": None, "offsets": offsets, "row_of_slot": row_of_slot, "grad_x": None}
    if st["x_scale"] is not None:
        out["scale"] = st["x_scale"][token] * live
    if case["train"]:
        parts = st["grad"][row_of_slot.clamp_min(0).long()].float() * (row_of_slot >= 0)[..., None]
        out["grad_x"] = parts.sum(1).to(x.dtype)
    return out


def _plain_combine(st):
    rows, at, weights = st["rows"].detach(), st["row_of_slot"], st["weights"].detach()
    live = at >= 0
    w = torch.where(live, weights, 0.0)
    picked = rows[at.clamp_min(0).long()].float() * live[..., None]
    out = {"out": (picked * w[..., None]).sum(1).to(rows.dtype), "grad_rows": None, "grad_weights": None}
    if st["case"]["train"]:
        g = st["grad"].float()
        out["grad_weights"] = (picked * g[:, None]).sum(-1)
        grad = torch.empty_like(rows)
        grad[torch.where(live, at, ~at).flatten().long()] = (g[:, None] * w[..., None]).to(rows.dtype).flatten(0, 1)
        out["grad_rows"] = grad
    return out


def _plain_grouped(st):
    # every expert's rows padded to the largest expert's number, one product of batches
    E, N, K = st["w"].shape
    most, offsets = st["most"], st["offsets"].long()
    x = (st["x"].float().reshape(-1, K // 128, 128) * st["x_scale"][:, :, None]).reshape(-1, K)
    scale = st["w_scale"].repeat_interleave(128, 1)[:, :N]
    w = (st["w"].float().reshape(E, N, K // 128, 128) * scale[..., None]).reshape(E, N, K)
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    live = expert < E
    place = torch.where(live, expert * most + row - offsets[expert.clamp_max(E)], E * most)
    batches = x.new_zeros((E * most + 1, K)).index_copy_(0, place, x)[:-1].reshape(E, most, K)
    out = torch.bmm(batches, w.transpose(1, 2).contiguous()).reshape(E * most, N)
    return (out[place.clamp_max(E * most - 1)] * live[:, None]).to(torch.bfloat16)


def _plain_adapters(st):
    # all adapters on all tokens, and of a token's results those of its own
    x, ids = st["x"].float(), st["ids"].long()
    M, K = x.shape
    L, N, rank = st["b"].shape
    if st["x_scale"] is not None:
        x = (x.reshape(M, K // 128, 128) * st["x_scale"][:, :, None]).reshape(M, K)
    mine = (ids[:, None] == torch.arange(L, device=ids.device)) * st["scale"]
    v = (x @ st["a"].float().reshape(L * rank, K).t()).reshape(M, L, rank) * mine[..., None]
    b = st["b"].float().transpose(1, 2).reshape(L * rank, N)
    return (st["base"].float() + v.reshape(M, L * rank) @ b).to(torch.bfloat16)


# ---- the framework's operators -----------------------------------------------------------------------------
def _own(st):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from alpha_moe_python import layer_hip
    case = st["case"]
    if case["op"] == "sort":
        s = layer_hip.sort_tokens(st["x"], st["ids"], case["E"], x_scale=st["x_scale"])
        grad = torch.autograd.grad(s.rows, st["x"], st["grad"])[0] if case["train"] else None
        return {"rows": s.rows, "scale": s.scale, "offsets": s.offsets, "row_of_slot": s.row_of_slot, "grad_x": grad}
    if case["op"] == "combine":
        out = layer_hip.combine_tokens(st["rows"], st["row_of_slot"], st["weights"])
        if not case["train"]:
            return {"out": out, "grad_rows": None, "grad_weights": None}
        grad_rows, grad_weights = torch.autograd.grad(out, (st["rows"], st["weights"]), st["grad"])
        return {"out": out, "grad_rows": grad_rows, "grad_weights": grad_weights}
    if case["op"] == "grouped":
        return layer_hip.grouped_block_scaled_mm(st["x"], st["x_scale"], st["offsets"], st["w"], st["w_scale"])
    return layer_hip.add_adapters(st["base"], st["x"], st["a"], st["b"], st["ids"], scale=st["scale"], x_scale=st["x_scale"])


_PLAIN = {"sort": _plain_sort, "combine": _plain_combine, "grouped": _plain_grouped, "adapters": _plain_adapters}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "adapters":
        x = st["x"].to(torch.float64)
        if st["x_scale"] is not None:
            x = x * torch.repeat_interleave(st["x_scale"].double(), 128, 1)
        out = st["base"].to(torch.float64)
        for one in range(case["adapters"]):
            rows = torch.nonzero(st["ids"] == one).flatten()
            inner = torch.mm(x[rows], st["a"][one].double().t())
            out[rows] += torch.mm(inner, st["b"][one].double().t()) * st["scale"][one].double()
        return out
    if case["op"] == "grouped":
        out = torch.zeros((st["x"].shape[0], case["N"]), dtype=torch.float64, device=_DEV)
        bounds = st["offsets"].tolist()
        block_of = torch.arange(case["N"], device=_DEV) // 128
        x = st["x"].double() * torch.repeat_interleave(st["x_scale"].double(), 128, 1)
        for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            if lo < hi:
                w = st["w"][e].double() * torch.repeat_interleave(st["w_scale"][e].double()[block_of], 128, 1)
                out[lo:hi] = torch.mm(x[lo:hi], w.t())
        return out
    top_k, E = case["top_k"], case["E"]
    if case["op"] == "combine":
        rows = st["rows"].detach().double()
        out = torch.zeros((case["M"], case["K"]), dtype=torch.float64, device=_DEV)
        train = case["train"]
        grad_rows = torch.zeros_like(rows) if train else None
        grad_weights = torch.zeros((case["M"], top_k), dtype=torch.float64, device=_DEV) if train else None
        for s in range(top_k):
            token = torch.nonzero(st["row_of_slot"][:, s] >= 0).flatten()
            at, w = st["row_of_slot"][token, s].long(), st["weights"].detach()[token, s].double()
            out[token] += rows[at] * w[:, None]
            if train:
                g = st["grad"][token].double()
                grad_rows[at] = g * w[:, None]
                grad_weights[token, s] = torch.linalg.vecdot(g, rows[at])
        return {"out": out, "grad_rows": grad_rows, "grad_weights": grad_weights}
    # one expert after the other; what has none comes last
    ids = st["ids"].flatten()
    has = (ids >= 0) & (ids < E)
    slots = [torch.nonzero(ids == e).flatten() for e in range(E)]
    offsets = torch.tensor([0] + [len(s) for s in slots]).cumsum(0)
    live = torch.cat(slots)
    order = torch.cat([live, torch.nonzero(~has).flatten()])
    row_of_slot = torch.argsort(order)
    row_of_slot = torch.where(has, row_of_slot, -1 - row_of_slot).reshape(-1, top_k)
    token = torch.div(live, top_k, rounding_mode="floor")
    rows = torch.zeros((ids.numel(), case["K"]), dtype=torch.float64, device=_DEV)
    rows[:len(live)] = st["x"].detach().double()[token]
    scale = grad = None
    if case["dtype"] == "fp8":
        scale = torch.zeros((ids.numel(), case["K"] // 128), dtype=torch.float64, device=_DEV)
        scale[:len(live)] = st["x_scale"].double()[token]
    if case["train"]:
        grad = torch.zeros((case["M"], case["K"]), dtype=torch.float64, device=_DEV)
        grad.index_add_(0, token, st["grad"][:len(live)].double())
    return {"rows": rows, "scale": scale, "offsets": offsets.to(torch.int32).to(_DEV), "row_of_slot": row_of_slot.to(torch.int32),
            "grad_x": grad}


def work(case):
    M, K = case["M"], case["K"]
    if case["op"] == "adapters":
        N, rank = case["N"], case["rank"]
        used = min(case["adapters"], case["requests"])
        x = M * K + M * K // 32 if case["fp8"] else 2 * M * K
        return {"bytes": x + 4 * M * N + 2 * used * rank * (N + K) + 4 * M, "flops": 2.0 * M * rank * (N + K)}
    top_k, E = case["top_k"], case["E"]
    R = M * top_k
    live = (M - case["padding"]) * top_k
    if case["op"] == "grouped":
        N, used = case["N"], min(E, live)
        return {"bytes": (K + 4 * (K // 128)) * live + used * (N * K + 4 * ((N + 127) // 128) * (K // 128)) + 2 * R * N + 4 * E,
                "flops": 2.0 * live * N * K}
    size = _SIZES[case["dtype"]] * K
    if case["op"] == "sort":
        if case["dtype"] == "fp8":
            size += 4 * (K // 128)
        forward = (M + R) * size + 8 * R + 4 * E
        return {"bytes": forward + (live * size + M * size if case["train"] else 0), "flops": R * K}
    forward = live * size + M * size + 8 * R
    backward = (R + M) * size + 4 * R if case["train"] else 0          # (the rows are read once for both)
    return {"bytes": forward + backward, "flops": (6.0 if case["train"] else 2.0) * live * K}
