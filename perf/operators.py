"""The operators around the product with compressed weights, as cases that can be timed and checked: the product
with bias, activation (gated or not) and residual in its epilogue, the product grouped by expert, the choice of
experts with the lists the grouped product reads, and the weighted sum of the experts' rows.

Where `own` is false `run` computes a case with elementary torch operations; where it is true it calls the
framework's operators.  `exact` computes the same from the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
GRID_VALUES = (0.25, 0.75, 1.25, 1.75, 2.25, 2.75)


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # decode step, one sequence: the MLP's way back to the hidden size, added to the residual stream
        {"name": "fused_down_residual_m1", "op": "fused", "M": 1, "N": 4096, "K": 11008, "gated": False,
         "act": "none", "bias": "", "residual": "half", "out": "half"},
        # decode step, one sequence, the largest matrix of a layer: gate and up projections with the gated activation
        {"name": "fused_gate_up_m1", "op": "fused", "M": 1, "N": 28672, "K": 8192, "gated": True,
         "act": "silu", "bias": "", "residual": "", "out": "half"},
        # a ragged batch of thirteen sequences: a classic MLP's first half, an odd number of outputs, 32-bit result
        {"name": "fused_bias_gelu_m13", "op": "fused", "M": 13, "N": 11007, "K": 4096, "gated": False,
         "act": "gelu", "bias": "float", "residual": "", "out": "float"},
        # a prompt: gate and up projections
        {"name": "fused_gate_up_prompt", "op": "fused", "M": 2048, "N": 11008, "K": 4096, "gated": True,
         "act": "silu", "bias": "half", "residual": "", "out": "half"},
        # decode step of one sequence: two of eight experts, one row each
        {"name": "grouped_gate_up_one_token", "op": "grouped", "E": 8, "active": 2, "T": 1, "k": 2, "N": 11008, "K": 4096,
         "gated": True, "act": "silu", "bias": "", "out": "half", "gather": True},
        # decode step of 24 sequences: most experts have a few rows, some none; the way back, rows already in order
        {"name": "grouped_down_24_tokens", "op": "grouped", "E": 16, "active": 15, "T": 24, "k": 2, "N": 4096, "K": 11008,
         "gated": False, "act": "none", "bias": "", "out": "half", "gather": False},
        # many small experts, a short prompt: tens of rows each, ragged
        {"name": "grouped_small_experts", "op": "grouped", "E": 64, "active": 61, "T": 333, "k": 6, "N": 1408, "K": 2048,
         "gated": True, "act": "gelu_tanh", "bias": "half", "out": "half", "gather": True},
        # a prompt through eight large experts
        {"name": "grouped_gate_up_prompt", "op": "grouped", "E": 8, "active": 8, "T": 2048, "k": 2, "N": 11008, "K": 4096,
         "gated": True, "act": "silu", "bias": "", "out": "half", "gather": True},
        # decode step of 24 sequences
        {"name": "route_24_tokens", "op": "route", "T": 24, "E": 16, "k": 2, "dtype": "half", "scoring": "softmax",
         "normalize": True, "masked": 0},
        # a long packed prompt, padded rows masked out, many experts
        {"name": "route_prompt", "op": "route", "T": 16384, "E": 128, "k": 8, "dtype": "float", "scoring": "sigmoid",
         "normalize": True, "masked": 37},
        # decode step of 24 sequences
        {"name": "combine_24_tokens", "op": "combine", "T": 24, "k": 2, "N": 4096, "dropped": 0, "residual": "half", "out": "half"},
        # a prompt, some choices dropped
        {"name": "combine_prompt", "op": "combine", "T": 4099, "k": 6, "N": 4096, "dropped": 3, "residual": "half", "out": "half"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fused", "fused", "grouped", "grouped", "route", "combine"])
    act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
    some = ["", "half", "float"]
    if op == "fused":
        while True:
            gated = rng.random() < 0.4
            M, N, K = _log(rng, 1, 4096), _log(rng, 16, 32768), 64 * _log(rng, 4, 256)
            N2 = 2 * N if gated else N
            if M * N2 * K <= 2048 * 22016 * 4096 and N2 * K <= 57344 * 8192:
                break
        return {"op": op, "M": M, "N": N, "K": K, "gated": gated, "act": act, "bias": rng.choice(some),
                "residual": rng.choice(some), "out": rng.choice(["half", "half", "float"])}
    if op == "grouped":
        while True:
            E = _log(rng, 2, 128)
            k = rng.randint(1, min(8, E))
            T, N, K = _log(rng, 1, 4096), _log(rng, 64, 11008), 64 * _log(rng, 4, 172)
            gated = rng.random() < 0.5
            N2 = 2 * N if gated else N
            if T * k * N2 * K <= 4096 * 22016 * 4096 and E * N2 * K <= 16 * 4096 * 11008:
                break
        active = rng.randint(max(1, min(E, T * k) // 2), min(E, T * k))
        return {"op": op, "E": E, "active": active, "T": T, "k": k, "N": N, "K": K, "gated": gated, "act": act,
                "bias": rng.choice(some), "out": rng.choice(["half", "half", "float"]), "gather": rng.random() < 0.7}
    if op == "route":
        E = _log(rng, 4, 512)
        T = _log(rng, 1, 16384)
        return {"op": op, "T": T, "E": E, "k": rng.randint(1, min(12, E)), "dtype": rng.choice(["half", "bfloat", "float"]),
                "scoring": rng.choice(["softmax", "sigmoid"]), "normalize": rng.random() < 0.7,
                "masked": rng.choice([0, 0, T // 7])}
    T, k, N = _log(rng, 1, 8192), rng.randint(1, 8), _log(rng, 64, 16384)
    while T * k * N > 4099 * 6 * 4096:
        T = max(1, T // 2)
    return {"op": op, "T": T, "k": k, "N": N, "dropped": rng.choice([0, T // 5]), "residual": rng.choice(some),
            "out": rng.choice(["half", "float"])}


# ------------------------------------------------------------------------------------------ inputs
_TYPES = {"half": torch.float16, "bfloat": torch.bfloat16, "float": torch.float32}


def _maybe(kind, gen, *shape, std=1.0):
    if not kind:
        return None
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(_TYPES[kind])


def _weights(gen, *shape):
    codes = torch.randint(-32768, 32768, shape, generator=gen, device=DEV, dtype=torch.int32).to(torch.int16)
    pick = torch.randint(0, len(GRID_VALUES), (256, 8), generator=gen, device=DEV)
    grid = torch.tensor(GRID_VALUES, device=DEV)[pick].to(torch.float16)
    return codes, grid


def _activations(gen, rows, K):
    """Unit normal with every 500th channel three times as wide, as hidden states have them."""
    x = torch.randn(rows, K, generator=gen, device=DEV)
    x[:, ::500] *= 3.0
    return x.to(torch.float16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "fused":
        M, N, K = case["M"], case["N"], case["K"]
        N2 = 2 * N if case["gated"] else N
        s["x"] = _activations(gen, M, K)
        s["codes"], s["grid"] = _weights(gen, N2, K // 8)
        s["scale"] = 1.0 / math.sqrt(K)
        s["bias"] = _maybe(case["bias"], gen, N2, std=0.5)
        s["residual"] = _maybe(case["residual"], gen, M, N)
    elif case["op"] == "grouped":
        E, T, k, N, K = case["E"], case["T"], case["k"], case["N"], case["K"]
        N2 = 2 * N if case["gated"] else N
        R = T * k
        s["codes"], s["grid"] = _weights(gen, E, N2, K // 8)
        s["scale"] = (0.8 + 0.4 * torch.rand(E, generator=gen, device=DEV)) / math.sqrt(K)
        s["bias"] = _maybe(case["bias"], gen, E, N2, std=0.5)
        # every expert that is active has at least one row, the others share the rest unevenly
        act = torch.randperm(E, generator=gen, device=DEV)[:case["active"]]
        share = torch.softmax(torch.randn(case["active"], generator=gen, device=DEV), 0)
        extra = torch.multinomial(share, R - case["active"], replacement=True, generator=gen) if R > case["active"] else act[:0]
        of = torch.cat([act, act[extra]])
        counts = torch.bincount(of, minlength=E)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        order = torch.argsort(of, stable=True)
        tokens = (torch.randperm(R, generator=gen, device=DEV) // k)[order]
        if case["gather"]:
            s["x"] = _activations(gen, T, K)
            s["rows"] = tokens.to(torch.int32)
        else:
            s["x"] = _activations(gen, R, K)
            s["rows"] = None
    elif case["op"] == "route":
        T, E = case["T"], case["E"]
        logits = torch.randn(T, E, generator=gen, device=DEV) * 1.5 + torch.randn(E, generator=gen, device=DEV) * 0.5
        if case["masked"]:
            logits[torch.randperm(T, generator=gen, device=DEV)[:case["masked"]]] = -math.inf   # padded rows
        s["logits"] = logits.to(_TYPES[case["dtype"]])
    else:
        T, k, N = case["T"], case["k"], case["N"]
        s["y"] = torch.randn(T * k, N, generator=gen, device=DEV).to(torch.float16)
        slots = torch.randperm(T * k, generator=gen, device=DEV).view(T, k).to(torch.int32)
        if case["dropped"]:
            slots[torch.randperm(T, generator=gen, device=DEV)[:case["dropped"]], k - 1] = -1
        s["slots"] = slots
        s["weights"] = torch.softmax(torch.randn(T, k, generator=gen, device=DEV), 1)
        s["residual"] = _maybe(case["residual"], gen, T, N)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        import decode_matmul_amd as dmm
        s = state
        if case["op"] == "fused":
            return dmm.decode_matmul_fused(s["x"], s["codes"], s["grid"], s["scale"], bias=s["bias"], activation=case["act"],
                                           gated=case["gated"], residual=s["residual"], out_dtype=_TYPES[case["out"]])
        if case["op"] == "grouped":
            return dmm.decode_matmul_grouped(s["x"], s["codes"], s["grid"], s["scale"], s["offsets"], rows=s["rows"],
                                             bias=s["bias"], activation=case["act"], gated=case["gated"],
                                             out_dtype=_TYPES[case["out"]])
        if case["op"] == "route":
            r = dmm.route_experts(s["logits"], case["k"], scoring=case["scoring"], normalize=case["normalize"])
            return {"weights": r.weights, "experts": r.experts, "offsets": r.offsets, "rows": r.rows, "slots": r.slots}
        return dmm.combine_experts(s["y"], s["slots"], s["weights"], residual=s["residual"], out_dtype=_TYPES[case["out"]])
    return {"fused": _plain_fused, "grouped": _plain_grouped, "route": _plain_route, "combine": _plain_combine}[case["op"]](state)


def _plain_decode(codes, grid):
    """float32 W [N, K] of codes [N, K/8]: grid row, seven signs and their parity, then plus or minus a quarter."""
    c = codes.to(torch.int32) & 0xFFFF
    s7 = (c >> 8) & 0x7F
    par = s7 ^ (s7 >> 4)
    par = par ^ (par >> 2)
    par = (par ^ (par >> 1)) & 1
    s8 = s7 | (par << 7)
    sign = 1.0 - 2.0 * ((s8.unsqueeze(-1) >> torch.arange(8, device=c.device, dtype=torch.int32)) & 1).float()
    shift = 0.25 - 0.5 * (c >> 15).float()
    w = grid.float()[(c & 0xFF).long()] * sign + shift.unsqueeze(-1)
    return w.to(torch.float16).float().view(codes.shape[0], -1)


def _plain_act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * (1.0 / math.sqrt(2.0))))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_fused(s):
    case = s["case"]
    z = (s["x"].float() @ _plain_decode(s["codes"], s["grid"]).t()) * s["scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if case["gated"]:
        z = _plain_act(z[:, :case["N"]], case["act"]) * z[:, case["N"]:]
    else:
        z = _plain_act(z, case["act"])
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(_TYPES[case["out"]])


def _plain_grouped(s):
    case = s["case"]
    N = case["N"]
    x = s["x"] if s["rows"] is None else s["x"][s["rows"].long()]
    y = torch.empty(x.shape[0], N, device=x.device, dtype=_TYPES[case["out"]])
    edges = s["offsets"].tolist()
    for e in range(case["E"]):
        lo, hi = edges[e], edges[e + 1]
        if lo == hi:
            continue
        z = (x[lo:hi].float() @ _plain_decode(s["codes"][e], s["grid"]).t()) * s["scale"][e]
        if s["bias"] is not None:
            z = z + s["bias"][e].float()
        if case["gated"]:
            z = _plain_act(z[:, :N], case["act"]) * z[:, N:]
        else:
            z = _plain_act(z, case["act"])
        y[lo:hi] = z.to(y.dtype)
    return y


def _plain_route(s):
    case = s["case"]
    T, E, k = case["T"], case["E"], case["k"]
    logits = s["logits"].float()
    top, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    chosen = top > -math.inf
    if case["scoring"] == "softmax":
        big = torch.clamp(logits.max(dim=1, keepdim=True).values, min=-3e38)
        w = torch.exp(top - big)
        total = torch.exp(logits - big).sum(1, keepdim=True)
    else:
        w = 1.0 / (1.0 + torch.exp(-top))
        total = torch.ones_like(w[:, :1])
    if case["normalize"]:
        total = w.sum(1, keepdim=True)
    w = torch.where(chosen, w / total, torch.zeros_like(w))
    experts = torch.where(chosen, idx, torch.full_like(idx, -1))
    key = torch.where(chosen, idx, torch.full_like(idx, E)).reshape(-1)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=E + 1)[:E]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=order.device)
    live = key < E
    rows = torch.where(live[order], order // k, torch.full_like(order, -1))
    slots = torch.where(live, place, torch.full_like(place, -1)).view(T, k)
    i32 = torch.int32
    return {"weights": w, "experts": experts.to(i32), "offsets": offsets.to(i32), "rows": rows.to(i32), "slots": slots.to(i32)}


def _plain_combine(s):
    case = s["case"]
    slots = s["slots"].long()
    z = s["y"][slots.clamp(min=0)].float()
    z = (torch.where(slots < 0, torch.zeros_like(s["weights"]), s["weights"]).unsqueeze(-1) * z).sum(1)
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(_TYPES[case["out"]])


# ------------------------------------------------------------------------------------------ 64 bits
def _exact_weights(codes, grid):
    """float64 W from a table of all 65536 codes."""
    c = torch.arange(65536, device=codes.device)
    table = grid.double()[c % 256]
    bits = torch.stack([(c // 2 ** (8 + d)) % 2 for d in range(7)], 1)
    bits = torch.cat([bits, bits.sum(1, keepdim=True) % 2], 1)
    table = torch.where(bits == 1, -table, table) + torch.where(c >= 32768, -0.25, 0.25).double().unsqueeze(1)
    table = table.to(torch.float16).double()
    return table[codes.long() % 65536].flatten(-2)


def _exact_act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def _exact_rows(x, codes, grid, scale, bias, gated, act):
    z = torch.matmul(x.double(), _exact_weights(codes, grid).t()) * scale
    if bias is not None:
        z += bias.double()
    if not gated:
        return _exact_act(z, act)
    gate, up = z.chunk(2, dim=1)
    return _exact_act(gate, act) * up


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fused":
        y = _exact_rows(s["x"], s["codes"], s["grid"], s["scale"], s["bias"], case["gated"], case["act"])
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "grouped":
        parts = []
        edges = s["offsets"].cpu()
        for e in range(case["E"]):
            p = torch.arange(int(edges[e]), int(edges[e + 1]), device=DEV)
            if p.numel():
                rows = p if s["rows"] is None else s["rows"][p].long()
                parts.append(_exact_rows(s["x"][rows], s["codes"][e], s["grid"], s["scale"][e].double(),
                                         None if s["bias"] is None else s["bias"][e], case["gated"], case["act"]))
        return torch.cat(parts)
    if case["op"] == "route":
        z = s["logits"].double()
        val = torch.sort(z, dim=1, descending=True, stable=True).values[:, :case["k"]]
        if case["scoring"] == "softmax":
            p = torch.exp(val - torch.logsumexp(z, 1, keepdim=True))
        else:
            p = torch.sigmoid(val)
        if case["normalize"]:
            p = p / p.sum(1, keepdim=True)
        return {"weights": torch.where(val == -math.inf, 0.0, p), "experts": None, "offsets": None, "rows": None, "slots": None}
    w = s["weights"].double() * (s["slots"] >= 0)
    z = torch.zeros(case["T"], case["N"], device=DEV, dtype=torch.float64)
    for j in range(case["k"]):
        z += w[:, j:j + 1] * s["y"][s["slots"][:, j].long().clamp(min=0)].double()
    return z if s["residual"] is None else z + s["residual"].double()


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"": 0, "half": 2, "bfloat": 2, "float": 4}
    if case["op"] == "fused":
        M, N, K = case["M"], case["N"], case["K"]
        N2 = 2 * N if case["gated"] else N
        return {"bytes": N2 * K // 4 + 4096 + 2 * M * K + size[case["bias"]] * N2 + size[case["residual"]] * M * N
                + size[case["out"]] * M * N, "flops": 2 * M * N2 * K}
    if case["op"] == "grouped":
        N, K, R = case["N"], case["K"], case["T"] * case["k"]
        N2 = 2 * N if case["gated"] else N
        rows = case["T"] if case["gather"] else R
        return {"bytes": case["active"] * (N2 * K // 4 + size[case["bias"]] * N2 + 4) + 4096 + 2 * rows * K + size[case["out"]] * R * N
                + 4 * (case["E"] + 1) + (4 * R if case["gather"] else 0), "flops": 2 * R * N2 * K}
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": size[case["dtype"]] * T * E + 16 * T * k + 4 * (E + 1), "flops": 5 * T * E}
    T, k, N = case["T"], case["k"], case["N"]
    return {"bytes": 2 * (T * k - case["dropped"]) * N + 8 * T * k + (size[case["residual"]] + size[case["out"]]) * T * N,
            "flops": 2 * T * k * N}
