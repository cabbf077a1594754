"""The gated feed-forward block (forward, backward) and the Muon step of include/ngp_hip.h: cases to measure, their plain forms and their values in 64 bits."""
import math
import os
import sys

import numpy as np
import torch

own = False   # False: the plain forms below; True: the library's entry points

DTYPES = {"f16": (0, torch.float16), "bf16": (1, torch.bfloat16), "f32": (2, torch.float32)}
ACTIVATIONS = {"none": 0, "relu": 1, "logistic": 2, "silu": 4, "gelu": 5}
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315   # the quintic of the Newton-Schulz iteration
LEARNING_RATE, MOMENTUM, WEIGHT_DECAY, EPSILON, LOSS_SCALE = 0.02, 0.95, 0.01, 1e-7, 128.0


def listed():
    return [
        # one token through a wide block: the weights are read once and nothing else counts
        {"name": "forward one row", "op": "forward", "rows": 1, "n_in": 2048, "n_hidden": 8192, "n_out": 2048, "dtype": "bf16", "activation": "silu"},
        # a few tokens decoded together
        {"name": "forward few rows", "op": "forward", "rows": 24, "n_in": 4096, "n_hidden": 10240, "n_out": 4096, "dtype": "f16", "activation": "gelu"},
        # the block in place of the 64-neuron MLP of the image / SDF configurations: 2^18 samples, 32 encoded features, 16 (padded) outputs
        {"name": "forward samples", "op": "forward", "rows": 262144, "n_in": 32, "n_hidden": 64, "n_out": 16, "dtype": "f16", "activation": "relu"},
        # a prompt through a wide block
        {"name": "forward wide", "op": "forward", "rows": 8192, "n_in": 4096, "n_hidden": 8192, "n_out": 4096, "dtype": "bf16", "activation": "silu"},
        # the training step of those samples
        {"name": "backward samples", "op": "backward", "rows": 262144, "n_in": 32, "n_hidden": 64, "n_out": 16, "dtype": "f16", "activation": "relu"},
        # an ordinary training batch
        {"name": "backward ordinary", "op": "backward", "rows": 4096, "n_in": 1024, "n_hidden": 2816, "n_out": 1024, "dtype": "bf16", "activation": "gelu"},
        # widths that are no multiple of a vector, rows that end inside a tile
        {"name": "backward odd", "op": "backward", "rows": 1537, "n_in": 387, "n_hidden": 1061, "n_out": 259, "dtype": "f16", "activation": "silu"},
        # a large training batch
        {"name": "backward wide", "op": "backward", "rows": 8192, "n_in": 4096, "n_hidden": 8192, "n_out": 4096, "dtype": "f16", "activation": "silu"},
        # the matrices of a small network: 64 neurons
        {"name": "muon small", "op": "muon", "count": 5, "n_rows": 64, "n_cols": 64, "dtype": "f16", "nesterov": True},
        # the square matrices of the layers of a middling model, together
        {"name": "muon layers", "op": "muon", "count": 24, "n_rows": 768, "n_cols": 768, "dtype": "bf16", "nesterov": True},
        # one matrix of odd sides, single-precision gradients
        {"name": "muon odd", "op": "muon", "count": 1, "n_rows": 1531, "n_cols": 1000, "dtype": "f32", "nesterov": False},
        # the projections of a wide block
        {"name": "muon wide", "op": "muon", "count": 2, "n_rows": 8192, "n_cols": 4096, "dtype": "bf16", "nesterov": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width of the range: mostly multiples of 8, some odd ones."""
    w = _log_int(rng, low, high)
    return w if rng.random() < 0.25 else max(8, (w + 4) // 8 * 8)


def draw(rng):
    largest = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["forward", "backward", "muon"])
        if op == "muon":
            case = {"op": op, "count": _log_int(rng, 1, 32), "n_rows": _width(rng, 16, 8192), "n_cols": _width(rng, 16, 8192),
                    "dtype": rng.choice(["f16", "bf16", "f32"]), "nesterov": rng.random() < 0.5}
            if case["count"] * case["n_rows"] * case["n_cols"] > 1 << 27:
                continue
        else:
            case = {"op": op, "rows": _log_int(rng, 1, 262144), "n_in": _width(rng, 16, 4096), "n_hidden": _width(rng, 32, 10240), "n_out": _width(rng, 3, 4096),
                    "dtype": rng.choice(["f16", "bf16"]), "activation": rng.choice(sorted(ACTIVATIONS))}
            if case["rows"] * max(case["n_in"], case["n_hidden"], case["n_out"]) > 1 << 27:
                continue
        if _cost(case) <= largest:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 1e14)


def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "muon":
        n, k = sorted((case["n_rows"], case["n_cols"]))
        elements = case["count"] * n * k
        params = size if case["dtype"] != "f32" else 0
        return {"bytes": elements * (size + 4 + 4 + 4 + 4 + params), "flops": case["count"] * 5 * (n * n * k + n ** 3 + 2 * n * n * k)}
    m, d, f, o = case["rows"], case["n_in"], case["n_hidden"], case["n_out"]
    weights = 2 * f * d + o * f
    if case["op"] == "forward":
        return {"bytes": size * (m * (d + o) + weights), "flops": 2 * m * f * (2 * d + o)}
    return {"bytes": size * (m * (d + o) + weights + m * d + weights), "flops": 2 * m * f * (6 * d + 2 * o)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]][1]

    def normal(*shape, scale, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(to)

    state = {"case": dict(case)}
    if case["op"] == "muon":
        b, r, c = case["count"], case["n_rows"], case["n_cols"]
        state["grads"] = normal(b, r, c, scale=LOSS_SCALE * 1e-2)
        state["momentum"] = normal(b, r, c, scale=5e-2, to=torch.float32)
        state["master"] = normal(b, r, c, scale=c ** -0.5, to=torch.float32)
        state["params"] = None if case["dtype"] == "f32" else state["master"].to(dtype)
        return state
    m, d, f, o = case["rows"], case["n_in"], case["n_hidden"], case["n_out"]
    state["x"] = normal(m, d, scale=1.0)
    state["w_gate"], state["w_up"], state["w_down"] = normal(f, d, scale=d ** -0.5), normal(f, d, scale=d ** -0.5), normal(o, f, scale=f ** -0.5)
    if case["op"] == "backward":
        state["dy"] = normal(m, o, scale=m ** -0.5)   # a mean over the batch, with a loss scale
        state["dx"] = torch.empty_like(state["x"])
        state["dw_gate"], state["dw_up"], state["dw_down"] = (torch.empty_like(state[k]) for k in ("w_gate", "w_up", "w_down"))
    else:
        state["y"] = torch.empty(m, o, device="cuda", dtype=dtype)
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return {"forward": _own_forward, "backward": _own_backward, "muon": _own_muon}[op](state)
    return {"forward": _plain_forward, "backward": _plain_backward, "muon": _plain_muon}[op](state)


# ---- the plain forms -------------------------------------------------------------------------------------------------------------------

def _activate(g, activation):
    """(act(g), act'(g))"""
    if activation == "none":
        return g, torch.ones_like(g)
    if activation == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if activation == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    s = 1.0 / (1.0 + torch.exp(-g))
    if activation == "logistic":
        return s, s * (1.0 - s)
    return g * s, s * (1.0 + g * (1.0 - s))


def _plain_forward(state):
    x, w_gate, w_up, w_down = (state[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    a, _ = _activate(x @ w_gate.T, state["case"]["activation"])
    return {"y": ((a * (x @ w_up.T)) @ w_down.T).to(state["x"].dtype)}


def _plain_backward(state):
    dtype = state["x"].dtype
    x, w_gate, w_up, w_down, dy = (state[k].float() for k in ("x", "w_gate", "w_up", "w_down", "dy"))
    g, u = x @ w_gate.T, x @ w_up.T
    a, slope = _activate(g, state["case"]["activation"])
    dh = dy @ w_down
    dg, du = dh * u * slope, dh * a
    return {"dx": (dg @ w_gate + du @ w_up).to(dtype), "dw_gate": (dg.T @ x).to(dtype), "dw_up": (du.T @ x).to(dtype), "dw_down": (dy.T @ (a * u)).to(dtype)}


def _plain_muon(state):
    case = state["case"]
    r, c = case["n_rows"], case["n_cols"]
    g = state["grads"].float() * (1.0 / LOSS_SCALE)
    state["momentum"].mul_(MOMENTUM).add_(g)
    x = g + MOMENTUM * state["momentum"] if case["nesterov"] else state["momentum"]
    x = x / (x.square().sum(dim=(1, 2), keepdim=True).sqrt() + EPSILON)
    x = x.transpose(1, 2).contiguous() if r > c else x
    for _ in range(5):
        a = x @ x.transpose(1, 2).contiguous()
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    x = x.transpose(1, 2) if r > c else x
    state["master"].mul_(1.0 - LEARNING_RATE * WEIGHT_DECAY).sub_(LEARNING_RATE * math.sqrt(max(1.0, r / c)) * x)
    out = {"momentum": state["momentum"], "master": state["master"]}
    if state["params"] is not None:
        out["params"] = state["params"].copy_(state["master"])
    return out


# ---- the library's entry points ---------------------------------------------------------------------------------------------------------

def _library():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blender-ngp_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import capi
    return capi, capi.load_ngp_hip()


def _handle(state):
    """What a program keeps from call to call: the library, the block's or the matrices' description and the workspace."""
    if "handle" not in state:
        capi, ngp = _library()
        case = state["case"]
        code = DTYPES[case["dtype"]][0]
        if case["op"] == "muon":
            desc = np.zeros(case["count"], capi.MUON_MATRIX)
            desc["offset"] = np.arange(case["count"], dtype="u8") * (case["n_rows"] * case["n_cols"])
            desc["rows"], desc["cols"] = case["n_rows"], case["n_cols"]
            size = ngp.ngp_hip_muon_workspace_bytes(case["count"], desc.ctypes.data)
        else:
            desc = np.zeros(1, capi.GATED_FFN)
            desc["n_in"], desc["n_hidden"], desc["n_out"] = case["n_in"], case["n_hidden"], case["n_out"]
            desc["dtype"], desc["activation"] = code, ACTIVATIONS[case["activation"]]
            size = ngp.ngp_hip_gated_ffn_workspace_bytes(desc.ctypes.data, case["rows"], int(case["op"] == "backward"))
        state["handle"] = capi, ngp, desc, code, torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    return state["handle"]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_forward(state):
    capi, ngp, desc, _, ws = _handle(state)
    x, y = state["x"], state["y"]
    capi.check(ngp.ngp_hip_gated_ffn_forward(_stream(), desc.ctypes.data, x.shape[0], x.data_ptr(), x.stride(0), state["w_gate"].data_ptr(), state["w_up"].data_ptr(),
                                             state["w_down"].data_ptr(), y.data_ptr(), y.stride(0), ws.data_ptr(), ws.numel()))
    return {"y": y}


def _own_backward(state):
    capi, ngp, desc, _, ws = _handle(state)
    x, dy, dx = state["x"], state["dy"], state["dx"]
    capi.check(ngp.ngp_hip_gated_ffn_backward(_stream(), desc.ctypes.data, x.shape[0], x.data_ptr(), x.stride(0), state["w_gate"].data_ptr(), state["w_up"].data_ptr(),
                                              state["w_down"].data_ptr(), dy.data_ptr(), dy.stride(0), dx.data_ptr(), dx.stride(0), state["dw_gate"].data_ptr(),
                                              state["dw_up"].data_ptr(), state["dw_down"].data_ptr(), ws.data_ptr(), ws.numel()))
    return {k: state[k] for k in ("dx", "dw_gate", "dw_up", "dw_down")}


def _own_muon(state):
    capi, ngp, desc, code, ws = _handle(state)
    params = state["params"]
    capi.check(ngp.ngp_hip_muon_step(_stream(), len(desc), desc.ctypes.data, LEARNING_RATE, MOMENTUM, WEIGHT_DECAY, EPSILON, int(state["case"]["nesterov"]), 5, LOSS_SCALE,
                                     code, state["grads"].data_ptr(), state["master"].data_ptr(), None if params is None else params.data_ptr(),
                                     state["momentum"].data_ptr(), ws.data_ptr(), ws.numel()))
    out = {"momentum": state["momentum"], "master": state["master"]}
    if params is not None:
        out["params"] = params
    return out


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "muon":
        return _exact_muon(case, s)
    x, wg, wu, wd = (s[k].double() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    kind = case["activation"]
    sigma = torch.sigmoid(g)
    phi = torch.special.ndtr(g) if kind == "gelu" else None
    act = {"none": lambda: g, "relu": lambda: g.clamp(min=0), "logistic": lambda: sigma, "silu": lambda: g * sigma, "gelu": lambda: g * phi}[kind]()
    if case["op"] == "forward":
        return {"y": torch.mm(act * u, wd.t())}
    slope = {"none": lambda: torch.ones_like(g), "relu": lambda: torch.where(g > 0, 1.0, 0.0).double(), "logistic": lambda: sigma - sigma.square(),
             "silu": lambda: sigma + g * (sigma - sigma.square()), "gelu": lambda: phi + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)}[kind]()
    dy = s["dy"].double()
    dh = torch.mm(dy, wd)
    dgate, dup = dh * u * slope, dh * act
    return {"dx": torch.mm(dgate, wg) + torch.mm(dup, wu), "dw_gate": torch.mm(dgate.t(), x), "dw_up": torch.mm(dup.t(), x), "dw_down": torch.mm(dy.t(), act * u)}


def _exact_muon(case, s):
    r, c = case["n_rows"], case["n_cols"]
    momentum, master = [], []
    for grad, mom, w in zip(s["grads"].double(), s["momentum"].double(), s["master"].double()):
        grad = grad / LOSS_SCALE
        mom = MOMENTUM * mom + grad
        x = grad + MOMENTUM * mom if case["nesterov"] else mom.clone()
        x = x / (torch.linalg.norm(x) + EPSILON)
        for _ in range(5):   # the Gram matrix on the short side: X p(X^T X) = p(X X^T) X
            gram = x @ x.t() if r <= c else x.t() @ x
            poly = NS_B * gram + NS_C * gram @ gram
            x = NS_A * x + (poly @ x if r <= c else x @ poly)
        momentum.append(mom)
        master.append((1.0 - LEARNING_RATE * WEIGHT_DECAY) * w - LEARNING_RATE * math.sqrt(max(1.0, r / c)) * x)
    out = {"momentum": torch.stack(momentum), "master": torch.stack(master)}
    if s["params"] is not None:
        out["params"] = out["master"]
    return out
