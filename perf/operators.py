"""The 8-bit path of a decode step, hidden state to token, as measured cases.

Four operators: the RMS norm with the residual's addition whose output is one int8 code per
element and one scale per token (norm); rows as codes and scales, of a matrix laid out once or of
the gated intermediate act(gate) * up (quant); the product of two matrices of codes with a scale
for each token and each row of weights (gemm); and the choice of a token from the logits with
temperature, top-k, top-p and min-p and a given random number (sample).

Where `own` is false, run() computes them from elementary torch operations; where it is true it
calls HipEngine on the same tensors' memory; its outputs are whole, to other streams than the engine's,
after a synchronization of the device.  Codes are returned as the values they stand for.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a 135M-parameter model's token before its FFN: launch and latency bound
        {"name": "norm token 576", "kind": "norm", "type": "f32", "rows": 1, "cols": 576, "res": True},
        # a decode batch of a 70B-shaped model, half-width residual stream
        {"name": "norm batch 64x8192", "kind": "norm", "type": "bf16", "rows": 64, "cols": 8192, "res": True},
        # a prompt of an 8B-shaped model
        {"name": "norm prompt 2048x4096", "kind": "norm", "type": "f32", "rows": 2048, "cols": 4096, "res": True},
        # an 8B-shaped gate matrix turned into codes, once per model
        {"name": "quant weights 14336x4096", "kind": "quant", "type": "f32", "rows": 14336, "cols": 4096,
         "act": "none"},
        # the gated intermediate of a ragged prompt: gate and up are halves of one product's rows
        {"name": "quant swiglu 509x14336", "kind": "quant", "type": "bf16", "rows": 509, "cols": 14336,
         "act": "silu"},
        # one token's gate and up of an 8B-shaped layer
        {"name": "gemm token 28672x4096", "kind": "gemm", "type": "f32", "m": 28672, "n": 4096, "tokens": 1,
         "res": False},
        # a small decode batch through an 8B-shaped model's output projection
        {"name": "gemm head 8x128256", "kind": "gemm", "type": "f32", "m": 128256, "n": 4096, "tokens": 8,
         "res": False},
        # a larger, odd decode batch through down, onto the residual stream
        {"name": "gemm down 61x14336", "kind": "gemm", "type": "bf16", "m": 4096, "n": 14336, "tokens": 61,
         "res": True},
        # a prompt's gate and up
        {"name": "gemm prompt 2048x28672", "kind": "gemm", "type": "bf16", "m": 28672, "n": 4096, "tokens": 2048,
         "res": False},
        # one token's logits, and a decode batch's
        {"name": "sample 1x128256", "kind": "sample", "type": "f32", "rows": 1, "vocab": 128256},
        {"name": "sample 64x128256", "kind": "sample", "type": "f32", "rows": 64, "vocab": 128256},
        # a larger batch of a smaller vocabulary, half-width logits (many equal values)
        {"name": "sample 250x32000", "kind": "sample", "type": "f16", "rows": 250, "vocab": 32000},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "quant", "gemm", "sample"])
    case = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"])}
    if kind in ("norm", "quant"):
        case["cols"] = _spread(rng, 64, 16384)
        case["rows"] = _spread(rng, 1, min(16384, (1 << 24) // case["cols"]))
        if kind == "norm":
            case["res"] = rng.random() < 0.7
        else:
            case["act"] = rng.choice(["none", "silu", "gelu"])
    elif kind == "gemm":
        case["n"] = _spread(rng, 64, 16384)
        case["m"] = _spread(rng, 64, 32768)
        case["tokens"] = _spread(rng, 1, min(2048, int(2.4e11 / (case["n"] * case["m"]))))
        case["res"] = rng.random() < 0.4
    else:
        case["vocab"] = _spread(rng, 1000, 160000)
        case["rows"] = _spread(rng, 1, min(512, (1 << 23) // case["vocab"]))
    return case


# ------------------------------------------------------------------------------- inputs


def _padded(n):
    """Rows of codes start on 16-byte boundaries."""
    return (n + 15) // 16 * 16


def _codes(rows, n, g):
    """Codes as a normal matrix's rows have them, in rows of _padded(n) bytes."""
    q = torch.randn(rows, _padded(n), device="cuda", generator=g).mul_(31.0).round_().clamp_(-127, 127)
    return q.to(torch.int8)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    state = {"case": case}

    def empty(name, *shape, dtype=torch.float32):
        state[name] = torch.empty(*shape, device="cuda", dtype=dtype)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if kind == "norm":
        t, n = case["rows"], case["cols"]
        # a residual stream has channels far larger than the others
        channels = torch.exp(0.7 * normal(n))
        state["x"] = (0.3 * normal(t, n)).to(dtype)
        if case["res"]:
            state["res"] = (normal(t, n) * channels).to(dtype)
            empty("sum", t, n, dtype=dtype)
        state["norm"] = torch.rand(n, device="cuda", generator=g) + 0.5
    elif kind == "quant":
        t, n = case["rows"], case["cols"]
        if case["act"] == "none":
            state["x"] = (normal(t, n) / math.sqrt(n)).to(dtype)
        else:
            state["x"] = (1.5 * normal(t, 2 * n)).to(dtype)  # gate | up
    elif kind == "gemm":
        t, m, n = case["tokens"], case["m"], case["n"]
        state["x"], state["w"] = _codes(t, n, g), _codes(m, n, g)
        state["x_scale"] = (torch.rand(t, device="cuda", generator=g) + 0.5) / 31.0
        state["w_scale"] = (torch.rand(m, device="cuda", generator=g) + 0.5) / (31.0 * math.sqrt(n))
        if case["res"]:
            state["res"] = normal(t, m).to(dtype)
        empty("y", t, m, dtype=dtype)
    else:
        t, n = case["rows"], case["vocab"]
        # logits of a trained head: a wide body and a few words that fit
        top = torch.randint(0, n, (t, 40), device="cuda", generator=g)
        x = 2.0 * normal(t, n)
        x.scatter_add_(1, top, 4.0 + 6.0 * torch.rand(t, 40, device="cuda", generator=g))
        state["logits"] = x.to(dtype)
        # what requests ask for: greedy, temperature alone, top-k, top-p, min-p and their mixtures
        table = torch.tensor([[0.7, 50.0, 0.9, 0.0], [1.0, 0.0, 0.95, 0.0], [0.8, 40.0, 0.95, 0.05], [1.0, 0.0, 1.0, 0.1],
                              [0.0, 0.0, 1.0, 0.0], [1.2, 200.0, 1.0, 0.02], [1.0, 0.0, 1.0, 0.0], [0.6, 20.0, 0.95, 0.0]],
                             device="cuda")
        which = (torch.arange(t, device="cuda") + seed) % len(table) if t > 1 else torch.zeros(1, dtype=torch.long, device="cuda")
        state["params"] = table[which].contiguous()
        state["params"].view(torch.int32)[:, 1] = table[which][:, 1].int()  # top_k is a whole number
        state["u"] = torch.rand(t, device="cuda", generator=g)
        empty("ids", t, dtype=torch.int32)
        empty("probs", t)
    if kind in ("norm", "quant"):
        empty("q", t, n, dtype=torch.int8)
        empty("scale", t)
        empty("values", t, n)
    return state


# -------------------------------------------------------------------------- plain forms


def _rows_as_codes(u, by):
    """Codes of the rows of u (64 bits, as which code is nearest is decided at borders) and their
    values, where a code's step is max|u| * by / 127."""
    top = u.abs().amax(1, keepdim=True)
    safe = torch.where(top > 0, top, torch.ones_like(top))
    scale = (top * by / 127.0).float()
    return {"scale": scale.squeeze(1), "values": torch.round(u * 127.0 / safe).float() * scale}


def _plain_norm(state):
    v = state["x"].double()
    out = {}
    if "res" in state:
        v = v + state["res"].double()
        out["sum"] = v.to(state["x"].dtype)
    by = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    out.update(_rows_as_codes(v * state["norm"].double(), by))
    return out


def _plain_quant(state):
    case, x = state["case"], state["x"].double()
    if case["act"] != "none":
        gate, up = x[:, :case["cols"]], x[:, case["cols"]:]
        if case["act"] == "silu":
            x = gate / (1.0 + torch.exp(-gate)) * up
        else:
            inner = math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate)
            x = 0.5 * gate * (1.0 + torch.tanh(inner)) * up
    return _rows_as_codes(x, 1.0)


def _plain_gemm(state):
    n = state["case"]["n"]
    y = state["x"][:, :n].float() @ state["w"][:, :n].float().t()
    y = y * state["x_scale"].unsqueeze(1) * state["w_scale"]
    if "res" in state:
        y = y + state["res"].float()
    return y.to(state["y"].dtype)


def _plain_sample(state):
    x = state["logits"].double()
    t, n = x.shape
    params = state["params"].double()
    temperature, top_p, min_p = params[:, 0:1], params[:, 2:3], params[:, 3:4]
    top_k = state["params"].view(torch.int32)[:, 1:2].long()
    greedy = temperature <= 0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest index first
    weight = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    rank = torch.arange(n, device=x.device).unsqueeze(0)
    weight = torch.where((top_k <= 0) | (rank < top_k), weight, torch.zeros_like(weight))
    running = torch.cumsum(weight, 1)
    before = running - weight
    keep = (top_p >= 1) | (before < top_p * running[:, -1:])
    keep = keep & (weight >= min_p) | (rank == 0)
    keep = torch.where(greedy, rank == 0, keep)
    weight = torch.where(keep, weight, torch.zeros_like(weight))
    by_index = torch.zeros_like(weight).scatter_(1, order, weight)
    running = torch.cumsum(by_index, 1)
    total = running[:, -1:]
    wanted = state["u"].double().unsqueeze(1) * total
    ids = (running <= wanted).sum(1, keepdim=True).clamp_(max=n - 1)
    return {"ids": ids.squeeze(1).int(), "probs": (by_index.gather(1, ids) / total).squeeze(1).float()}


# ------------------------------------------------------------------ the framework's calls

_engine = None


def _buffers(state):
    """Handles on the tensors' memory, kept with them as a program keeps them."""
    global _engine
    from hayai_amd import HipEngine
    if _engine is None:
        _engine = HipEngine(0)
    case, e = state["case"], _engine
    types = {"f32": 0, "f16": 1, "bf16": 30}  # GGML type ids
    state["handles"] = h = {k: e.wrap(v.data_ptr(), v.numel() * v.element_size())
                            for k, v in state.items() if isinstance(v, torch.Tensor)}
    kind, ty = case["kind"], types[case["type"]]
    if kind == "norm":
        h["desc"] = e.rms_norm_i8_desc(ty, case["rows"], case["cols"], EPS)
    elif kind == "quant":
        wide = case["cols"] * (1 if case["act"] == "none" else 2)
        h["desc"] = e.quant_i8_desc(ty, case["rows"], case["cols"], x_stride=wide, up_stride=wide,
                                    act=1 if case["act"] == "gelu" else 0)
        h["up_off"] = case["cols"] * state["x"].element_size()
    elif kind == "gemm":
        wide = _padded(case["n"])
        h["desc"] = e.gemm_i8_desc(ty, case["m"], case["n"], case["tokens"], w_stride=wide, x_stride=wide)
    else:
        h["desc"] = e.sample_desc(ty, case["rows"], case["vocab"])
    # the engine's stream does not wait for torch's: the inputs are whole before its first call
    torch.cuda.synchronize()
    return h


def _own(state):
    h = state.get("handles") or _buffers(state)
    case, e = state["case"], _engine
    kind = case["kind"]
    if kind == "norm":
        e.rms_norm_i8_dev(h["desc"], h["x"], 0, h.get("res"), 0, h["norm"], 0, h.get("sum"), 0, h["q"], 0,
                          h["scale"], 0, h["values"], 0)
    elif kind == "quant":
        gated = case["act"] != "none"
        e.quant_i8_dev(h["desc"], h["x"], 0, h["x"] if gated else None, h["up_off"] if gated else 0, h["q"], 0,
                       h["scale"], 0, h["values"], 0)
    elif kind == "gemm":
        e.gemm_i8_dev(h["desc"], h["w"], 0, h["w_scale"], 0, h["x"], 0, h["x_scale"], 0, h.get("res"), 0, h["y"], 0)
        return state["y"]
    else:
        e.sample_dev(h["desc"], h["logits"], 0, h["params"], 0, h["u"], 0, h["ids"], 0, h["probs"], 0)
        return {"ids": state["ids"], "probs": state["probs"]}
    out = {"scale": state["scale"], "values": state["values"]}
    if "sum" in state:
        out["sum"] = state["sum"]
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "quant": _plain_quant, "gemm": _plain_gemm,
            "sample": _plain_sample}[state["case"]["kind"]](state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind in ("norm", "quant"):
        t, n = case["rows"], case["cols"]
        if kind == "norm":  # x, the residual and the sum; codes and values
            each, more = size * (3 if case["res"] else 1) + 1 + 4, 4 * n
        else:
            each, more = size * (1 if case["act"] == "none" else 2) + 1 + 4, 0
        return {"bytes": t * n * each + more + 4 * t, "flops": 8 * t * n}
    if kind == "gemm":
        t, m, n = case["tokens"], case["m"], case["n"]
        return {"bytes": (t + m) * n + 4 * (t + m) + size * t * m * (2 if case["res"] else 1), "flops": 2 * t * m * n}
    return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 4 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------- the definitions in 64 bits


def _host(v):
    return v.double().cpu().numpy()


def _exact_codes(u, unit):
    """Nearest multiples of each row's step max|u| / 127, times the row's unit."""
    top = np.max(np.abs(u), axis=1, keepdims=True)
    codes = np.rint(127.0 * u / np.where(top == 0.0, 1.0, top))
    step = top / 127.0 * unit
    return {"scale": step[:, 0], "values": codes * step}


def _exact_token(logits, temperature, top_k, top_p, min_p, u):
    if temperature <= 0:
        return int(np.argmax(logits)), 1.0
    order = np.argsort(-logits, kind="stable")
    p = np.exp((logits[order] - logits.max()) / temperature)
    length = len(p) if top_k <= 0 else min(int(top_k), len(p))
    p = p[:length]
    if top_p < 1:
        length = min(length, int(np.searchsorted(np.cumsum(p), top_p * p.sum(), side="left")) + 1)
    length = max(1, min(length, int(np.count_nonzero(p >= min_p))))
    kept = np.sort(order[:length])
    p = np.exp((logits[kept] - logits.max()) / temperature)
    running = np.cumsum(p)
    at = min(int(np.searchsorted(running, u * running[-1], side="right")), length - 1)
    return int(kept[at]), p[at] / running[-1]


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        v, out = _host(state["x"]), {}
        if case["res"]:
            v = v + _host(state["res"])
            out["sum"] = v
        out.update(_exact_codes(v * _host(state["norm"]), (np.mean(np.square(v), axis=1, keepdims=True) + EPS) ** -0.5))
        return out
    if kind == "quant":
        x = _host(state["x"])
        if case["act"] != "none":
            gate, up = np.split(x, 2, axis=1)
            if case["act"] == "silu":
                x = up * gate / (1.0 + np.exp(-gate))
            else:
                x = up * gate / (1.0 + np.exp(-2.0 * np.sqrt(2.0 / np.pi) * (gate + 0.044715 * gate ** 3)))
        return _exact_codes(x, 1.0)
    if kind == "gemm":  # whole numbers below 2^53: exact in any order
        n = case["n"]
        y = torch.mm(state["w"][:, :n].double(), state["x"][:, :n].double().t().contiguous()).t()
        y = y * torch.outer(state["x_scale"].double(), state["w_scale"].double())
        return y + state["res"].double() if case["res"] else y
    top_k, params = state["params"].view(torch.int32)[:, 1].cpu().numpy(), _host(state["params"])
    got = [_exact_token(row, t, k, p, m, u) for row, (t, _, p, m), k, u
           in zip(_host(state["logits"]), params, top_k, _host(state["u"]))]
    return {"ids": np.array([i for i, _ in got], np.int32), "probs": np.array([p for _, p in got])}
