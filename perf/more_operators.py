"""A decoder layer's attention over a cache of pages, as measured cases.

Four operators: the rotation of queries and keys by their positions, with the new keys and values
put into the cache's pages (rope); copies of whole pages through all layers, for forked sequences
and for a cache that is made dense again (pages); causal attention of a prompt's tokens over their
sequences' pages, packed sequences of different lengths (prompt); and attention of one token a
sequence for a batch whose sequences begin with the same tokens, kept once (decode).

A cache is a tensor of n_pages rows: a page's keys as [kv_heads][page][dim], then its values as
[kv_heads][dim][page], turned so that a value's neighbours in memory are the next tokens'.

Where `own` is false, run() computes the operators from elementary torch operations; where it is
true it calls HipEngine on the same tensors' memory; its outputs are whole, to other streams than
the engine's, after a synchronization of the device.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a 135M-parameter model's token, f32 throughout: launch bound
        {"name": "rope token 9/3x64", "kind": "rope", "type": "f32", "tokens": 1, "heads": 9, "kv": 3, "dim": 64,
         "rot": 64, "layout": "pairs", "factors": False, "past": 700, "page": 16},
        # a decode batch of a 70B-shaped model at far positions, frequencies scaled for them
        {"name": "rope batch 61 64/8x128", "kind": "rope", "type": "bf16", "tokens": 61, "heads": 64, "kv": 8,
         "dim": 128, "rot": 128, "layout": "halves", "factors": True, "past": 120000, "page": 64},
        # a prompt of a mixture-of-experts model's layer, part of each head turned
        {"name": "rope prompt 2048 32/4x128", "kind": "rope", "type": "f16", "tokens": 2048, "heads": 32, "kv": 4,
         "dim": 128, "rot": 64, "layout": "halves", "factors": False, "past": 0, "page": 64},
        # five forks of a short conversation, one layer
        {"name": "pages fork 5", "kind": "pages", "type": "f32", "kv": 3, "dim": 64, "page": 16, "n_pages": 300,
         "layers": 1, "pairs": 5, "fork": True},
        # a cache made dense again, all layers of one type of page
        {"name": "pages compact 40x16", "kind": "pages", "type": "bf16", "kv": 8, "dim": 128, "page": 64,
         "n_pages": 96, "layers": 16, "pairs": 40, "fork": False},
        # a short prompt of the 135M-parameter model
        {"name": "prompt 30 9/3x64", "kind": "prompt", "type": "f32", "tokens": 30, "seqs": 1, "past": 0,
         "heads": 9, "kv": 3, "dim": 64, "page": 16},
        # ragged prompts of an 8B-shaped model in one pass
        {"name": "prompt 7 packed 2051 32/8x128", "kind": "prompt", "type": "bf16", "tokens": 2051, "seqs": 7,
         "past": 0, "heads": 32, "kv": 8, "dim": 128, "page": 64},
        # a long document, 70B-shaped
        {"name": "prompt 8192 64/8x128", "kind": "prompt", "type": "bf16", "tokens": 8192, "seqs": 1, "past": 0,
         "heads": 64, "kv": 8, "dim": 128, "page": 128},
        # a short question behind a long cached document
        {"name": "prompt 45 behind 16000 32/8x128", "kind": "prompt", "type": "f16", "tokens": 45, "seqs": 1,
         "past": 16000, "heads": 32, "kv": 8, "dim": 128, "page": 32},
        # one conversation's next token
        {"name": "decode 1 of 4000 32/8x128", "kind": "decode", "type": "f16", "seqs": 1, "prefix": 0,
         "past": 4000, "heads": 32, "kv": 8, "dim": 128, "page": 64},
        # requests that share a long instruction
        {"name": "decode 64 of 8192+500 32/8x128", "kind": "decode", "type": "bf16", "seqs": 64, "prefix": 8192,
         "past": 500, "heads": 32, "kv": 8, "dim": 128, "page": 64},
        # many small conversations behind a shorter one, f32
        {"name": "decode 250 of 1000+90 9/3x64", "kind": "decode", "type": "f32", "seqs": 250, "prefix": 1000,
         "past": 90, "heads": 9, "kv": 3, "dim": 64, "page": 16},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "pages", "prompt", "decode"])
    case = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256]),
            "kv": rng.choice([1, 2, 3, 4, 8]), "dim": rng.choice([64, 64, 72, 80, 96, 128, 128, 128, 256])}
    heads = case["kv"] * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if kind == "rope":
        case.update(heads=heads, tokens=_spread(rng, 1, 4096), rot=case["dim"] // rng.choice([1, 1, 2]),
                    layout=rng.choice(["halves", "pairs"]), factors=rng.random() < 0.5, past=_spread(rng, 1, 200000))
    elif kind == "pages":
        layers, n_pages = _spread(rng, 1, 16), _spread(rng, 8, 200)
        case.update(layers=layers, n_pages=n_pages, fork=rng.random() < 0.5)
        size = 2 * case["kv"] * case["dim"] * case["page"] * 4 * layers
        case["pairs"] = _spread(rng, 1, max(1, min(n_pages // 2 - 1, (160 << 20) // size)))
    elif kind == "prompt":
        seqs = _spread(rng, 1, 16)
        past = _spread(rng, 1, min(20000, (24 << 20) // (case["kv"] * case["dim"] * seqs))) if rng.random() < 0.4 else 0
        pairs = 2.0e11 / (4 * case["dim"] * heads)  # of a token and a key that it sees
        tokens = max(seqs, _spread(rng, 1, max(1, min(6000, int(pairs / (past + 1000))))))
        case.update(heads=heads, past=past, tokens=tokens, seqs=seqs)
    else:
        keys = (96 << 20) // (case["kv"] * case["dim"] * 2)
        seqs = _spread(rng, 1, 256)
        prefix = _spread(rng, 16, min(16000, keys // 2)) if rng.random() < 0.7 else 0
        case.update(heads=heads, seqs=seqs, prefix=prefix, past=_spread(rng, 1, min(32000, max(1, keys // 2 // seqs))))
    return case


def _parts(total, n, salt):
    """n whole numbers of 1 at least that add up to total, ragged."""
    rng = random.Random(salt * 1000003 + total * 31 + n)
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence."""
    if case["kind"] == "prompt":
        new = _parts(case["tokens"], case["seqs"], 1)
        old = [0] * case["seqs"] if not case["past"] else _parts(case["past"] * case["seqs"], case["seqs"], 2)
        return new, [a + b for a, b in zip(new, old)]
    rest = _parts(case["past"] * case["seqs"], case["seqs"], 3)
    return [1] * case["seqs"], [case["prefix"] + n for n in rest]


# ------------------------------------------------------------------------------- inputs


def _page_size(case):
    return 2 * case["kv"] * case["dim"] * case["page"]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dtype, dim, page = case["kind"], TYPES[case["type"]], case["dim"], case["page"]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def shuffled(n):
        return torch.randperm(n, device="cuda", generator=g)

    if kind == "rope":
        t, heads, kv = case["tokens"], case["heads"], case["kv"]
        # one product's rows: queries, keys, values
        state["qkv"] = normal(t, (heads + 2 * kv) * dim).to(dtype)
        state["out"] = torch.empty(t, heads * dim, device="cuda", dtype=dtype)
        if t > 256:  # a prompt: consecutive positions in whole pages
            pages = -(-t // page) + 3
            state["positions"] = ints(case["past"]) + torch.arange(t, device="cuda", dtype=torch.int32)
            at = torch.arange(t, device="cuda")
            state["slots"] = (shuffled(pages)[at // page] * page + at % page).int()
        else:  # one token each of t sequences
            pages = t + 3
            state["positions"] = torch.randint(0, case["past"] + 1, (t,), device="cuda", generator=g).int()
            state["slots"] = (shuffled(pages)[:t] * page + torch.randint(0, page, (t,), device="cuda", generator=g)).int()
        state["cache"] = normal(pages, _page_size(case)).to(dtype)
        if case["factors"]:  # slow turns are slowed down eightfold, fast ones are left alone
            x = torch.linspace(-4, 4, case["rot"] // 2, device="cuda")
            state["factors"] = 1 + 7 * torch.sigmoid(2 * x)
    elif kind == "pages":
        n, k = case["n_pages"], case["pairs"]
        state["cache"] = torch.empty(case["layers"], n, _page_size(case), device="cuda", dtype=dtype)
        for layer in state["cache"]:
            layer.copy_(normal(n, _page_size(case)))
        at = shuffled(n).int()
        # forks copy few pages to many, a denser cache moves each page once
        source = at[torch.randint(0, max(1, k // 4), (k,), device="cuda", generator=g)] if case["fork"] else at[:k]
        state["moves"] = torch.stack([source, at[-k:]], 1).contiguous()
    else:
        heads, kv = case["heads"], case["kv"]
        new, lens = _lengths(case)
        prefix = case.get("prefix", 0)
        shared = prefix // page  # whole pages are shared
        own_pages = [-(-n // page) - shared for n in lens]
        ids = shuffled(shared + sum(own_pages) + 2).int()
        state["shared"] = ids[:-(-prefix // page)].contiguous()
        wide = max(shared + n for n in own_pages)
        state["tables"] = torch.full((len(lens), wide), -1, dtype=torch.int32, device="cuda")
        at = shared
        for s, n in enumerate(own_pages):
            state["tables"][s, :shared] = ids[:shared]
            state["tables"][s, shared:shared + n] = ids[at:at + n]
            at += n
        # keys have channels larger than the others; what is not in use is left from earlier requests
        cache = normal(len(ids), _page_size(case)).mul_(0.8)
        keys = cache[:, :_page_size(case) // 2].view(len(ids), kv, page, dim)
        keys.mul_(torch.exp(0.4 * normal(kv, 1, dim)))
        state["cache"] = cache.to(dtype)
        if prefix % page:  # the page that the prefix ends in: each sequence has its own copy of those tokens
            mine = state["tables"][:, shared].long()
            end = prefix % page
            half = _page_size(case) // 2
            k = state["cache"][:, :half].view(-1, kv, page, dim)
            v = state["cache"][:, half:].view(-1, kv, dim, page)
            k[mine, :, :end] = k[mine[0], :, :end].clone()
            v[mine, :, :, :end] = v[mine[0], :, :, :end].clone()
            state["shared"][shared] = mine[0].int()
        state["q"] = (1.2 * normal(sum(new), heads * dim)).to(dtype)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["starts"], state["lens"] = ints(starts), ints(lens)
        state["out"] = torch.empty_like(state["q"])
    return state


# -------------------------------------------------------------------------- plain forms

BASE = 500000.0


def _plain_rope(state):
    case, x = state["case"], state["qkv"].float()
    t, heads, kv, dim, rot = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"]
    i = torch.arange(rot // 2, device=x.device, dtype=torch.float64)
    turn = BASE ** (-2.0 * i / rot)
    if case["factors"]:
        turn = turn / state["factors"].double()
    angle = state["positions"].double().unsqueeze(1) * turn  # 64 bits: far positions
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    x = x.view(t, heads + 2 * kv, dim)
    turned = x[:, :heads + kv].clone()
    if case["layout"] == "halves":
        a, b = x[:, :heads + kv, :rot // 2], x[:, :heads + kv, rot // 2:rot]
        turned[..., :rot // 2], turned[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[:, :heads + kv, 0:rot:2], x[:, :heads + kv, 1:rot:2]
        turned[..., 0:rot:2], turned[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    dtype, half = state["cache"].dtype, _page_size(case) // 2
    k = state["cache"][:, :half].view(-1, kv, case["page"], dim)
    v = state["cache"][:, half:].view(-1, kv, dim, case["page"])
    page, at = (state["slots"] // case["page"]).long(), (state["slots"] % case["page"]).long()
    k[page, :, at] = turned[:, heads:].to(dtype)
    v[page, :, :, at] = x[:, heads + kv:].to(dtype)
    state["out"].copy_(turned[:, :heads].reshape(t, -1))
    return {"q": state["out"], "cache": state["cache"]}


def _plain_pages(state):
    moves = state["moves"].long()
    state["cache"][:, moves[:, 1]] = state["cache"][:, moves[:, 0]]
    return state["cache"]


def _plain_attention(state):
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    half = _page_size(case) // 2
    keys = state["cache"][:, :half].view(-1, kv, page, dim)
    values = state["cache"][:, half:].view(-1, kv, dim, page)
    new, lens = _lengths(case)
    at = 0
    for s, (n, length) in enumerate(zip(new, lens)):
        pages = state["tables"][s, :-(-length // page)].long()
        k = keys[pages].permute(1, 3, 0, 2).reshape(kv, dim, -1)[:, :, :length].float().contiguous()
        v = values[pages].permute(1, 0, 3, 2).reshape(kv, -1, dim)[:, :length].float().contiguous()
        for t in range(0, n, 512):  # a block of tokens: their scores are held whole
            m = min(512, n - t)
            q = state["q"][at + t:at + t + m].float().view(m, kv, heads // kv, dim)
            q = q.permute(1, 2, 0, 3).reshape(kv, -1, dim).contiguous()
            scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).view(kv, heads // kv, m, length)
            if n > 1:
                last = length - n + t + torch.arange(m, device=q.device).unsqueeze(1)
                scores.masked_fill_(torch.arange(length, device=q.device) > last, float("-inf"))
            scores = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
            total = scores.sum(-1, keepdim=True)
            out = torch.matmul(scores.view(kv, -1, length), v).view(kv, heads // kv, m, dim) / total
            state["out"][at + t:at + t + m] = out.permute(2, 0, 1, 3).reshape(m, -1)
        at += n
    return state["out"]


# ------------------------------------------------------------------ the framework's calls

_engine = None


def _buffers(state):
    """Handles on the tensors' memory, kept with them as a program keeps them."""
    global _engine
    import hayai_amd
    if _engine is None:
        _engine = hayai_amd.HipEngine(0)
    case, e = state["case"], _engine
    ty = {"f32": hayai_amd.F32, "f16": hayai_amd.F16, "bf16": hayai_amd.BF16}[case["type"]]
    state["handles"] = h = {k: e.wrap(v.data_ptr(), v.numel() * v.element_size())
                            for k, v in state.items() if isinstance(v, torch.Tensor) and v.numel()}
    kind, cache = case["kind"], state["cache"]
    n_pages = cache.shape[-2]
    h["kv"] = e.kv_desc(ty, case["kv"], case["dim"], case["page"], n_pages)
    if kind == "rope":
        wide = (case["heads"] + 2 * case["kv"]) * case["dim"]
        h["desc"] = e.rope_desc(ty, case["tokens"], case["heads"], case["rot"], BASE, q_stride=wide, k_stride=wide,
                                v_stride=wide, layout=hayai_amd.ROPE_HALVES if case["layout"] == "halves"
                                else hayai_amd.ROPE_PAIRS)
    elif kind == "prompt":
        h["desc"] = e.attn_prompt_desc(ty, case["tokens"], case["seqs"], case["heads"], 1.0 / math.sqrt(case["dim"]),
                                       state["tables"].shape[1])
    elif kind == "decode":
        h["desc"] = e.attn_decode_desc(ty, case["seqs"], case["heads"], 1.0 / math.sqrt(case["dim"]),
                                       state["tables"].shape[1], prefix=case["prefix"])
    # the engine's stream does not wait for torch's: the inputs are whole before its first call
    torch.cuda.synchronize()
    return h


def _own(state):
    h = state.get("handles") or _buffers(state)
    case, e = state["case"], _engine
    kind = case["kind"]
    if kind == "rope":
        size = state["qkv"].element_size()
        k_off, v_off = case["heads"] * case["dim"] * size, (case["heads"] + case["kv"]) * case["dim"] * size
        e.rope_kv_dev(h["desc"], h["kv"], h["qkv"], 0, h["qkv"], k_off, h["qkv"], v_off, h["positions"], 0, h["slots"], 0,
                      h.get("factors"), 0, h["out"], 0, h["cache"], 0)
        return {"q": state["out"], "cache": state["cache"]}
    if kind == "pages":
        e.kv_copy_dev(h["kv"], h["cache"], 0, h["moves"], 0, case["pairs"], layers=case["layers"])
        return state["cache"]
    if kind == "prompt":
        e.attn_prompt_dev(h["desc"], h["kv"], h["q"], 0, h["cache"], 0, h["starts"], 0, h["lens"], 0, h["tables"], 0,
                          h["out"], 0)
    else:
        e.attn_decode_dev(h["desc"], h["kv"], h["q"], 0, h["cache"], 0, h.get("shared"), 0, h["lens"], 0, h["tables"], 0,
                          h["out"], 0)
    return state["out"]


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "pages": _plain_pages, "prompt": _plain_attention,
            "decode": _plain_attention}[state["case"]["kind"]](state)


def work(case):
    size, kind = 4 if case["type"] == "f32" else 2, case["kind"]
    if kind == "pages":
        reads = max(1, case["pairs"] // 4) if case["fork"] else case["pairs"]
        return {"bytes": (reads + case["pairs"]) * case["layers"] * _page_size(case) * size, "flops": 0}
    if kind == "rope":
        wide = (case["heads"] + 2 * case["kv"]) * case["dim"]
        return {"bytes": case["tokens"] * (2 * wide * size + 8), "flops": case["tokens"] * wide * 3}
    new, lens = _lengths(case)
    token, row = 2 * case["kv"] * case["dim"] * size, 2 * case["heads"] * case["dim"] * size
    prefix = case.get("prefix", 0)
    seen = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lens))
    return {"bytes": (prefix + sum(length - prefix for length in lens)) * token + sum(new) * row,
            "flops": 4 * case["heads"] * case["dim"] * seen}


# ------------------------------------------------------------- the definitions in 64 bits


def _exact_rope(case, state):
    t, heads, kv, dim, rot, page = (case[k] for k in ("tokens", "heads", "kv", "dim", "rot", "page"))
    x = state["qkv"].double().reshape(t, -1, dim)
    pair = torch.arange(rot // 2, device=x.device)
    first = pair if case["layout"] == "halves" else 2 * pair
    second = pair + rot // 2 if case["layout"] == "halves" else 2 * pair + 1
    turn = torch.exp(pair.double() * (-2.0 * math.log(BASE) / rot))
    if case["factors"]:
        turn = turn / state["factors"].double()
    unit = torch.polar(torch.ones(t, 1, rot // 2, device=x.device, dtype=torch.float64),
                       torch.outer(state["positions"].double(), turn).unsqueeze(1))
    z = torch.complex(x[:, :heads + kv][..., first], x[:, :heads + kv][..., second]) * unit
    x[:, :heads + kv, first], x[:, :heads + kv, second] = z.real.contiguous(), z.imag.contiguous()
    cache, slots = state["cache"].double(), state["slots"].tolist()
    half = cache.shape[1] // 2
    for i, slot in enumerate(slots):
        p, at = divmod(slot, page)
        cache[p, :half].view(kv, page, dim)[:, at] = x[i, heads:heads + kv]
        cache[p, half:].view(kv, dim, page)[:, :, at] = x[i, heads + kv:]
    return {"q": x[:, :heads].reshape(t, -1), "cache": cache}


def _exact_attention(case, state):
    heads, kv, dim, page = (case[k] for k in ("heads", "kv", "dim", "page"))
    new, lens = _lengths(case)
    if 4 * heads * dim * sum(n * length for n, length in zip(new, lens)) > 4e12:
        return None
    out = torch.empty_like(state["q"], dtype=torch.float64)
    half, row = _page_size(case) // 2, 0
    for s, (n, length) in enumerate(zip(new, lens)):
        where = torch.arange(length, device=out.device)
        pages, at = state["tables"][s].long()[where // page], where % page
        keys = state["cache"][:, :half].view(-1, kv, page, dim)[pages, :, at].double()  # length, kv, dim
        values = state["cache"][:, half:].view(-1, kv, dim, page)[pages, :, :, at].double()
        for t in range(0, n, 256):
            m = min(256, n - t)
            q = state["q"][row + t:row + t + m].double().view(m, heads, dim)
            visible = where.unsqueeze(0) <= length - n + t + torch.arange(m, device=out.device).unsqueeze(1)
            for h in range(heads):
                k, v = keys[:, h // (heads // kv)], values[:, h // (heads // kv)]
                score = torch.where(visible, torch.mm(q[:, h], k.t()) / math.sqrt(dim), -math.inf)
                out[row + t:row + t + m, h * dim:(h + 1) * dim] = torch.mm(torch.softmax(score, 1), v)
        row += n
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, state)
    if case["kind"] == "pages":
        cache = state["cache"].double()
        for source, target in state["moves"].tolist():
            cache[:, target] = cache[:, source]
        return cache
    return _exact_attention(case, state)
