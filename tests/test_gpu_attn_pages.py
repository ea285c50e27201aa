"""GPU tests of the cache's entry points: rotary positions into the cache (rope_kv) and copies of its
pages (kv_copy), against their definitions in 64 bits.

A turned element is a cos - b sin with cos and sin rounded to f32 once (2^-24 each, times mscale), one
product, one fused multiply-add: off by less than (|a| + |b|) * 2^-24 * 4, then one rounding to the
output's type (eps / 2 of the value).  What only goes through is rounded once.
"""
import numpy as np
import pytest
import torch

import hayai_amd
from hayai_amd import BF16, F16, F32, ROPE_HALVES, ROPE_PAIRS

pytestmark = pytest.mark.gpu

DT = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]


def normal(seed, *shape, scale=1.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape) * scale)


def put(engine, t, lead=0):
    t = t.contiguous()
    raw = t.view(torch.uint8).numpy().reshape(-1) if t.numel() else np.zeros(0, np.uint8)
    b = engine.alloc(max(lead + raw.size, 1))
    if raw.size:
        b.write(raw, lead)
    return b


def ints(engine, values, lead=0):
    return put(engine, torch.tensor(values, dtype=torch.int32), lead)


def get(b, dtype, shape, lead=0):
    n = int(np.prod(shape))
    if n == 0:
        return torch.empty(shape, dtype=dtype)
    raw = b.read(np.uint8, n * torch.empty(0, dtype=dtype).element_size(), lead)
    return torch.from_numpy(raw).view(dtype).reshape(shape)


def turned(x, positions, rot, base, layout, factors, mscale):
    """x: (tokens, heads, dim) in 64 bits."""
    y = x.clone()
    i = np.arange(rot // 2)
    w = base ** (-2.0 * i / max(rot, 1))
    if factors is not None:
        w = w / factors.astype(np.float64)
    angle = torch.from_numpy(np.outer(positions.astype(np.float64), w))[:, None, :]
    c, s = torch.cos(angle) * mscale, torch.sin(angle) * mscale
    a_at, b_at = (i, i + rot // 2) if layout == ROPE_HALVES else (2 * i, 2 * i + 1)
    a, b = x[..., a_at], x[..., b_at]
    y[..., a_at], y[..., b_at] = a * c - b * s, a * s + b * c
    return y


def near(got, want, dtype, slack):
    err = (got.double() - want).abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # a step below the normal range
    bound = slack * (1 + torch.finfo(dtype).eps) + want.abs() * torch.finfo(dtype).eps / 2 + tiny
    assert torch.all(err <= bound), (err / bound).max()


# tokens, q heads, kv heads, dim, rot, page, strides beyond a row, byte lead
SHAPES = [(1, 9, 3, 64, 64, 16, 0, 0), (1, 32, 8, 128, 128, 64, 0, 0), (5, 4, 4, 72, 36, 32, 3, 4), (3, 0, 1, 8, 0, 16, 0, 0),
          (61, 8, 1, 128, 64, 64, 0, 0), (7, 3, 1, 80, 80, 256, 1, 8), (2, 2, 2, 256, 256, 128, 5, 4),
          (300, 6, 2, 40, 2, 16, 0, 0), (2, 64, 8, 96, 18, 64, 0, 0)]


@pytest.mark.parametrize("layout", [ROPE_HALVES, ROPE_PAIRS])
@pytest.mark.parametrize("ty,cty", TYPES)
def test_rope(engine, ty, cty, layout):
    for case, (t, heads, kvh, dim, rot, page, pad, lead) in enumerate(SHAPES):
        print(f"[case] rope {ty} {cty} {layout} {SHAPES[case]}", flush=True)
        rng = np.random.default_rng(case)
        el = torch.empty(0, dtype=DT[ty]).element_size()
        lead = lead // el * el
        cols, base, mscale = (heads + 2 * kvh) * dim, 10000.0, float(np.float32([1.0, 1.25][case % 2]))
        x = normal(case, t, cols + pad, scale=2.0).to(DT[ty])
        n_pages = t // page + 3
        # far positions, negative ones, slots outside the cache
        positions = rng.integers(-3, [200, 200000, 2**31 - 1][case % 3], t).astype(np.int32)
        slots = rng.permutation(n_pages * page)[:t].astype(np.int32)
        if t > 2:
            slots[1], slots[2] = -1, n_pages * page
        factors = (1 + 7 * rng.random(rot // 2)).astype(np.float32) if case % 2 and rot else None
        per = 2 * kvh * page * dim
        stride = per + (16 if case % 2 else 0)
        cache = normal(case + 100, n_pages, stride).to(DT[cty])
        xb, cb = put(engine, x, lead), put(engine, cache)
        out = put(engine, torch.full((t, heads * dim + pad), 9.0).to(DT[ty]), lead)
        pb, sb = ints(engine, positions.tolist(), 4), ints(engine, slots.tolist())
        fb = None if factors is None else put(engine, torch.from_numpy(factors))
        d = engine.rope_desc(ty, t, heads, rot, base, q_stride=cols + pad, k_stride=cols + pad, v_stride=cols + pad,
                             out_stride=heads * dim + pad, layout=layout, mscale=mscale)
        kv = engine.kv_desc(cty, kvh, dim, page, n_pages, stride if case % 2 else 0)
        engine.rope_kv_dev(d, kv, xb if heads else None, lead, xb, lead + heads * dim * el, xb,
                           lead + (heads + kvh) * dim * el, pb, 4, sb, 0, fb, 0, out if heads else None, lead, cb, 0)
        x64 = x[:, :cols].double().reshape(t, heads + 2 * kvh, dim)
        want = turned(x64[:, :heads + kvh], positions, rot, base, layout, factors, mscale)
        # the two products' and their sum's roundings: |a| + |b| of a pair, at most sqrt(2) of its length
        size = (x64[:, :heads + kvh] ** 2).sum(-1, keepdim=True).sqrt().expand_as(want) * 1.5 * mscale * 4 * 2.0**-24
        size[..., rot:] = 0
        got = get(out, DT[ty], (t, heads * dim + pad), lead)
        near(got[:, :heads * dim].reshape(t, heads, dim), want[:, :heads], DT[ty], size[:, :heads])
        assert torch.all(got[:, heads * dim:] == 9.0)
        new = get(cb, DT[cty], (n_pages, stride))
        expect, slack = cache.double().clone(), torch.zeros(n_pages, stride, dtype=torch.float64)
        for i, slot in enumerate(slots.tolist()):
            if not 0 <= slot < n_pages * page:
                continue
            p, at = divmod(slot, page)
            expect[p, :per // 2].view(kvh, page, dim)[:, at] = want[i, heads:]
            slack[p, :per // 2].view(kvh, page, dim)[:, at] = size[i, heads:]
            expect[p, per // 2:per].view(kvh, dim, page)[:, :, at] = x64[i, heads + kvh:]
        near(new, expect, DT[cty], slack)
        untouched = torch.ones(n_pages, stride, dtype=torch.bool)
        for slot in slots.tolist():
            if 0 <= slot < n_pages * page:
                p, at = divmod(slot, page)
                untouched[p, :per // 2].view(kvh, page, dim)[:, at] = False
                untouched[p, per // 2:per].view(kvh, dim, page)[:, :, at] = False
        assert torch.equal(new[untouched], cache[untouched])


@pytest.mark.parametrize("layout", [ROPE_HALVES, ROPE_PAIRS])
@pytest.mark.parametrize("ty,cty", TYPES)
def test_rope_prompt(engine, ty, cty, layout):
    """Enough tokens for several of them a workgroup: runs of slots, runs that a page ends, slots of nobody's, a
    rest of less than eight."""
    t, heads, kvh, dim, rot, page = 8 * engine.device_info.compute_units + 13, 3, 2, 72, 44, 16
    rng = np.random.default_rng(21)
    x = normal(22, t, (heads + 2 * kvh) * dim).to(DT[ty])
    n_pages = t // page + 40
    slots = np.arange(t, dtype=np.int32) + page * 3
    slots[200:900] = rng.permutation(np.arange(page * 3 + 200, page * 3 + 900))
    slots[1000:1200] += 3  # runs that do not begin at a multiple of eight
    slots[1200:1203] = -1
    slots[1400:] += 64
    positions = rng.integers(0, 100000, t).astype(np.int32)
    el, wide = torch.empty(0, dtype=DT[ty]).element_size(), x.shape[1]
    per = 2 * kvh * page * dim
    cache = normal(23, n_pages, per).to(DT[cty])
    xb, cb, out = put(engine, x), put(engine, cache), engine.alloc(t * heads * dim * el)
    d = engine.rope_desc(ty, t, heads, rot, 10000.0, q_stride=wide, k_stride=wide, v_stride=wide, layout=layout)
    engine.rope_kv_dev(d, engine.kv_desc(cty, kvh, dim, page, n_pages), xb, 0, xb, heads * dim * el, xb,
                       (heads + kvh) * dim * el, ints(engine, positions.tolist()), 0, ints(engine, slots.tolist()), 0, None, 0,
                       out, 0, cb, 0)
    x64 = x.double().reshape(t, heads + 2 * kvh, dim)
    want = turned(x64[:, :heads + kvh], positions, rot, 10000.0, layout, None, 1.0)
    size = (x64[:, :heads + kvh] ** 2).sum(-1, keepdim=True).sqrt().expand_as(want) * 1.5 * 4 * 2.0**-24
    size[..., rot:] = 0
    near(get(out, DT[ty], (t, heads, dim)), want[:, :heads], DT[ty], size[:, :heads])
    expect, slack = cache.double().clone(), torch.zeros(n_pages, per, dtype=torch.float64)
    keep = np.nonzero(slots >= 0)[0]
    p, at = torch.from_numpy(slots[keep] // page).long(), torch.from_numpy(slots[keep] % page).long()
    expect[:, :per // 2].view(-1, kvh, page, dim)[p, :, at] = want[keep, heads:]
    slack[:, :per // 2].view(-1, kvh, page, dim)[p, :, at] = size[keep, heads:]
    expect[:, per // 2:].view(-1, kvh, dim, page)[p, :, :, at] = x64[keep, heads + kvh:]
    new = get(cb, DT[cty], (n_pages, per))
    near(new, expect, DT[cty], slack)
    assert torch.equal(new[:3], cache[:3])


def test_rope_more_tokens_than_a_launch(engine):
    t, dim, page = (1 << 20) + 11, 8, 256
    n_pages = t // page + 1
    x = torch.from_numpy(np.random.default_rng(30).standard_normal((t, 3 * dim), dtype=np.float32)).half()
    xb, cb, out = put(engine, x), engine.alloc(n_pages * 2 * page * dim * 2), engine.alloc(t * dim * 2)
    cb.fill(0)
    order = np.arange(t, dtype=np.int32)
    d = engine.rope_desc(F16, t, 1, dim, q_stride=3 * dim, k_stride=3 * dim, v_stride=3 * dim)
    engine.rope_kv_dev(d, engine.kv_desc(F16, 1, dim, page, n_pages), xb, 0, xb, 2 * dim, xb, 4 * dim, engine.upload(order % 1000), 0,
                       engine.upload(order), 0, None, 0, out, 0, cb, 0)
    at = np.r_[0:50, (1 << 20) - 20:t]
    x64 = x[at].double().reshape(len(at), 3, dim)
    want = turned(x64[:, :2], at % 1000, dim, 10000.0, ROPE_HALVES, None, 1.0)
    size = (x64[:, :2] ** 2).sum(-1, keepdim=True).sqrt().expand_as(want) * 6 * 2.0**-24
    near(get(out, torch.float16, (t, 1, dim))[at], want[:, :1], torch.float16, size[:, :1])
    cache = get(cb, torch.float16, (n_pages, 2, page * dim))
    near(cache[:, 0].reshape(-1, dim)[at], want[:, 1], torch.float16, size[:, 1])
    assert torch.equal(cache[:, 1].reshape(n_pages, dim, page).permute(0, 2, 1).reshape(-1, dim)[:t], x[:, 2 * dim:])


def test_rope_in_place(engine):
    heads, kvh, dim, page = 12, 2, 128, 16
    for layout, t in ((ROPE_HALVES, 130), (ROPE_PAIRS, 130), (ROPE_HALVES, 2500), (ROPE_PAIRS, 2500)):
        x = normal(7, t, (heads + 2 * kvh) * dim).to(torch.bfloat16)
        outs = []
        for in_place in (False, True):
            xb, cb = put(engine, x), engine.alloc(160 * 2 * kvh * page * dim * 2)
            cb.fill(0)
            out = xb if in_place else engine.alloc(x.numel() * 2)
            wide = x.shape[1]
            d = engine.rope_desc(BF16, t, heads, dim, q_stride=wide, k_stride=wide, v_stride=wide, out_stride=wide, layout=layout)
            kv = engine.kv_desc(BF16, kvh, dim, page, 160)
            engine.rope_kv_dev(d, kv, xb, 0, xb, heads * dim * 2, xb, (heads + kvh) * dim * 2, ints(engine, list(range(t))), 0,
                               ints(engine, list(range(t))), 0, None, 0, out, 0, cb, 0)
            outs.append((get(out, torch.bfloat16, (t, wide))[:, :heads * dim], get(cb, torch.bfloat16, (160, 2 * kvh * page * dim))))
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def copied(cache, moves, n_pages, per):
    out = cache.copy()
    for s, d in moves:
        if 0 <= s < n_pages and 0 <= d < n_pages:
            out[:, d, :per] = out[:, s, :per]
    return out


# heads, dim, page, pages, layers, moves: few and many, in layers enough to keep all in one part or not
COPIES = [(1, 8, 16, 2, 1, 1), (3, 64, 16, 300, 1, 5), (8, 128, 64, 20, 2, 9), (2, 72, 32, 50, 3, 100), (1, 64, 16, 40, 5, 257),
          (8, 256, 256, 6, 4, 3), (1, 8, 16, 300000, 1, 40)]


@pytest.mark.parametrize("kind", ["forks", "holes", "chain", "any"])
def test_kv_copy(engine, kind):
    for case, (kvh, dim, page, n_pages, layers, n) in enumerate(COPIES):
        print(f"[case] kv_copy {kind} {COPIES[case]}", flush=True)
        rng = np.random.default_rng(case)
        at = rng.permutation(n_pages)
        if kind in ("forks", "holes"):
            n = min(n, n_pages // 2)
            source = at[rng.integers(0, max(1, n // 3), n)] if kind == "forks" else at[:n]
            moves = np.stack([source, at[n_pages - n:]], 1)
        elif kind == "chain":  # every page one down, the first to the end
            n = min(n, n_pages - 1)
            moves = np.stack([np.arange(1, n + 1), np.arange(n)], 1)
        else:  # pages twice, pages outside, padding
            moves = rng.integers(-2, min(n_pages, 12) + 2, (n, 2))
            moves[moves >= min(n_pages, 12)] += n_pages
            moves = np.concatenate([moves, [[-1, -1], [0, -1], [-1, 0]]])
        per = 2 * kvh * dim * page
        stride = per + 8 * (case % 3)
        cache = rng.integers(0, 1 << 16, (layers, n_pages, stride), dtype=np.uint16)
        b = engine.upload(cache)
        kv = engine.kv_desc(F16, kvh, dim, page, n_pages, stride)
        engine.kv_copy_dev(kv, b, 0, engine.upload(moves.astype(np.int32)), 0, len(moves), layers=layers)
        assert np.array_equal(b.read(np.uint16, cache.size).reshape(cache.shape), copied(cache, moves.tolist(), n_pages, per))


def test_kv_copy_layers_between_pages(engine):
    """page_stride leaves room for the layers: layer l's pages begin one page further."""
    kvh, dim, page, n_pages, layers = 2, 64, 16, 12, 3
    per = 2 * kvh * dim * page
    cache = np.random.default_rng(0).integers(0, 1 << 16, (n_pages, layers, per), dtype=np.uint16)
    b = engine.upload(cache)
    kv = engine.kv_desc(BF16, kvh, dim, page, n_pages, layers * per)
    moves = [(3, 1), (1, 2), (11, 0)]
    engine.kv_copy_dev(kv, b, 0, engine.upload(np.array(moves, np.int32)), 0, 3, layers=layers, layer_stride=per)
    want = np.ascontiguousarray(copied(cache.transpose(1, 0, 2), moves, n_pages, per).transpose(1, 0, 2))
    assert np.array_equal(b.read(np.uint16, cache.size).reshape(cache.shape), want)


def test_no_tokens_no_moves(engine):
    b = engine.alloc(1 << 16)
    b.fill(0x5B)
    kv = engine.kv_desc(F16, 1, 64, 16, 2)
    engine.kv_copy_dev(kv, b, 0, b, 0, 0)
    engine.rope_kv_dev(engine.rope_desc(F16, 0, 1, 64), kv, b, 0, b, 0, b, 0, b, 0, b, 0, None, 0, b, 0, b, 0)
    assert np.all(b.read(np.uint8, 1 << 16) == 0x5B)


def test_refusals(engine):
    b, small = engine.alloc(1 << 16), engine.alloc(8)
    kv = engine.kv_desc(F16, 2, 64, 16, 2)
    good = dict(ggml_type=F16, tokens=4, q_heads=4, rot_dim=64)

    def rope(kv=kv, q=b, k=b, slots=b, factors=None, out=b, cache=b, cache_off=0, **changes):
        engine.rope_kv_dev(engine.rope_desc(**{**good, **changes}), kv, q, 0, k, 0, b, 0, b, 0, slots, 0, factors, 0, out, 0, cache,
                           cache_off)

    rope()
    for status, changes in [(3, dict(ggml_type=2)), (3, dict(ggml_type=BF16)), (3, dict(kv=engine.kv_desc(F32, 2, 64, 16, 1))),
                            (2, dict(layout=2)), (2, dict(rot_dim=66)), (2, dict(rot_dim=3)), (2, dict(base=0.0)),
                            (2, dict(base=float("inf"))), (2, dict(base=float("nan"))), (2, dict(mscale=float("inf"))),
                            (2, dict(q_heads=65536)), (2, dict(tokens=1 << 40)), (2, dict(tokens=1 << 14)), (2, dict(q_stride=255)),
                            (2, dict(k_stride=127)), (2, dict(v_stride=127)), (2, dict(out_stride=255)), (2, dict(q=None)),
                            (2, dict(out=None)), (2, dict(k=small)), (2, dict(slots=small)), (2, dict(factors=small)),
                            (2, dict(cache=small)), (2, dict(cache_off=2)), (2, dict(cache_off=1 << 16)),
                            (2, dict(kv=engine.kv_desc(F16, 1025, 64, 16, 2)))]:
        with pytest.raises(hayai_amd.HipError) as err:
            rope(**changes)
        assert err.value.status == status, changes
    engine.kv_copy_dev(kv, b, 0, small, 0, 1)
    for args, kw in [((kv, b, 0, small, 0, 2), {}), ((kv, b, 0, small, 0, 1), dict(layers=0)), ((kv, b, 0, small, 0, 1), dict(layers=1 << 16)),
                     ((kv, b, 0, small, 0, 1), dict(layers=9)), ((kv, b, 0, small, 0, 1), dict(layers=2, layer_stride=4)),
                     ((kv, b, 0, small, 0, 1), dict(layers=3, layer_stride=1 << 62)), ((kv, b, 0, small, 0, 1 << 40), {}),
                     ((kv, b, 0, small, 2, 1), {}), ((kv, small, 0, b, 0, 1), {})]:
        with pytest.raises(hayai_amd.HipError) as err:
            engine.kv_copy_dev(*args, **kw)
        assert err.value.status == 2, (args[2:], kw)


def test_kv_copy_layers_that_overlap(engine):
    """Layers whose pages have bytes in common are refused: their copies have no order.  Layers apart, one page's next to each other,
    and others in the gaps between pages go through."""
    kvh, dim, page = 1, 8, 16
    per = 2 * kvh * dim * page
    size = 1 << 20
    b, moves = engine.alloc(size), engine.upload(np.array([(0, 1)], np.int32))

    def elements(n, stride, layer_stride, layers):
        return [set(range(p * stride + l * layer_stride, p * stride + l * layer_stride + per)) for l in range(layers) for p in range(n)]

    refused = 0
    for n, stride, layer_stride, layers in [
            (2, per, 8, 2), (2, per, per, 2), (2, 3 * per, 2 * per + 8, 2), (2, 3 * per, per - 8, 3), (3, 2 * per, 2 * per, 2),
            (2, 2 * per, per, 3), (4, 2 * per, 3 * per - 8, 3), (1, per, per - 8, 5), (3, 5 * per, 4 * per, 4), (3, 2 * per, 6 * per - 8, 2),
            (2, per, 2 * per, 3), (2, 3 * per, per, 3), (3, 10 * per, 11 * per, 4), (1, per, per, 9), (3, 2 * per, 5 * per, 2),
            (3, 2 * per + 8, per + 8, 2), (4, 2 * per, 9 * per, 3), (3, 4 * per, 14 * per, 4)]:
        kv = engine.kv_desc(F16, kvh, dim, page, n, stride)
        parts = elements(n, stride, layer_stride, layers)
        if len(set().union(*parts)) < sum(len(p) for p in parts):
            with pytest.raises(hayai_amd.HipError) as err:
                engine.kv_copy_dev(kv, b, 0, moves, 0, 1, layers=layers, layer_stride=layer_stride)
            assert err.value.status == 2, (n, stride, layer_stride, layers)
            refused += 1
            continue
        cache = np.random.default_rng(0).integers(0, 1 << 16, size // 2, dtype=np.uint16)
        b.write(cache)
        engine.kv_copy_dev(kv, b, 0, moves, 0, 1 if n > 1 else 0, layers=layers, layer_stride=layer_stride)
        if n > 1:
            for l in range(layers):
                cache[l * layer_stride + stride:][:per] = cache[l * layer_stride:][:per]
        assert np.array_equal(b.read(np.uint16, size // 2), cache), (n, stride, layer_stride, layers)
    assert refused == 8
