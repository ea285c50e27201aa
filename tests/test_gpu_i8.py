"""GPU tests of the 8-bit path: rows into codes (quant_i8, rms_norm_i8), products of codes (gemm_i8)
and the steps together, against their definitions in 64 bits.

Codes are decided as in 64-bit arithmetic, so they have to equal the oracle's; a scale is one f32
rounding (2^-24 relative) of the 64-bit value.  A product's sum is exact; its conversion to f32, the
two scales and the residual round once each (2^-24 of the product, of the result), then the output
type (eps / 2).
"""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import hayai_amd
from hayai_amd import BF16, F16, F32

pytestmark = pytest.mark.gpu

DT = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
TYPES = [F32, F16, BF16]
EPS = float(np.float32(1e-5))  # as the descriptor holds it


def normal(seed, *shape, scale=1.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape) * scale)


def put(engine, t, lead=0):
    """A tensor's bytes on the device, `lead` bytes into a buffer."""
    t = t.contiguous()
    raw = t.view(torch.uint8).numpy().reshape(-1) if t.numel() else np.zeros(0, np.uint8)
    b = engine.alloc(lead + raw.size)
    if raw.size:
        b.write(raw, lead)
    return b


def get(b, dtype, shape, lead=0):
    n = int(np.prod(shape))
    size = torch.empty(0, dtype=dtype).element_size()
    raw = b.read(np.uint8, n * size, lead)
    return torch.from_numpy(raw).view(dtype).reshape(shape)


def f64(t):
    return t.double().numpy()


def codes_of(u, unit=1.0):
    """(codes, scale in 64 bits) of rows u; rows that are not finite: codes 0, scale NaN."""
    top = np.max(np.abs(u), axis=1, keepdims=True)
    bad = ~np.isfinite(top)
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.rint(127.0 * np.where(bad, 0.0, u) / np.where((top == 0) | bad, 1.0, top))
        scale = np.where(bad, np.nan, np.where(top == 0, 0.0, top * unit / 127.0))
    q = np.where(scale.astype(np.float32) == 0, 0, q)
    return q.astype(np.int8), scale[:, 0]


def check_codes(q, scale, values, want_q, want_scale):
    assert np.array_equal(q, want_q), f"{np.count_nonzero(q != want_q)} codes differ"
    bad = np.isnan(want_scale)
    assert np.array_equal(np.isnan(scale), bad)
    err = np.abs(scale[~bad].astype(np.float64) - want_scale[~bad])
    # half a step of f32: 2^-24 relative, or 2^-150 below its normal range; the 64-bit value itself is
    # a few 2^-53 off
    assert np.all(err <= want_scale[~bad] * 2.0**-24 * (1 + 1e-6) + 2.0**-150 * (1 + 1e-6))
    if values is not None:
        assert np.array_equal(values, q.astype(np.float32) * scale[:, None], equal_nan=True)


def act64(g, u, act):
    if act == hayai_amd.ACT_SILU:
        return g / (1.0 + np.exp(-g)) * u
    return g / (1.0 + np.exp(-2.0 * np.sqrt(2.0 / np.pi) * (g + 0.044715 * g**3))) * u


# rows, cols, extra stride elements, byte lead: one element, odd rows, whole vectors, a workgroup's edge
# (256 threads x 4 f32, 1024 x 4), rows past what stays in registers
SHAPES = [(1, 1, 0, 0), (3, 5, 1, 4), (2, 64, 0, 0), (5, 577, 3, 4), (1, 576, 0, 0), (33, 1000, 0, 0), (2, 4096, 16, 0),
          (3, 4099, 0, 4), (1, 8192, 0, 0), (2, 8195, 5, 0), (2, 16384, 0, 0), (1, 16391, 0, 4), (2, 33001, 0, 0)]


@pytest.mark.parametrize("act", [None, hayai_amd.ACT_SILU, hayai_amd.ACT_GELU_TANH])
@pytest.mark.parametrize("ty", TYPES)
def test_quant_rows(engine, ty, act):
    size = torch.empty(0, dtype=DT[ty]).element_size()
    for k, (rows, cols, pad, lead) in enumerate(SHAPES):
        print(f"[case] quant type={ty} act={act} {rows}x{cols} +{pad}", flush=True)
        stride = (cols if act is None else 2 * cols) + pad
        x = normal(k, rows, stride, scale=2.0).to(DT[ty])
        b = put(engine, x, lead)
        qs = cols + pad
        q, s, v = engine.alloc(rows * qs + 7), engine.alloc(4 * rows + 4), engine.alloc(4 * rows * cols + 4)
        for o in (q, s, v):
            o.fill(0x5B)
        d = engine.quant_i8_desc(ty, rows, cols, x_stride=stride, up_stride=stride, q_stride=qs, act=act or 0)
        engine.quant_i8_dev(d, b, lead, None if act is None else b, lead + cols * size, q, 0, s, 0, v, 0)
        u = f64(x[:, :cols]) if act is None else act64(f64(x[:, :cols]), f64(x[:, cols:2 * cols]), act)
        raw = q.read(np.int8, rows * qs + 7)
        got = raw[:rows * qs].reshape(rows, qs)
        check_codes(got[:, :cols], s.read(np.float32, rows), v.read(np.float32, rows * cols).reshape(rows, cols),
                    *codes_of(u))
        # nothing past the columns, the last row, the scales or the values is touched
        assert np.all(got[:, cols:] == 0x5B) and np.all(raw[rows * qs:] == 0x5B)
        assert s.read(np.uint8, 4, 4 * rows).tolist() == [0x5B] * 4
        assert v.read(np.uint8, 4, 4 * rows * cols).tolist() == [0x5B] * 4


@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("ty", TYPES)
def test_rms_norm_rows(engine, ty, res):
    for k, (rows, cols, pad, lead) in enumerate(SHAPES):
        print(f"[case] norm type={ty} res={res} {rows}x{cols} +{pad}", flush=True)
        stride = cols + pad
        x, r = normal(10 + k, rows, stride).to(DT[ty]), (8.0 * normal(50 + k, rows, stride)).to(DT[ty])
        w = (normal(90 + k, cols) + 1.0).float()
        bx, br, bw = put(engine, x, lead), put(engine, r, lead), put(engine, w)
        q, s, v = engine.alloc(rows * cols), engine.alloc(4 * rows), engine.alloc(4 * rows * cols)
        o = put(engine, torch.full((rows, stride), -3.0, dtype=DT[ty]))
        d = engine.rms_norm_i8_desc(ty, rows, cols, EPS, x_stride=stride, res_stride=stride, sum_stride=stride)
        engine.rms_norm_i8_dev(d, bx, lead, br if res else None, lead, bw, 0, o if res else None, 0, q, 0, s, 0, v, 0)
        sum64 = f64(x[:, :cols]) + (f64(r[:, :cols]) if res else 0.0)
        unit = 1.0 / np.sqrt((sum64**2).mean(1, keepdims=True) + EPS)
        check_codes(q.read(np.int8, rows * cols).reshape(rows, cols), s.read(np.float32, rows),
                    v.read(np.float32, rows * cols).reshape(rows, cols), *codes_of(sum64 * f64(w), unit))
        got = get(o, DT[ty], (rows, stride))
        if res:
            assert torch.equal(got[:, :cols], torch.from_numpy(sum64).float().to(DT[ty]))
        assert torch.all(got[:, (cols if res else 0):] == -3.0)


@pytest.mark.parametrize("over", ["res", "x"])
@pytest.mark.parametrize("cols", [577, 20003])
def test_rms_norm_sum_in_place(engine, cols, over):
    x, r, w = normal(1, 3, cols).float(), normal(2, 3, cols).float(), normal(3, cols).float()
    bx, br, bw = put(engine, x), put(engine, r), put(engine, w)
    q, s = engine.alloc(3 * cols), engine.alloc(12)
    to = br if over == "res" else bx
    engine.rms_norm_i8_dev(engine.rms_norm_i8_desc(F32, 3, cols, 0.0), bx, 0, br, 0, bw, 0, to, 0, q, 0, s, 0)
    v = f64(x) + f64(r)
    check_codes(q.read(np.int8, 3 * cols).reshape(3, cols), s.read(np.float32, 3), None,
                *codes_of(v * f64(w), 1.0 / np.sqrt((v**2).mean(1, keepdims=True))))
    assert torch.equal(get(to, torch.float32, (3, cols)), torch.from_numpy(v).float())


def test_rows_of_zeros_extremes_and_non_finite_values(engine):
    cols = 300
    x = normal(4, 8, cols).float()
    x[0] = 0.0
    x[1, 17] = float("nan")
    x[2, 299] = float("inf")
    x[3, 0] = float("-inf")
    x[4] *= 1e38 / x[4].abs().max()
    x[5] *= 1e-40 / x[5].abs().max()   # f32 subnormals: the scale is one too
    x[6] = 0.0
    x[6, 5] = 1e-45                    # a scale below the smallest f32: 0, and codes 0
    b = put(engine, x)
    w = torch.ones(cols)
    bw = put(engine, w)
    for eps in (0.0, EPS):
        q, s, v = engine.alloc(8 * cols), engine.alloc(32), engine.alloc(32 * cols)
        engine.rms_norm_i8_dev(engine.rms_norm_i8_desc(F32, 8, cols, eps), b, 0, None, 0, bw, 0, None, 0, q, 0, s, 0,
                               v, 0)
        with np.errstate(all="ignore"):
            unit = 1.0 / np.sqrt((f64(x)**2).mean(1, keepdims=True) + float(np.float32(eps)))
            want = codes_of(f64(x), unit)
        check_codes(q.read(np.int8, 8 * cols).reshape(8, cols), s.read(np.float32, 8),
                    v.read(np.float32, 8 * cols).reshape(8, cols), *want)
    q, s, v = engine.alloc(8 * cols), engine.alloc(32), engine.alloc(32 * cols)
    engine.quant_i8_dev(engine.quant_i8_desc(F32, 8, cols), b, 0, None, 0, q, 0, s, 0, v, 0)
    check_codes(q.read(np.int8, 8 * cols).reshape(8, cols), s.read(np.float32, 8),
                v.read(np.float32, 8 * cols).reshape(8, cols), *codes_of(f64(x)))


def test_ties_between_codes_go_to_even(engine):
    # 127 u / a = 63.5, 0.5, 1.5 exactly, and one step of u to either side
    a = 254.0
    u = [a, 127.0, 1.0, 3.0, -127.0, -1.0, np.nextafter(np.float32(127), np.float32(0)),
         np.nextafter(np.float32(1), np.float32(2)), np.nextafter(np.float32(3), np.float32(0))]
    x = torch.tensor([u, [3 * v for v in u]], dtype=torch.float32)
    b = put(engine, x)
    q, s = engine.alloc(18), engine.alloc(8)
    engine.quant_i8_dev(engine.quant_i8_desc(F32, 2, 9), b, 0, None, 0, q, 0, s, 0)
    got = q.read(np.int8, 18).reshape(2, 9)
    assert got[0].tolist() == [127, 64, 0, 2, -64, 0, 63, 1, 1]
    assert np.array_equal(got, codes_of(f64(x))[0])


# ------------------------------------------------------------------------------- product


def codes(seed, rows, n, stride):
    c = np.random.default_rng(seed).integers(-127, 128, (rows, stride), dtype=np.int8)
    return torch.from_numpy(c), c[:, :n].astype(np.int64)


def run_gemm(engine, ty, m, n, t, wpad=0, xpad=0, ypad=0, res=False, in_place=False, seed=0, w=None, x=None,
             behind=0):
    ws, xs = (n + 15) // 16 * 16 + wpad, (n + 15) // 16 * 16 + xpad
    wt, w64 = codes(seed, m, n, ws) if w is None else w
    xt, x64 = codes(seed + 1, t, n, xs) if x is None else x
    sw = (normal(seed + 2, m).abs() * 0.01 + 1e-3).float()
    sx = (normal(seed + 3, t).abs() * 0.01 + 1e-3).float()
    ys = m + ypad
    r = (normal(seed + 4, t, ys) * np.sqrt(n) * 0.5).to(DT[ty])
    y0 = r if in_place else torch.full((t + behind, ys), 7.0, dtype=DT[ty])
    by = put(engine, y0)
    br = by if in_place else put(engine, r) if res else None
    d = engine.gemm_i8_desc(ty, m, n, t, w_stride=ws, x_stride=xs, res_stride=ys, y_stride=ys)
    engine.gemm_i8_dev(d, put(engine, wt), 0, put(engine, sw), 0, put(engine, xt), 0, put(engine, sx), 0, br, 0, by, 0)
    got = get(by, DT[ty], (t + behind, ys))
    assert torch.equal(got[t:], y0[t:])  # rows behind the last token's are left as they were
    got, y0 = got[:t], y0[:t]
    assert torch.equal(got[:, m:], y0[:, m:])
    # whole numbers below 2^53 in float64: exact
    prod = (x64.astype(np.float64) @ w64.astype(np.float64).T) * f64(sx)[:, None] * f64(sw)
    want = prod + (f64(r[:, :m]) if res or in_place else 0.0)
    u = 2.0**-24
    fi = torch.finfo(DT[ty])
    f32_err = np.abs(prod) * 3 * u * (1 + 4 * u) + np.abs(want) * u
    bound = f32_err + ((np.abs(want) + f32_err) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2 if ty != F32 else 0.0)
    err = np.abs(f64(got[:, :m]) - want)
    assert np.all(err <= bound), f"{ty} {m}x{n}x{t}: {np.count_nonzero(err > bound)} of {err.size} off"
    return got


GEMM = [(1, 1, 1), (3, 16, 2), (17, 64, 5), (64, 63, 16), (65, 65, 17), (130, 129, 33), (100, 1000, 1), (1000, 576, 7),
        (576, 1537, 65), (300, 4096, 16), (257, 2048, 128), (515, 300, 259), (48, 14336, 64), (2049, 130, 3),
        (768, 512, 600), (1111, 1040, 130)]


@pytest.mark.parametrize("ty", TYPES)
def test_gemm_shapes(engine, ty):
    for k, (m, n, t) in enumerate(GEMM):
        print(f"[case] gemm type={ty} m={m} n={n} t={t}", flush=True)
        run_gemm(engine, ty, m, n, t, wpad=16 * (k % 3), xpad=16 * (k % 2), ypad=k % 4, res=k % 2 == 0, seed=10 * k)


@pytest.mark.parametrize("ty", TYPES)
def test_gemm_onto_the_residual_in_place(engine, ty):
    for m, n, t in [(70, 200, 3), (512, 4096, 1), (512, 4096, 40), (640, 1024, 300)]:
        print(f"[case] in place type={ty} m={m} n={n} t={t}", flush=True)
        run_gemm(engine, ty, m, n, t, ypad=3, in_place=True, seed=m + t)


@pytest.mark.parametrize("t", [1, 20, 200])
def test_gemm_largest_sums(engine, t):
    n, stride = 131071, 131072
    for a, b in ((-128, -128), (-128, 127), (127, 127)):
        print(f"[case] largest sums t={t} {a} {b}", flush=True)
        w = (torch.full((24, stride), a, dtype=torch.int8), np.full((24, n), a, np.int64))
        x = (torch.full((t, stride), b, dtype=torch.int8), np.full((t, n), b, np.int64))
        run_gemm(engine, F32, 24, n, t, w=w, x=x)


def test_gemm_ignores_what_lies_between_rows(engine):
    """Bytes n..stride of codes hold anything: other bytes there leave every bit of y."""
    for n, t in ((100, 4), (1001, 50), (1000, 300)):
        got = []
        for fill in (0, -128, 77):
            w, w64 = codes(5, 200, n, n // 16 * 16 + 32)
            x, x64 = codes(6, t, n, n // 16 * 16 + 32)
            w[:, n:] = fill
            x[:, n:] = fill
            got.append(run_gemm(engine, F32, 200, n, t, wpad=(n // 16 * 16 + 32) - (n + 15) // 16 * 16,
                                xpad=(n // 16 * 16 + 32) - (n + 15) // 16 * 16, w=(w, w64), x=(x, x64)))
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_scales_carry_non_finite_rows_through(engine):
    """A token whose codes came from a NaN has scale NaN: its outputs are NaN, the others' untouched."""
    m, n, t = 40, 64, 3
    x = normal(1, t, n).float()
    x[1, 3] = float("nan")
    q, s = engine.alloc(t * n), engine.alloc(4 * t)
    engine.quant_i8_dev(engine.quant_i8_desc(F32, t, n), put(engine, x), 0, None, 0, q, 0, s, 0)
    w, _ = codes(2, m, n, n)
    y = engine.alloc(4 * t * m)
    engine.gemm_i8_dev(engine.gemm_i8_desc(F32, m, n, t), put(engine, w), 0, put(engine, torch.ones(m)), 0, q, 0, s, 0,
                       None, 0, y, 0)
    got = y.read(np.float32, t * m).reshape(t, m)
    assert np.all(np.isnan(got[1])) and np.all(np.isfinite(got[[0, 2]]))


# ------------------------------------------------------------------------------ together


class Layer:
    """An FFN block, the final norm and the head in codes, on resident buffers."""

    def __init__(self, engine, ty, t, d_model, d_ff, vocab, seed):
        self.e, self.ty, self.t, self.dm, self.df, self.v = engine, ty, t, d_model, d_ff, vocab
        size = torch.empty(0, dtype=DT[ty]).element_size()
        self.x = normal(seed, t, d_model).to(DT[ty])
        self.delta = (0.5 * normal(seed + 1, t, d_model)).to(DT[ty])
        self.norms = [(normal(seed + 2 + i, d_model) * 0.1 + 1.0).float() for i in range(2)]
        mats = [normal(seed + 5, 2 * d_ff, d_model, scale=d_model**-0.5).float(),
                normal(seed + 6, d_model, d_ff, scale=d_ff**-0.5).float(),
                normal(seed + 7, vocab, d_model, scale=3 * d_model**-0.5).float()]
        self.w = []
        for a in mats:  # weights laid out once
            rows, cols = a.shape
            q, s = engine.alloc(rows * cols), engine.alloc(4 * rows)
            engine.quant_i8_dev(engine.quant_i8_desc(F32, rows, cols), put(engine, a), 0, None, 0, q, 0, s, 0)
            self.w.append((q, s, rows, cols))
        self.bx, self.bd = put(engine, self.x), put(engine, self.delta)
        self.bn = [put(engine, n) for n in self.norms]
        self.params = engine.upload(engine.sample_params(0.8, [40 + i for i in range(t)], 0.9, 0.01))
        self.u = np.random.default_rng(seed + 8).random(t, dtype=np.float32)
        self.bu = engine.upload(self.u)
        a = engine.alloc
        self.r1, self.r2 = a(size * t * d_model), a(size * t * d_model)
        self.q1, self.s1, self.gu = a(t * d_model), a(4 * t), a(size * t * 2 * d_ff)
        self.q2, self.s2 = a(t * d_ff), a(4 * t)
        self.q3, self.s3, self.logits = a(t * d_model), a(4 * t), a(4 * t * vocab)
        self.ids, self.probs = a(4 * t), a(4 * t)
        self.size = size

    def step(self):
        e, ty, t, dm, df, v = self.e, self.ty, self.t, self.dm, self.df, self.v
        wg, wd, wh = self.w
        nd = e.rms_norm_i8_desc(ty, t, dm, EPS)
        # attention's output onto the stream, the FFN onto it again, then the head
        e.rms_norm_i8_dev(nd, self.bd, 0, self.bx, 0, self.bn[0], 0, self.r1, 0, self.q1, 0, self.s1, 0)
        e.gemm_i8_dev(e.gemm_i8_desc(ty, 2 * df, dm, t), wg[0], 0, wg[1], 0, self.q1, 0, self.s1, 0, None, 0, self.gu, 0)
        e.quant_i8_dev(e.quant_i8_desc(ty, t, df, x_stride=2 * df, up_stride=2 * df), self.gu, 0, self.gu,
                       df * self.size, self.q2, 0, self.s2, 0)
        e.gemm_i8_dev(e.gemm_i8_desc(ty, dm, df, t), wd[0], 0, wd[1], 0, self.q2, 0, self.s2, 0, self.r1, 0, self.r2, 0)
        e.rms_norm_i8_dev(nd, self.r2, 0, None, 0, self.bn[1], 0, None, 0, self.q3, 0, self.s3, 0)
        e.gemm_i8_dev(e.gemm_i8_desc(F32, v, dm, t), wh[0], 0, wh[1], 0, self.q3, 0, self.s3, 0, None, 0, self.logits, 0)
        e.sample_dev(e.sample_desc(F32, t, v), self.logits, 0, self.params, 0, self.bu, 0, self.ids, 0, self.probs, 0)

    def outputs(self):
        t = self.t
        return [get(self.r2, DT[self.ty], (t, self.dm)).clone(), get(self.logits, torch.float32, (t, self.v)).clone(),
                get(self.ids, torch.int32, (t,)).clone(), get(self.probs, torch.float32, (t,)).clone()]


@pytest.mark.parametrize("ty,t,d_model,d_ff,vocab", [(F32, 1, 576, 1536, 5000), (BF16, 5, 1024, 2816, 4097),
                                                     (F16, 130, 256, 704, 1000)])
def test_decode_step(engine, ty, t, d_model, d_ff, vocab):
    """Each step against its definition on the step's own inputs, and the whole against float weights."""
    L = Layer(engine, ty, t, d_model, d_ff, vocab, 31)
    L.step()
    r2, logits, ids, probs = L.outputs()
    w = [(q.read(np.int8, rows * cols).reshape(rows, cols).astype(np.float64), s.read(np.float32, rows).astype(np.float64))
         for q, s, rows, cols in L.w]
    v = f64(L.delta) + f64(L.x)
    q1, s1 = codes_of(v * f64(L.norms[0]), 1.0 / np.sqrt((v**2).mean(1, keepdims=True) + EPS))
    check_codes(L.q1.read(np.int8, q1.size).reshape(q1.shape), L.s1.read(np.float32, t), None, q1, s1)
    gu = f64(get(L.gu, DT[ty], (t, 2 * d_ff)))
    q2, s2 = codes_of(act64(gu[:, :d_ff], gu[:, d_ff:], 0))
    check_codes(L.q2.read(np.int8, q2.size).reshape(q2.shape), L.s2.read(np.float32, t), None, q2, s2)
    a = f64(r2)
    q3, s3 = codes_of(a * f64(L.norms[1]), 1.0 / np.sqrt((a**2).mean(1, keepdims=True) + EPS))
    check_codes(L.q3.read(np.int8, q3.size).reshape(q3.shape), L.s3.read(np.float32, t), None, q3, s3)
    # products, from the codes the steps left: three f32 roundings and the output's
    half = torch.finfo(DT[ty]).eps / 2
    p1 = q1.astype(np.float64) @ w[0][0].T * s1[:, None] * w[0][1]
    assert np.all(np.abs(gu - p1) <= np.abs(p1) * (half + 2.0**-22) + 2.0**-25)
    r1 = f64(get(L.r1, DT[ty], (t, d_model)))
    p2 = q2.astype(np.float64) @ w[1][0].T * s2[:, None] * w[1][1]
    assert np.all(np.abs(a - (p2 + r1)) <= np.abs(p2) * 2.0**-22 + np.abs(p2 + r1) * (half + 2.0**-23) + 2.0**-25)
    p3 = q3.astype(np.float64) @ w[2][0].T * s3[:, None] * w[2][1]
    assert np.all(np.abs(f64(logits) - p3) <= np.abs(p3) * 2.0**-22)
    assert torch.all((ids >= 0) & (ids < vocab)) and torch.all((probs > 0) & (probs <= 1))


def test_decode_step_captured(engine):
    """Replays give the eager bits, with eager work of another layer and other inputs between them."""
    L, other = Layer(engine, BF16, 9, 512, 1408, 6000, 7), Layer(engine, BF16, 20, 256, 704, 9000, 8)
    L.step()
    other.step()
    want, want_other = L.outputs(), other.outputs()
    g, g2 = engine.capture(L.step), engine.capture(other.step)
    x2 = normal(99, 9, 512).to(torch.bfloat16)
    first = L.bx.read(np.uint8, L.bx.nbytes)
    for k in range(4):
        print(f"[case] replay {k}", flush=True)
        for b in (L.r2, L.logits, L.ids, L.probs):
            b.fill(0xFF)
        g.launch()
        g2.launch()
        for a, b in zip(L.outputs(), want):
            assert torch.equal(a, b)
        for a, b in zip(other.outputs(), want_other):
            assert torch.equal(a, b)
        L.bx.write(x2.view(torch.uint8).numpy())
        L.step()
        eager = L.outputs()
        g.launch()
        for a, b in zip(L.outputs(), eager):
            assert torch.equal(a, b)
        L.bx.write(first)
        other.step()
    g.close()
    g2.close()


def test_same_bits_every_time(engine):
    L = Layer(engine, F32, 33, 512, 1408, 20000, 17)
    got = []
    for _ in range(5):
        L.step()
        got.append(L.outputs())
    for o in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, got[0]))


# ------------------------------------------------------------------------------ refusals


def refused(call, status, word):
    with pytest.raises(hayai_amd.HipError) as err:
        call()
    assert err.value.status_name == status and word in str(err.value), err.value


def test_quant_and_norm_refusals(engine):
    e = engine
    b, s, w = e.alloc(4096), e.alloc(64), e.alloc(256)

    def quant(ty=F32, rows=4, cols=64, up=None, q=b, q_off=0, off=0, so=0, v=None, **kw):
        e.quant_i8_dev(e.quant_i8_desc(ty, rows, cols, **kw), b, off, up, 0, q, q_off, s, so, v, 0)

    def norm(ty=F32, rows=4, cols=64, eps=EPS, res=None, sum=None, no=0, **kw):
        e.rms_norm_i8_dev(e.rms_norm_i8_desc(ty, rows, cols, eps, **kw), b, 0, res, 0, w, no, sum, 0, b, 0, s, 0)

    refused(lambda: quant(ty=hayai_amd.Q8_0), "HH_ERR_KERNEL_MISSING", "GGML type 8")
    refused(lambda: norm(ty=1000), "HH_ERR_KERNEL_MISSING", "GGML type 1000")
    refused(lambda: quant(cols=0), "HH_ERR_INVALID", "no columns")
    refused(lambda: norm(cols=0), "HH_ERR_INVALID", "no columns")
    refused(lambda: quant(rows=17), "HH_ERR_INVALID", "outside")
    refused(lambda: quant(x_stride=63), "HH_ERR_INVALID", "stride 63")
    refused(lambda: quant(q_stride=8), "HH_ERR_INVALID", "stride 8")
    refused(lambda: quant(off=2), "HH_ERR_INVALID", "splits an element")
    refused(lambda: quant(so=60), "HH_ERR_INVALID", "outside")
    refused(lambda: quant(so=2), "HH_ERR_INVALID", "splits an element")
    refused(lambda: quant(up=b, act=2), "HH_ERR_INVALID", "act 2")
    refused(lambda: quant(v=s), "HH_ERR_INVALID", "outside")
    refused(lambda: quant(rows=1 << 40), "HH_ERR_INVALID", "31-bit")
    refused(lambda: quant(rows=1 << 20, x_stride=1 << 60), "HH_ERR_INVALID", "overflow")
    refused(lambda: norm(eps=-1.0), "HH_ERR_INVALID", "eps")
    refused(lambda: norm(eps=float("nan")), "HH_ERR_INVALID", "eps")
    refused(lambda: norm(res=b), "HH_ERR_INVALID", "together")
    refused(lambda: norm(sum=b), "HH_ERR_INVALID", "together")
    refused(lambda: norm(no=4), "HH_ERR_INVALID", "outside")
    refused(lambda: norm(res=b, sum=b, sum_stride=1 << 20), "HH_ERR_INVALID", "outside")
    quant(rows=0)
    norm(rows=0)
    e.sync()


def test_gemm_refusals(engine):
    e = engine
    b, s = e.alloc(4096), e.alloc(256)

    def gemm(ty=F32, m=8, n=64, t=4, w_off=0, x_off=0, so=0, res=None, y_off=0, **kw):
        e.gemm_i8_dev(e.gemm_i8_desc(ty, m, n, t, **kw), b, w_off, s, so, b, x_off, s, 0, res, 0, b, y_off)

    refused(lambda: gemm(ty=hayai_amd.Q4_K), "HH_ERR_KERNEL_MISSING", "GGML type 12")
    refused(lambda: gemm(m=0), "HH_ERR_INVALID", "")
    refused(lambda: gemm(n=0), "HH_ERR_INVALID", "no columns")
    refused(lambda: gemm(n=131072), "HH_ERR_INVALID", "pass 32 bits")
    refused(lambda: gemm(n=60), "HH_ERR_INVALID", "16-byte")
    refused(lambda: gemm(w_off=8), "HH_ERR_INVALID", "16-byte")
    refused(lambda: gemm(x_off=4), "HH_ERR_INVALID", "16-byte")
    refused(lambda: gemm(x_stride=72), "HH_ERR_INVALID", "16-byte")
    refused(lambda: gemm(w_stride=48), "HH_ERR_INVALID", "stride 48")
    refused(lambda: gemm(m=65), "HH_ERR_INVALID", "outside")
    refused(lambda: gemm(x_off=3856), "HH_ERR_INVALID", "outside")
    refused(lambda: gemm(n=50, x_stride=64, w_stride=64, x_off=4096 - 4 * 64 + 16), "HH_ERR_INVALID", "outside")
    refused(lambda: gemm(t=65), "HH_ERR_INVALID", "outside")
    refused(lambda: gemm(y_off=2), "HH_ERR_INVALID", "splits an element")
    refused(lambda: gemm(y_off=4096 - 4 * 32 + 4), "HH_ERR_INVALID", "outside")
    refused(lambda: gemm(y_stride=7), "HH_ERR_INVALID", "stride 7")
    refused(lambda: gemm(res=s, res_stride=300), "HH_ERR_INVALID", "outside")
    gemm(t=0)
    e.sync()


def test_wrapped_memory(engine):
    """Handles on another library's device memory: the same results, ranges and pointers checked."""
    x = torch.randn(6, 100, device="cuda", dtype=torch.float32)
    q, s = torch.zeros(6, 100, device="cuda", dtype=torch.int8), torch.zeros(6, device="cuda")
    torch.cuda.synchronize()
    bx, bq, bs = (engine.wrap(v.data_ptr(), v.numel() * v.element_size()) for v in (x, q, s))
    engine.quant_i8_dev(engine.quant_i8_desc(F32, 6, 100), bx, 0, None, 0, bq, 0, bs, 0)
    engine.sync()
    check_codes(q.cpu().numpy(), s.cpu().numpy(), None, *codes_of(f64(x.cpu())))
    refused(lambda: engine.quant_i8_dev(engine.quant_i8_desc(F32, 7, 100), bx, 0, None, 0, bq, 0, bs, 0),
            "HH_ERR_INVALID", "outside")
    for b in (bx, bq, bs):
        b.free()
    assert torch.isfinite(x).all()  # the memory is still the tensors'
    host = np.zeros(64, np.float32)
    refused(lambda: engine.wrap(host.ctypes.data, 256), "HH_ERR_INVALID", "not device memory")
    refused(lambda: engine.wrap(0, 256), "HH_ERR_INVALID", "NULL")
    refused(lambda: engine.wrap(x.data_ptr(), 1 << 50), "HH_ERR_INVALID", "past the allocation")
    other = hayai_amd.HipEngine(0)
    try:
        with pytest.raises(hayai_amd.HipError, match="another engine"):
            engine.quant_i8_dev(engine.quant_i8_desc(F32, 1, 4), other.alloc(64), 0, None, 0, engine.alloc(64), 0,
                                engine.alloc(64), 0)
    finally:
        other.close()


# Rows enough to fill the chip twice: a workgroup of few threads with four chunks a thread, whose last
# chunks lie partly or wholly past the row.  One element; inside, at and past a chunk of 64 threads; in
# the third chunk; full; two waves; twelve or six.
MANY = [1, 5, 89, 255, 257, 577, 1000, 1024, 1029, 2500, 4099, 12001]
SLACK = 1 << 16


@pytest.mark.parametrize("kind", ["plain", "act", "norm"])
@pytest.mark.parametrize("ty", TYPES)
def test_many_rows(engine, ty, kind):
    rows = 2 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    size = torch.empty(0, dtype=DT[ty]).element_size()
    for k, cols in enumerate(MANY):
        print(f"[case] many {kind} type={ty} {rows}x{cols}", flush=True)
        wide = kind == "act"
        x = normal(200 + k, rows, 2 * cols if wide else cols, scale=2.0).to(DT[ty])
        w = (normal(300 + k, cols) + 1.0).float()
        bx, bw = put(engine, x), put(engine, w)
        q, s, v = engine.alloc(rows * cols + SLACK), engine.alloc(4 * rows), engine.alloc(4 * rows * cols + SLACK)
        o = engine.alloc(rows * cols * size + SLACK)
        for b in (q, s, v, o):
            b.fill(0x5B)
        u, unit = f64(x), 1.0
        if kind == "norm":
            d = engine.rms_norm_i8_desc(ty, rows, cols, EPS)
            engine.rms_norm_i8_dev(d, bx, 0, bx, 0, bw, 0, o, 0, q, 0, s, 0, v, 0)
            u = 2.0 * u
            assert torch.equal(get(o, DT[ty], (rows, cols)), torch.from_numpy(u).to(DT[ty]))
            unit = 1.0 / np.sqrt((u**2).mean(1, keepdims=True) + EPS)
            u = u * f64(w)
        elif wide:
            d = engine.quant_i8_desc(ty, rows, cols, x_stride=2 * cols, up_stride=2 * cols)
            engine.quant_i8_dev(d, bx, 0, bx, cols * size, q, 0, s, 0, v, 0)
            u = act64(u[:, :cols], u[:, cols:], hayai_amd.ACT_SILU)
        else:
            engine.quant_i8_dev(engine.quant_i8_desc(ty, rows, cols), bx, 0, None, 0, q, 0, s, 0, v, 0)
        check_codes(q.read(np.int8, rows * cols).reshape(rows, cols), s.read(np.float32, rows),
                    v.read(np.float32, rows * cols).reshape(rows, cols), *codes_of(u, unit))
        assert np.all(q.read(np.uint8, SLACK, rows * cols) == 0x5B)
        assert np.all(v.read(np.uint8, SLACK, 4 * rows * cols) == 0x5B)
        assert np.all(o.read(np.uint8, SLACK, rows * cols * size if kind == "norm" else 0) == 0x5B)


@pytest.mark.parametrize("ty", TYPES)
def test_gemm_leaves_rows_behind(engine, ty):
    """Each small form, with an output that goes on behind the last token; a tile cut into one to many
    workgroups; fewer tiles than workgroups of an XCD."""
    for k, (m, n, t) in enumerate([(100, 1000, 1), (9, 40, 3), (1001, 577, 7), (33, 16327, 9), (102, 16327, 64),
                                   (40, 131071, 17), (71, 93, 185), (300, 300, 300), (1667, 1040, 515)]):
        print(f"[case] behind type={ty} m={m} n={n} t={t}", flush=True)
        run_gemm(engine, ty, m, n, t, xpad=16 * (k % 2), ypad=k % 3, res=k % 2 == 1, seed=700 + 10 * k, behind=300)


# Each form of whole tiles (128x128, 128x256, 192x256, 256x256) with ragged edges, then several tiles a
# workgroup one after the other.
@pytest.mark.parametrize("ty,m,n,t", [(BF16, 11657, 1040, 515), (F16, 4997, 577, 1500), (F32, 7661, 577, 1500),
                                      (BF16, 9993, 577, 1501), (F16, 23457, 1040, 600), (BF16, 5991, 577, 4003),
                                      (F32, 20462, 577, 1500), (F16, 20462, 577, 1500)])
def test_gemm_large(engine, ty, m, n, t):
    run_gemm(engine, ty, m, n, t, wpad=16, ypad=1, res=ty == BF16, seed=m, behind=260)


@pytest.mark.parametrize("far", ["w", "x"])
def test_gemm_rows_far_apart(engine, far):
    """Rows of codes more than 16 MB apart: 256 of them pass 32 bits of offset."""
    m, n, t = (11657, 1040, 515) if far == "x" else (515, 1040, 11657)
    stride, packed = (1 << 24) + 16, 1040
    w, w64 = codes(1, m, n, packed)
    x, x64 = codes(2, t, n, packed)
    apart = engine.alloc(515 * stride)
    for i, row in enumerate((w if far == "w" else x).numpy()):
        apart.write(row, i * stride)
    bw, bx = (apart, put(engine, x)) if far == "w" else (put(engine, w), apart)
    one = put(engine, torch.ones(max(m, t), dtype=torch.float32))
    y = engine.alloc(4 * t * m)
    d = engine.gemm_i8_desc(F32, m, n, t, w_stride=stride if far == "w" else packed,
                            x_stride=stride if far == "x" else packed)
    engine.gemm_i8_dev(d, bw, 0, one, 0, bx, 0, one, 0, None, 0, y, 0)
    # whole numbers below 127^2 * 1040 < 2^24: exact in f32
    want = x64.astype(np.float32) @ w64.astype(np.float32).T
    assert np.array_equal(y.read(np.float32, t * m).reshape(t, m), want)


def test_more_rows_than_a_grid(engine):
    rows, cols = (1 << 22) + 5, 3
    for kind in ("plain", "act", "norm"):
        print(f"[case] grid {kind}", flush=True)
        x, up = normal(1, rows, cols).half(), normal(2, rows, cols).half()
        w = (normal(3, cols) + 1.0).float()
        bx, bu, bw = put(engine, x), put(engine, up), put(engine, w)
        q, s, v = engine.alloc(rows * cols + SLACK), engine.alloc(4 * rows + SLACK), engine.alloc(4 * rows * cols + SLACK)
        o = engine.alloc(rows * cols * 2)
        for b in (q, s, v):
            b.fill(0x5B)
        u, unit = f64(x), 1.0
        if kind == "norm":
            engine.rms_norm_i8_dev(engine.rms_norm_i8_desc(F16, rows, cols, EPS), bx, 0, bu, 0, bw, 0, o, 0, q, 0, s, 0, v, 0)
            u = u + f64(up)
            assert torch.equal(get(o, torch.float16, (rows, cols)), torch.from_numpy(u).float().half())
            unit = 1.0 / np.sqrt((u**2).mean(1, keepdims=True) + EPS)
            u = u * f64(w)
        elif kind == "act":
            engine.quant_i8_dev(engine.quant_i8_desc(F16, rows, cols), bx, 0, bu, 0, q, 0, s, 0, v, 0)
            u = act64(u, f64(up), hayai_amd.ACT_SILU)
        else:
            engine.quant_i8_dev(engine.quant_i8_desc(F16, rows, cols), bx, 0, None, 0, q, 0, s, 0, v, 0)
        check_codes(q.read(np.int8, rows * cols).reshape(rows, cols), s.read(np.float32, rows),
                    v.read(np.float32, rows * cols).reshape(rows, cols), *codes_of(u, unit))
        for b, n in ((q, rows * cols), (s, 4 * rows), (v, 4 * rows * cols)):
            assert np.all(b.read(np.uint8, SLACK, n) == 0x5B)


@pytest.mark.parametrize("ty", TYPES)
def test_gemm_mid(engine, ty):
    """64 x 64 tiles cut between workgroups and whole, then each form of whole tiles at few tokens."""
    for k, (m, n, t) in enumerate([(2999, 2100, 131), (4096, 512, 256), (8200, 100, 40), (2999, 130, 130),
                                   (16653, 1040, 130), (21979, 131, 300), (24645, 1040, 300)]):
        print(f"[case] mid type={ty} m={m} n={n} t={t}", flush=True)
        run_gemm(engine, ty, m, n, t, ypad=k % 2, res=k % 2 == 0, in_place=k == 3, seed=900 + 10 * k, behind=0 if k == 3 else 256)


def test_workspaces_grow_after_a_capture():
    """A captured step keeps its workspaces when a larger eager one makes the engine's grow."""
    with hayai_amd.HipEngine(0) as e:
        L = Layer(e, F16, 20, 256, 704, 5000, 30)
        L.step()
        want = L.outputs()
        g = e.capture(L.step)
        big = Layer(e, F16, 260, 576, 1536, 30000, 31)
        big.step()
        want_big = big.outputs()
        for k in range(3):
            print(f"[case] replay after growth {k}", flush=True)
            for b in (L.r2, L.logits, L.ids, L.probs):
                b.fill(0xFF)
            g.launch()
            big.step()
            assert all(torch.equal(a, b) for a, b in zip(L.outputs(), want))
            assert all(torch.equal(a, b) for a, b in zip(big.outputs(), want_big))
        g.close()


def test_two_engines(engine):
    """Two engines on one GPU, each from a thread of its own, disturb nothing of each other."""
    with hayai_amd.HipEngine(0) as other:
        layers = [Layer(engine, BF16, 17, 512, 1408, 9000, 40), Layer(other, BF16, 70, 512, 1408, 9000, 41)]
        want = []
        for L in layers:
            L.step()
            want.append(L.outputs())
        with ThreadPoolExecutor(2) as pool:
            for f in [pool.submit(lambda L: [L.step() for _ in range(20)], L) for L in layers]:
                f.result()
        for L, w in zip(layers, want):
            assert all(torch.equal(a, b) for a, b in zip(L.outputs(), w))
        del layers, L


# --------------------------------------------------------------- gated rows, special values


def gated(engine, ty, act, gate, up):
    """(codes, scale, values) of act(gate) * up, and what they have to be."""
    rows, cols = gate.shape
    q, s, v = engine.alloc(rows * cols), engine.alloc(4 * rows), engine.alloc(4 * rows * cols)
    engine.quant_i8_dev(engine.quant_i8_desc(ty, rows, cols, act=act), put(engine, gate), 0, put(engine, up), 0, q, 0, s, 0, v, 0)
    with np.errstate(all="ignore"):
        want = codes_of(act64(f64(gate), f64(up), act))
    return (q.read(np.int8, rows * cols).reshape(rows, cols), s.read(np.float32, rows),
            v.read(np.float32, rows * cols).reshape(rows, cols)), want


def many_rows():
    return 2 * torch.cuda.get_device_properties(0).multi_processor_count + 3


@pytest.mark.parametrize("act", [hayai_amd.ACT_SILU, hayai_amd.ACT_GELU_TANH])
@pytest.mark.parametrize("ty", TYPES)
def test_gated_rows_of_subnormal_gates(engine, ty, act):
    """Gates below or just above the type's normal range, whose products with up are ordinary numbers."""
    fi = torch.finfo(DT[ty])
    least = fi.smallest_normal * fi.eps
    # the row's largest from the smallest gate, beside an ordinary pair; neighbours among the smallest gates
    some = torch.tensor([[least, 1e-3], [3 * least, 4 * least], [-least, 2 * least]], dtype=torch.float64)
    up = torch.tensor([[0.9 * fi.max, 1e-6], [0.33 * fi.max, 0.3 * fi.max], [0.5 * fi.max, 0.2 * fi.max]], dtype=torch.float64)
    got, want = gated(engine, ty, act, some.to(DT[ty]), up.to(DT[ty]))
    check_codes(*got, *want)
    for rows in (7, many_rows()):
        for cols in (5, 300, 1029, 4099):
            print(f"[case] subnormal gates type={ty} act={act} {rows}x{cols}", flush=True)
            rng = np.random.default_rng(cols + rows)
            # gates of a row around one magnitude in or near the subnormals, up's from 1 to the type's largest
            low = np.exp2(rng.uniform(np.log2(least) + 1, np.log2(fi.smallest_normal) + 6, (rows, 1)))
            high = np.exp2(rng.uniform(0.0, np.log2(fi.max) - 4, (rows, 1)))
            gate, up = low * rng.standard_normal((rows, cols)), high * rng.standard_normal((rows, cols))
            ordinary = rng.random((rows, cols)) < 0.3  # some of ordinary gates with the same products
            gate, up = np.where(ordinary, gate / low, gate), np.where(ordinary, up * low, up)
            got, want = gated(engine, ty, act, torch.from_numpy(gate).to(DT[ty]), torch.from_numpy(up).to(DT[ty]))
            check_codes(*got, *want)


def special_rows(ty, act, cols, seed):
    """One row for each thing that the gated form decides apart from ordinary elements."""
    rng = np.random.default_rng(seed)
    big = torch.finfo(DT[ty]).max
    inf, nan = float("inf"), float("nan")
    at = int(rng.integers(0, cols))
    # exp(-80) in front of up: SiLU's gate there, and tanh-GELU's, whose exponent is 1.6 (g + 0.045 g^3)
    edge = -80.0 if act == hayai_amd.ACT_SILU else -9.673
    out = []

    def row(gate=None, up=None, at_gate=None, at_up=None):
        g = 2.0 * rng.standard_normal(cols) if gate is None else np.broadcast_to(gate, cols).copy()
        u = 2.0 * rng.standard_normal(cols) if up is None else np.broadcast_to(up, cols).copy()
        if at_gate is not None:
            g[at] = at_gate
        if at_up is not None:
            u[at] = at_up
        out.append((g, u))

    row()
    row(gate=0.0)
    row(up=0.0)
    row(gate=-0.0, at_up=-3.0)
    row(at_gate=nan)
    row(at_up=nan)
    for v in (inf, -inf):
        row(at_gate=v)
        row(at_gate=v, at_up=0.0)
        row(at_up=v)
        row(at_up=v, at_gate=0.0)
        row(at_up=v, at_gate=edge * 4)
    row(gate=edge * (1.0 + 0.02 * rng.standard_normal(cols)))                 # on both sides of the edge, alone
    mixed = rng.random(cols) < 0.5                                            # and among ordinary gates
    row(gate=np.where(mixed, edge * (1.0 + 0.02 * rng.standard_normal(cols)), rng.standard_normal(cols)))
    row(gate=np.where(mixed, edge * 1.02, rng.standard_normal(cols)), up=np.where(mixed, 0.3 * big, 1e-3))
    row(gate=1e-2 * rng.standard_normal(cols), up=1e-7, at_gate=edge * 1.03, at_up=0.5 * big)  # the largest there
    row(gate=-1000.0)
    row(gate=edge * 9.0)
    # the largest outside 1e-25..1e25, and at either end of it, as far as the type goes
    for power in (-44, -40, -30, -25, -24, -12, 0, 4, 12, 24, 25, 30, 36):
        half = 10.0 ** (power / 2)
        if half < 0.5 * big:
            row(gate=half * np.abs(rng.standard_normal(cols)), up=half * rng.standard_normal(cols))
    # products past f32, of an element that is small all the same
    row(gate=np.where(mixed, edge * 0.9, 1.0), up=np.where(mixed, 0.9 * big, 1e-2))
    row(gate=np.where(mixed, -big, 1.0))
    row(gate=1.0, up=0.25 * big * np.where(rng.random(cols) < 0.5, 1.0, 0.3))
    gate, up = (torch.from_numpy(np.stack(v)).to(DT[ty]) for v in zip(*out))
    return gate, up


@pytest.mark.parametrize("act", [hayai_amd.ACT_SILU, hayai_amd.ACT_GELU_TANH])
@pytest.mark.parametrize("ty", TYPES)
def test_gated_special_rows(engine, ty, act):
    """Zero rows, NaN, infinities, gates where exp(-y) is large, largest values near the ends of f32: by
    each form of a row (one to four chunks a thread, read twice), few and many."""
    for many, columns in ((False, (1, 7, 300, 1029, 4099, 12001, 20003, 33001)), (True, (5, 300, 1029, 4099))):
        for cols in columns:
            print(f"[case] special rows type={ty} act={act} many={many} {cols}", flush=True)
            gate, up = special_rows(ty, act, cols, cols)
            if many:
                times = -(-many_rows() // len(gate))
                gate, up = gate.repeat(times, 1), up.repeat(times, 1)
            got, want = gated(engine, ty, act, gate, up)
            check_codes(*got, *want)


@pytest.mark.parametrize("ty", TYPES)
def test_gated_many_rows_gelu(engine, ty):
    for k, cols in enumerate(MANY):
        print(f"[case] many gelu type={ty} {cols}", flush=True)
        gate, up = (normal(400 + 50 * i + k, many_rows(), cols, scale=2.0).to(DT[ty]) for i in range(2))
        got, want = gated(engine, ty, hayai_amd.ACT_GELU_TANH, gate, up)
        check_codes(*got, *want)


@pytest.mark.parametrize("how", ["one stream", "events"])
def test_shared_tensors_without_a_host_synchronization(engine, how):
    """Another library's long work before the engine's calls and its reads after them, ordered by the
    engine's stream alone."""
    rows, cols = 64, 4096
    own = torch.cuda.ExternalStream(engine.stream)
    other = own if how == "one stream" else torch.cuda.Stream()
    a = torch.randn(4096, 4096, device="cuda") / 64.0
    x, first = torch.zeros(rows, cols, device="cuda"), torch.randn(rows, 4096, device="cuda")
    q, s = torch.zeros(rows, cols, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
    bx, bq, bs = (engine.wrap(v.data_ptr(), v.numel() * v.element_size()) for v in (x, q, s))
    d = engine.quant_i8_desc(F32, rows, cols)
    want = []
    with torch.cuda.stream(other):
        torch.mm(first, a)  # (the library's first product sets it up)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(other):
            v = first
            for _ in range(60):
                v = torch.mm(v, a)
                v = v / v.abs().amax()
            x.copy_(v)
            first = v + 0.25
        if other is not own:
            own.wait_stream(other)
        engine.quant_i8_dev(d, bx, 0, None, 0, bq, 0, bs, 0)
        if other is not own:
            other.wait_stream(own)
        with torch.cuda.stream(other):
            want.append((x.clone(), q.clone(), s.clone()))
            q.zero_()
            s.zero_()
    torch.cuda.synchronize()
    for x, q, s in want:
        check_codes(q.cpu().numpy(), s.cpu().numpy(), None, *codes_of(f64(x.cpu())))


def test_gated_rows_whose_scale_passes_f32(engine):
    """Finite u, a / 127 past f32: codes as ever, scale infinity."""
    gate, up = torch.tensor([[1e30, 5e29, 1.0, -1e30]]).repeat(2, 1), torch.tensor([[1e30, -1e30, 1.0, 1e30]]).repeat(2, 1)
    got, want = gated(engine, F32, hayai_amd.ACT_SILU, gate, up)
    assert want[0].tolist() == [[127, -64, 0, 0]] * 2  # (-63.5 to even; the last gate's act is 0)
    assert np.array_equal(got[0], want[0]) and np.all(got[1] == np.inf)


@pytest.mark.parametrize("t", [hayai_amd.Q4_0, hayai_amd.Q8_0, hayai_amd.Q4_K, hayai_amd.Q6_K, hayai_amd.IQ2_XXS,
                               hayai_amd.IQ3_XXS])
def test_codes_from_packed_weights(engine, t):
    """A GGUF matrix into codes on the device, and a product with them."""
    from hayai_amd import synth
    import oracle
    rows, cols, tokens = 300, 768, 5
    packed = synth.matrix(t, rows, cols, 77)
    f, q, s = engine.alloc(4 * rows * cols), engine.alloc(rows * cols), engine.alloc(4 * rows)
    engine.dequant_dev(t, engine.upload(packed), 0, rows * cols, f)
    engine.quant_i8_dev(engine.quant_i8_desc(F32, rows, cols), f, 0, None, 0, q, 0, s, 0)
    w = oracle.dequant(t, packed, rows * cols).reshape(rows, cols).astype(np.float64)
    want_q, want_s = codes_of(w)
    got_q, got_s = q.read(np.int8, rows * cols).reshape(rows, cols), s.read(np.float32, rows)
    check_codes(got_q, got_s, None, want_q, want_s)
    x, x64 = codes(3, tokens, cols, cols)
    y, one = engine.alloc(4 * tokens * rows), put(engine, torch.ones(tokens))
    engine.gemm_i8_dev(engine.gemm_i8_desc(F32, rows, cols, tokens), q, 0, s, 0, put(engine, x), 0, one, 0, None, 0, y, 0)
    want = (x64 @ got_q.astype(np.int64).T).astype(np.float64) * got_s.astype(np.float64)
    # the sum to f32 and its product with the scale: two roundings
    assert np.all(np.abs(y.read(np.float32, tokens * rows).reshape(tokens, rows) - want) <= np.abs(want) * 2.0**-23 * (1 + 1e-6))


def test_rows_four_gigabytes_apart(engine):
    """Strides and offsets past 32 bits in every operand that has rows of its own."""
    cols, rows, far = 300, 3, (1 << 31) + 64  # f16 elements: 4 GB and a little
    lead = 256
    x, r = normal(1, rows, cols).half(), normal(2, rows, cols).half()
    w = (normal(3, cols) + 1.0).float()
    big = engine.alloc(lead + 2 * ((rows - 1) * far + 2 * cols) + 64)
    big.fill(0x5B)
    for i in range(rows):
        big.write(x[i].view(torch.uint8).numpy(), lead + 2 * i * far)
        big.write(r[i].view(torch.uint8).numpy(), lead + 2 * (i * far + cols))
    qfar = (1 << 32) + 16
    q, s, v = engine.alloc((rows - 1) * qfar + cols + 64), engine.alloc(4 * rows), engine.alloc(4 * rows * cols)
    for i in range(rows):
        q.fill(0x5B, cols + 64, i * qfar)

    def codes_at(i):
        got = q.read(np.int8, cols + 64, i * qfar)
        assert np.all(got[cols:] == 0x5B)
        return got[:cols]

    d = engine.quant_i8_desc(F16, rows, cols, x_stride=far, up_stride=far, q_stride=qfar)
    engine.quant_i8_dev(d, big, lead, big, lead + 2 * cols, q, 0, s, 0, v, 0)
    check_codes(np.stack([codes_at(i) for i in range(rows)]), s.read(np.float32, rows),
                v.read(np.float32, rows * cols).reshape(rows, cols), *codes_of(act64(f64(x), f64(r), hayai_amd.ACT_SILU)))
    # the sum over the residual, in place
    d = engine.rms_norm_i8_desc(F16, rows, cols, EPS, x_stride=far, res_stride=far, sum_stride=far, q_stride=qfar)
    engine.rms_norm_i8_dev(d, big, lead, big, lead + 2 * cols, put(engine, w), 0, big, lead + 2 * cols, q, 0, s, 0, v, 0)
    sum64 = f64(x) + f64(r)
    check_codes(np.stack([codes_at(i) for i in range(rows)]), s.read(np.float32, rows),
                v.read(np.float32, rows * cols).reshape(rows, cols),
                *codes_of(sum64 * f64(w), 1.0 / np.sqrt((sum64**2).mean(1, keepdims=True) + EPS)))
    for i in range(rows):
        got = big.read(np.uint8, 4 * cols + 64, lead + 2 * i * far)
        assert torch.equal(torch.from_numpy(got[2 * cols:4 * cols]).view(torch.float16), torch.from_numpy(sum64[i]).float().half())
        assert np.array_equal(got[:2 * cols], x[i].view(torch.uint8).numpy()) and np.all(got[4 * cols:] == 0x5B)
    del big
    # a product with those codes, its rows as far apart: by rows of codes, and by tiles
    m, n = 70, 288
    for t, from_far in ((3, True), (40, False)):
        w8, w64 = codes(5, m, n, n)
        x8, x64 = codes(6, t, n, n)
        if from_far:
            x64 = np.stack([codes_at(i) for i in range(rows)])[:, :n].astype(np.int64)
            bx, xstride = q, qfar
        else:
            bx, xstride = put(engine, x8), n
        yfar = far if t == 3 else 1 << 26
        y = engine.alloc(2 * ((t - 1) * yfar + m) + 64)
        for i in range(t):
            y.fill(0x5B, 2 * m + 64, 2 * i * yfar)
        one = put(engine, torch.full((max(m, t),), 2.0**-4))
        if from_far:  # the last row has its whole stride in the buffer
            q2 = engine.alloc(rows * qfar)
            for i in range(rows):
                q2.copy_from(q, cols, i * qfar, i * qfar)
            bx = q2
        engine.gemm_i8_dev(engine.gemm_i8_desc(F16, m, n, t, x_stride=xstride, y_stride=yfar), put(engine, w8), 0, one, 0,
                           bx, 0, one, 0, None, 0, y, 0)
        want = (x64 @ w64.T).astype(np.float64) / 256.0
        for i in range(t):
            raw = y.read(np.uint8, 2 * m + 64, 2 * i * yfar)
            got = torch.from_numpy(raw[:2 * m]).view(torch.float16).double().numpy()
            # whole numbers below 2^24 and powers of two: one rounding, to f16
            assert np.all(np.abs(got - want[i]) <= np.abs(want[i]) * 2.0**-11 + 2.0**-25) and np.all(raw[2 * m:] == 0x5B)
        del y
