"""GPU test of a decoder layer's attention half as a program runs it: the norm into codes, one product for queries,
keys and values, rotary positions into the cache, attention of the prompts, codes, the output's product onto the
residual stream; then the first sequence forked, and a batch of tokens decoded behind the shared prompt, eagerly and
as a graph.

Each step is checked on what the step before it left: codes and products are those of the 8-bit path's definitions
(equal codes; one rounding for each of sum, scales, residual and type), the rest as in test_gpu_attn_pages and
attn_reference.
"""
import numpy as np
import pytest
import torch

from attn_reference import attend, check, gather, half_step, page_elements
from hayai_amd import BF16, F32, HipEngine
from test_gpu_attn_pages import get, ints, near, normal, put, turned
from test_gpu_i8 import codes_of

pytestmark = pytest.mark.gpu

D_MODEL, HEADS, KV, DIM, PAGE, BASE = 320, 8, 2, 64, 32, 10000.0
WIDE = (HEADS + 2 * KV) * DIM
SCALE = float(np.float32(DIM**-0.5))
EPS = float(np.float32(1e-5))


class Layer:
    """Weights and activations of one layer for up to `rows` tokens; type ty, a cache of type cty."""

    def __init__(self, engine, ty, cty, n_pages, rows):
        self.e, self.ty, self.cty, self.n_pages = engine, ty, cty, n_pages
        self.dt = {F32: torch.float32, BF16: torch.bfloat16}[ty]
        self.el = 4 if ty == F32 else 2
        rng = np.random.default_rng(0)
        self.norm = rng.uniform(0.5, 1.5, D_MODEL).astype(np.float32)
        self.w_qkv, self.w_out = (rng.integers(-127, 128, s).astype(np.int8) for s in ((WIDE, D_MODEL), (D_MODEL, HEADS * DIM)))
        self.s_qkv, self.s_out = (rng.uniform(1, 2, n).astype(np.float32) / (73 * k**0.5)
                                  for n, k in ((WIDE, D_MODEL), (D_MODEL, HEADS * DIM)))
        up, alloc = engine.upload, engine.alloc
        self.b = {"norm": up(self.norm), "w_qkv": up(self.w_qkv), "w_out": up(self.w_out), "s_qkv": up(self.s_qkv),
                  "s_out": up(self.s_out), "x": alloc(rows * D_MODEL * self.el), "codes": alloc(rows * D_MODEL), "scale": alloc(4 * rows),
                  "qkv": alloc(rows * WIDE * self.el), "q": alloc(rows * HEADS * DIM * self.el), "att": alloc(rows * HEADS * DIM * self.el),
                  "att_codes": alloc(rows * HEADS * DIM), "att_scale": alloc(4 * rows), "y": alloc(rows * D_MODEL * self.el),
                  "cache": alloc(n_pages * page_elements(KV, DIM, PAGE) * (4 if cty == F32 else 2)),
                  "positions": alloc(4 * rows), "slots": alloc(4 * rows)}
        self.b["cache"].fill(0xFF)  # NaN everywhere
        self.kv = engine.kv_desc(cty, KV, DIM, PAGE, n_pages)

    def run(self, rows, attention):
        """Enqueues the layer for the x, positions and slots that are in the buffers."""
        e, b, q_bytes, kv_bytes = self.e, self.b, HEADS * DIM * self.el, KV * DIM * self.el
        e.rms_norm_i8_dev(e.rms_norm_i8_desc(self.ty, rows, D_MODEL, 1e-5), b["x"], 0, None, 0, b["norm"], 0, None, 0, b["codes"], 0,
                          b["scale"], 0)
        e.gemm_i8_dev(e.gemm_i8_desc(self.ty, WIDE, D_MODEL, rows), b["w_qkv"], 0, b["s_qkv"], 0, b["codes"], 0, b["scale"], 0,
                      None, 0, b["qkv"], 0)
        e.rope_kv_dev(e.rope_desc(self.ty, rows, HEADS, DIM, BASE, q_stride=WIDE, k_stride=WIDE, v_stride=WIDE), self.kv, b["qkv"], 0,
                      b["qkv"], q_bytes, b["qkv"], q_bytes + kv_bytes, b["positions"], 0, b["slots"], 0, None, 0, b["q"], 0,
                      b["cache"], 0)
        attention()
        e.quant_i8_dev(e.quant_i8_desc(self.ty, rows, HEADS * DIM), b["att"], 0, None, 0, b["att_codes"], 0, b["att_scale"], 0)
        e.gemm_i8_dev(e.gemm_i8_desc(self.ty, D_MODEL, HEADS * DIM, rows), b["w_out"], 0, b["s_out"], 0, b["att_codes"], 0,
                      b["att_scale"], 0, b["x"], 0, b["y"], 0)

    def cache(self):
        dt = {F32: torch.float32, BF16: torch.bfloat16}[self.cty]
        return get(self.b["cache"], dt, (self.n_pages, page_elements(KV, DIM, PAGE)))

    def product(self, codes, scale, w, ws, res=None):
        y = (codes.astype(np.int64) @ w.astype(np.int64).T) * scale.astype(np.float64)[:, None] * ws.astype(np.float64)
        slack = np.abs(y) * 3 * 2.0**-24
        if res is not None:
            y = y + res
            slack = slack + np.abs(y) * 2.0**-24
        return torch.from_numpy(y), torch.from_numpy(slack)

    def check(self, x, positions, slots, sequences):
        """sequences: (rows, table, length) of each; their last rows see the whole length."""
        rows, b = len(positions), self.b
        x64 = x.double().numpy()
        u = x64 * self.norm.astype(np.float64)
        codes, scale = b["codes"].read(np.int8, rows * D_MODEL).reshape(rows, -1), b["scale"].read(np.float32, rows)
        want, want_scale = codes_of(u, 1.0 / np.sqrt(np.mean(x64**2, axis=1, keepdims=True) + EPS))
        assert np.array_equal(codes, want) and np.allclose(scale, want_scale, rtol=2.0**-23)
        qkv = get(b["qkv"], self.dt, (rows, HEADS + 2 * KV, DIM))
        want, slack = self.product(codes, scale, self.w_qkv, self.s_qkv)
        near(qkv, want.reshape(qkv.shape), self.dt, slack.reshape(qkv.shape))
        q = get(b["q"], self.dt, (rows, HEADS, DIM))
        want = turned(qkv.double(), np.array(positions), DIM, BASE, 0, None, 1.0)
        size = (qkv.double() ** 2).sum(-1, keepdim=True).sqrt().expand_as(want) * 6 * 2.0**-24
        near(q, want[:, :HEADS], self.dt, size[:, :HEADS])
        cache = self.cache()
        per = cache.shape[1] // 2
        for i, slot in enumerate(slots):
            page, at = divmod(slot, PAGE)
            near(cache[page, :per].view(KV, PAGE, DIM)[:, at], want[i, HEADS:HEADS + KV], cache.dtype, size[i, HEADS:HEADS + KV])
            near(cache[page, per:].view(KV, DIM, PAGE)[:, :, at], qkv[i, HEADS + KV:].double(), cache.dtype, torch.zeros(KV, DIM).double())
        att = get(b["att"], self.dt, (rows, HEADS, DIM))
        first = 0
        for n, table, length in sequences:
            k, v = gather(cache, table, length, KV, DIM, PAGE)
            out, bound = attend(q[first:first + n].double().numpy(), k, v, length - n + 1 + np.arange(n), SCALE, self.ty, self.cty)
            check(att[first:first + n], out, bound, self.ty)
            first += n
        codes, scale = b["att_codes"].read(np.int8, rows * HEADS * DIM).reshape(rows, -1), b["att_scale"].read(np.float32, rows)
        want, want_scale = codes_of(att.double().numpy().reshape(rows, -1))
        assert np.array_equal(codes, want) and np.allclose(scale, want_scale, rtol=2.0**-23)
        want, slack = self.product(codes, scale, self.w_out, self.s_out, x64)
        near(get(b["y"], self.dt, (rows, D_MODEL)), want, self.dt, slack)


@pytest.mark.parametrize("ty,cty,apart", [(BF16, BF16, True), (BF16, BF16, False), (F32, F32, True), (F32, BF16, False)])
def test_layer(engine, ty, cty, apart, monkeypatch):
    """apart: the decode steps' shared tokens, few as they are, by the kernel for many."""
    if apart:
        monkeypatch.setenv("HAYAI_HIP_ATTN_SHARE_MIN", "0")
        engine = HipEngine(0)
    lengths = [301, 40, 7]
    layer = Layer(engine, ty, cty, 40, sum(lengths))
    pages = list(np.random.default_rng(1).permutation(40))
    tables = np.full((3, 12), -1, np.int32)
    for s, n in enumerate(lengths):
        for i in range(-(-n // PAGE)):
            tables[s, i] = pages.pop()
    positions = [t for n in lengths for t in range(n)]
    slots = [int(tables[s, t // PAGE]) * PAGE + t % PAGE for s, n in enumerate(lengths) for t in range(n)]
    x = normal(2, sum(lengths), D_MODEL).to(layer.dt)
    layer.b["x"].write(x.view(torch.uint8).numpy())
    layer.b["positions"].write(np.array(positions, np.int32))
    layer.b["slots"].write(np.array(slots, np.int32))
    starts, lens, table_b = ints(engine, [0, 301, 341, 348]), ints(engine, lengths), engine.upload(tables)
    desc = engine.attn_prompt_desc(ty, 348, 3, HEADS, SCALE, 12)
    layer.run(348, lambda: engine.attn_prompt_dev(desc, layer.kv, layer.b["q"], 0, layer.b["cache"], 0, starts, 0, lens, 0, table_b, 0,
                                                  layer.b["att"], 0))
    layer.check(x, positions, slots, [(n, tables[s], n) for s, n in enumerate(lengths)])

    # five continuations of the first prompt: its whole pages are shared, the page it ends in is copied
    n, last = lengths[0], int(tables[0, 301 // PAGE])
    children = np.full((5, 12), -1, np.int32)
    children[:, :9] = tables[0, :9]
    children[0, 9] = last
    children[1:, 9] = [pages.pop() for _ in range(4)]
    engine.kv_copy_dev(layer.kv, layer.b["cache"], 0, engine.upload(np.array([(last, c) for c in children[1:, 9]], np.int32)), 0, 4)
    child_b, child_lens, prefix = engine.upload(children), engine.alloc(20), ints(engine, children[0, :10].tolist())
    desc5 = engine.attn_decode_desc(ty, 5, HEADS, SCALE, 12, prefix=n)

    def step():
        layer.run(5, lambda: engine.attn_decode_dev(desc5, layer.kv, layer.b["q"], 0, layer.b["cache"], 0, prefix, 0, child_lens, 0,
                                                    child_b, 0, layer.b["att"], 0))

    graph = None
    for token in range(4):
        at = n + token
        x = normal(10 + token, 5, D_MODEL).to(layer.dt)
        slots = [int(c[at // PAGE]) * PAGE + at % PAGE for c in children]
        layer.b["x"].write(x.view(torch.uint8).numpy())
        layer.b["positions"].write(np.full(5, at, np.int32))
        layer.b["slots"].write(np.array(slots, np.int32))
        child_lens.write(np.full(5, at + 1, np.int32))
        if token == 0:
            step()
        else:
            graph = graph or engine.capture(step)
            graph.launch()
        layer.check(x, [at] * 5, slots, [(1, c, at + 1) for c in children])
    graph.free()
    if apart:
        engine.close()
