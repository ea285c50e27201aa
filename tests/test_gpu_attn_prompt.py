"""GPU tests of causal attention over pages (attn_prompt) against its definition in 64 bits; the bounds'
derivation stands in attn_reference.py."""
import numpy as np
import pytest
import torch

from attn_reference import DT, attend, check, gather, page_elements
from hayai_amd import BF16, F16, F32, HipEngine, HipError
from test_gpu_attn_decode import far_smaller
from test_gpu_attn_pages import get, ints, normal, put

pytestmark = pytest.mark.gpu

TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]


class Problem:
    """Packed sequences of (new, cached) tokens, their pages at random places."""

    def __init__(self, ty, cty, seqs, heads, kvh, dim, page, seed=0, spare=2, pad=0, scale=None, width=None):
        self.ty, self.cty, self.seqs, self.heads, self.kvh, self.dim, self.page, self.pad = ty, cty, seqs, heads, kvh, dim, page, pad
        rng = np.random.default_rng(seed)
        per = page_elements(kvh, dim, page)
        need = [-(-max(length, 0) // page) for _, length in seqs]
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages)
        self.width = max(need + [1]) if width is None else width
        self.tables = np.full((len(seqs), self.width), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = ids[at:at + n]
            at += n
        self.cache = normal(seed + 1, self.n_pages, per).to(DT[cty])
        self.starts = np.cumsum([0] + [n for n, _ in seqs]).astype(np.int32)
        self.lens = np.array([length for _, length in seqs], np.int32)
        self.tokens = int(self.starts[-1])
        self.q = normal(seed + 2, self.tokens, heads * dim + pad).to(DT[ty])
        self.scale = float(np.float32(dim**-0.5 if scale is None else scale))

    def run(self, engine, tokens=None):
        tokens = self.tokens if tokens is None else tokens
        wide = self.heads * self.dim + self.pad
        self.out = put(engine, torch.full((max(tokens, self.tokens), wide), 5.0).to(DT[self.ty]))
        q = torch.zeros(max(tokens, len(self.q)), wide).to(DT[self.ty])
        q[:len(self.q)] = self.q
        d = engine.attn_prompt_desc(self.ty, tokens, len(self.seqs), self.heads, self.scale, self.width, wide, wide)
        kv = engine.kv_desc(self.cty, self.kvh, self.dim, self.page, self.n_pages)
        engine.attn_prompt_dev(d, kv, put(engine, q), 0, put(engine, self.cache), 0, ints(engine, self.starts.tolist()), 0,
                               ints(engine, self.lens.tolist()), 0, ints(engine, self.tables.reshape(-1).tolist()), 0, self.out, 0)
        return get(self.out, DT[self.ty], (max(tokens, self.tokens), wide))

    def want(self, cache=None):
        cache = self.cache if cache is None else cache
        q = self.q[:, :self.heads * self.dim].double().numpy().reshape(-1, self.heads, self.dim)
        out, bound = np.zeros_like(q), np.zeros_like(q)
        for s, (n, length) in enumerate(self.seqs):
            length = min(max(length, 0), self.width * self.page)
            rows = slice(self.starts[s], self.starts[s] + n)
            k, v = gather(cache, self.tables[s], length, self.kvh, self.dim, self.page)
            out[rows], bound[rows] = attend(q[rows], k, v, length - n + 1 + np.arange(n), self.scale, self.ty, self.cty)
        return out, bound

    def check(self, engine, cache=None):
        got = self.run(engine)
        want, bound = self.want(cache)
        check(got[:self.tokens, :self.heads * self.dim].reshape(want.shape), want, bound, self.ty)
        assert torch.all(got[:, self.heads * self.dim:] == 5.0)
        return got


# sequences (new, cached), heads, kv heads, dim, page: one token, tiles' edges, ragged packs, empty sequences, rows
# that see nothing (more new than cached tokens), parts of longer prompts, long ones whose keys are split, groups
# of 1, 3, 7, 64 heads
CASES = [([(1, 1)], 1, 1, 64, 16), ([(30, 30)], 9, 3, 64, 16), ([(33, 33), (1, 1), (0, 0), (70, 70)], 8, 2, 128, 32),
         ([(5, 3), (4, 0), (2, 40)], 4, 4, 64, 64), ([(64, 64)], 2, 2, 128, 64), ([(65, 129), (3, 700)], 7, 1, 128, 128),
         ([(17, 17)], 4, 1, 72, 16), ([(40, 101)], 3, 1, 256, 32), ([(3, 2500)], 8, 2, 128, 16), ([(1, 1300), (2, 15)], 64, 1, 64, 256),
         ([(9, 650)], 2, 1, 8, 16), ([(21, 21), (22, 150)], 6, 2, 200, 64), ([(130, 130), (0, 64), (140, 141)], 5, 5, 96, 32)]


@pytest.mark.parametrize("ty,cty", TYPES)
def test_prompt(engine, ty, cty):
    for i, (seqs, heads, kvh, dim, page) in enumerate(CASES):
        print(f"[case] prompt {ty} {cty} {CASES[i]}", flush=True)
        Problem(ty, cty, seqs, heads, kvh, dim, page, seed=i, pad=i % 3).check(engine)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_rows_of_no_sequence_stay(engine, ty):
    p = Problem(ty, ty, [(20, 20), (7, 31)], 4, 2, 64, 32)
    got = p.run(engine, tokens=60)
    want, bound = p.want()
    check(got[:27].reshape(want.shape), want, bound, ty)
    assert torch.all(got[27:] == 5.0)
    # a first sequence that begins later
    p.starts = p.starts + 5
    p.q = torch.cat([torch.zeros_like(p.q[:5]), p.q])
    got = p.run(engine, tokens=60)
    check(got[5:32].reshape(want.shape), want, bound, ty)
    assert torch.all(got[:5] == 5.0) and torch.all(got[32:] == 5.0)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see(engine, ty, bad):
    """Later tokens' keys and values, slots past the length and pages of no sequence hold no finite numbers."""
    for seqs, page in [([(50, 50)], 16), ([(70, 400)], 64), ([(3, 1201)], 32)]:
        p = Problem(ty, ty, seqs, 4, 2, 128, page, seed=3)
        n, length = seqs[0]
        want, bound = p.want()
        per, kvh, dim = page_elements(2, 128, page), 2, 128
        keys, values = p.cache[:, :per // 2].view(-1, kvh, page, dim), p.cache[:, per // 2:].view(-1, kvh, dim, page)
        used = set(p.tables[0].tolist())
        for other in range(p.n_pages):
            if other not in used:
                p.cache[other] = bad
        for t in range(length - n // 2, -(-length // page) * page):  # later half of the new tokens, and past them
            keys[p.tables[0, t // page], :, t % page] = bad
            values[p.tables[0, t // page], :, :, t % page] = bad
        got = p.run(engine).double().numpy().reshape(want.shape)
        free = n - n // 2
        check(torch.from_numpy(got[:free]), want[:free], bound[:free], ty)
        assert not np.any(np.isfinite(got[free:]))


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_infinite_value_is_seen(engine, ty):
    """An infinite value decides that element of every row that sees it, and of no other."""
    p = Problem(ty, ty, [(40, 90)], 2, 1, 64, 16, seed=5)
    values = p.cache[:, 16 * 64:].view(-1, 1, 64, 16)
    values[p.tables[0, 70 // 16], 0, 9, 70 % 16] = float("inf")
    values[p.tables[0, 75 // 16], 0, 9, 75 % 16] = -float("inf")
    got = p.run(engine).double().numpy().reshape(40, 2, 64)
    assert np.all(np.isfinite(got[:20])) and np.all(np.isfinite(np.delete(got, 9, axis=2)))
    assert np.all(got[20:25, :, 9] == np.inf) and np.all(np.isnan(got[25:, :, 9]))


def test_entries_outside_the_cache_are_zeros(engine):
    p = Problem(BF16, BF16, [(90, 90), (5, 200)], 4, 2, 128, 32, seed=8)
    p.tables[0, 1], p.tables[1, 0], p.tables[1, 3] = -1, p.n_pages, 2**31 - 1
    p.check(engine)


def test_lengths_past_the_table(engine):
    p = Problem(F16, F16, [(6, 64)], 4, 2, 64, 16, seed=9)
    p.lens[0] = 2**31 - 1  # as 64
    p.check(engine)
    p.lens[0], p.seqs = -5, [(6, -5)]
    got = p.run(engine)
    assert torch.all(got == 0)
    p.width, p.tables = 0, np.zeros((1, 0), np.int32)
    p.lens[0] = 64
    kv, wide = engine.kv_desc(F16, 2, 64, 16, p.n_pages), 256
    out = put(engine, torch.full((6, wide), 5.0).half())
    engine.attn_prompt_dev(engine.attn_prompt_desc(F16, 6, 1, 4, 0.125, 0), kv, put(engine, p.q), 0, put(engine, p.cache), 0,
                           ints(engine, [0, 6]), 0, ints(engine, [64]), 0, out, 0, out, 0)
    assert torch.all(get(out, torch.float16, (6, wide)) == 0)


def test_starts_that_do_not_ascend(engine):
    """Bad lists: no access outside, rows of no sequence stay, the good sequence is right where no other writes."""
    p = Problem(F16, F16, [(20, 20), (20, 20)], 4, 2, 64, 16, seed=10)
    want, bound = p.want()
    p.starts = np.array([0, 20, -3], np.int32)  # the second one ends before it begins
    got = p.run(engine, tokens=50)
    check(got[:20].reshape(20, 4, 64), want[:20], bound[:20], F16)
    assert torch.all(got[20:] == 5.0)
    p.starts = np.array([0, 20, 2**31 - 1], np.int32)  # it ends with the rows
    got = p.run(engine, tokens=50)
    check(got[:20].reshape(20, 4, 64), want[:20], bound[:20], F16)


@pytest.mark.parametrize("count", [2, 63, 64, 65, 300])
def test_many_sequences(engine, count):
    """As many as are put in order, and more than the search takes at once; many of them empty, some long."""
    rng = np.random.default_rng(count)
    new = rng.integers(0, 3, count) * rng.choice([1, 1, 1, 40], count)
    seqs = [(int(n), int(n) + int(m)) for n, m in zip(new, rng.integers(-5, 20, count))]
    Problem(F32, F32, seqs, 2, 1, 64, 16, seed=6).check(engine)
    Problem(BF16, BF16, seqs, 64, 1, 64, 16, seed=7).check(engine)  # two tokens a tile


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_as_many_tiles_as_can_be(engine, ty):
    """Every sequence ends one row into a tile: of 64 the last slot is taken.  More workgroups than CUs and at most twice as
    many, of one sequence and of many, some with parts; whole tiles only."""
    for seqs, heads, kvh, dim in [([(17, 17)] * 64, 8, 1, 64), ([(33, 40), (1, 300)] * 32, 4, 1, 64), ([(17, 19)] * 65, 8, 1, 64),
                                  ([(1100, 1100)], 32, 32, 80), ([(256, 256)], 16, 4, 128), ([(129, 200)] * 10, 16, 16, 96),
                                  ([(300, 2000), (20, 4000)], 28, 14, 64), ([(512, 512)], 8, 2, 128)]:
        print(f"[case] prompt {ty} {len(seqs)} of {seqs[0]} {heads} {kvh} {dim}", flush=True)
        Problem(ty, ty, seqs, heads, kvh, dim, 32, seed=23).check(engine)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_tables_with_room(engine, ty):
    """Tables for many more tokens than there are: parts without keys, tiles of one part beside tiles of many, both sides
    of where one is enough."""
    for seqs, dim in [([(100, 100)], 128), ([(3, 120), (40, 300), (0, 0), (1, 1), (5, 3)], 64), ([(1, 128), (1, 129), (1, 32), (1, 33)], 64),
                      ([(200, 200)], 80), ([(33, 1025), (64, 64)], 256)]:
        print(f"[case] prompt {ty} {seqs} {dim}", flush=True)
        p = Problem(ty, ty, seqs, 8, 2, dim, 64, seed=29, width=500)
        first = p.check(engine)
        p.seqs, p.lens[:] = [(n, min(length, n)) for n, length in p.seqs], np.minimum(p.lens, [n for n, _ in seqs])
        p.check(engine)
        p.seqs, p.lens[:] = seqs, [length for _, length in seqs]
        assert torch.equal(first, p.run(engine))


def test_captured(engine):
    """A captured prompt follows what its lists and queries hold at each replay; split keys and whole ones."""
    for seqs, page in [([(9, 900), (30, 64), (1, 70)], 16), ([(60, 60), (70, 80)], 64)]:
        p = Problem(BF16, BF16, seqs, 8, 2, 128, page, seed=15)
        wide, kv = 1024, engine.kv_desc(BF16, 2, 128, page, p.n_pages)
        b = {k: put(engine, v) for k, v in (("q", p.q), ("cache", p.cache), ("out", torch.zeros(p.tokens, wide).bfloat16()))}
        starts, lens, tables = ints(engine, p.starts.tolist()), ints(engine, p.lens.tolist()), ints(engine, p.tables.reshape(-1).tolist())
        d = engine.attn_prompt_desc(BF16, p.tokens, len(seqs), 8, p.scale, p.width)

        def call():
            engine.attn_prompt_dev(d, kv, b["q"], 0, b["cache"], 0, starts, 0, lens, 0, tables, 0, b["out"], 0)

        call()
        graph = engine.capture(call)
        for step in range(3):
            cut = [p.tokens // 3 + step, 0, 0][:len(seqs)]
            new = [cut[0], p.tokens - cut[0]] + [0] * (len(seqs) - 2)
            p.seqs = [(n, length) for n, (_, length) in zip(new, seqs)]
            p.starts = np.cumsum([0] + new).astype(np.int32)
            p.q = normal(step + 30, p.tokens, wide).bfloat16()
            starts.write(p.starts)
            b["q"].write(p.q.view(torch.uint8).numpy())
            graph.launch()
            want, bound = p.want()
            check(get(b["out"], torch.bfloat16, want.shape), want, bound, BF16)
            eager = get(b["out"], torch.bfloat16, (p.tokens, wide))
            call()
            assert torch.equal(eager, get(b["out"], torch.bfloat16, (p.tokens, wide)))
        graph.free()


def test_captured_first_of_all():
    """An engine's first call is captured, with more workgroups than CUs and at most twice as many."""
    p = Problem(F16, F16, [(1100, 1100)], 32, 32, 64, 64, seed=31)
    want, bound = p.want()
    engine = HipEngine(0)
    wide, kv = 32 * 64, engine.kv_desc(F16, 32, 64, 64, p.n_pages)
    q, cache, out = put(engine, p.q), put(engine, p.cache), put(engine, torch.zeros(p.tokens, wide).half())
    starts, lens, tables = ints(engine, p.starts.tolist()), ints(engine, p.lens.tolist()), ints(engine, p.tables.reshape(-1).tolist())
    d = engine.attn_prompt_desc(F16, p.tokens, 1, 32, p.scale, p.width)
    graph = engine.capture(lambda: engine.attn_prompt_dev(d, kv, q, 0, cache, 0, starts, 0, lens, 0, tables, 0, out, 0))
    for _ in range(3):
        out.write(torch.zeros(p.tokens, wide).half().view(torch.uint8).numpy())
        graph.launch()
        check(get(out, torch.float16, want.shape), want, bound, F16)
    graph.free()
    engine.close()


def test_large_scores(engine):
    """Scores far apart, growing along the keys: the running base has to follow."""
    for ty in (F32, F16, BF16):
        p = Problem(ty, ty, [(3, 900)], 2, 1, 64, 16, seed=11, scale=1.0)
        keys = p.cache[:, :16 * 64].view(-1, 16, 64)
        for t in range(900):
            keys[p.tables[0, t // 16], t % 16] *= 0.2 + t / 150
        p.check(engine)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("likely", [3, 29990])
def test_many_small_weights(engine, ty, likely):
    """30000 tokens of e^-17.5: 8e-4 together, each below f16's smallest number."""
    p = Problem(ty, ty, [(5, 30001)], 2, 1, 64, 64, seed=17)
    far_smaller(p, likely, 17.5)
    p.check(engine)


def test_far_pages(engine):
    """Pages three gigabytes apart: offsets past 32 bits."""
    kvh, dim, page, n_pages = 2, 128, 64, 4
    per, stride = page_elements(kvh, dim, page), 3 << 29
    p = Problem(BF16, BF16, [(40, 200)], 8, kvh, dim, page, seed=12, spare=0)
    b = engine.alloc(((n_pages - 1) * stride + per) * 2)
    for i in range(n_pages):
        b.write(p.cache[i].view(torch.uint8).numpy(), i * stride * 2)
    kv = engine.kv_desc(BF16, kvh, dim, page, n_pages, stride)
    out = engine.alloc(40 * 1024 * 2)
    engine.attn_prompt_dev(engine.attn_prompt_desc(BF16, 40, 1, 8, p.scale, p.width), kv, put(engine, p.q), 0, b, 0,
                           ints(engine, [0, 40]), 0, ints(engine, [200]), 0, ints(engine, p.tables[0].tolist()), 0, out, 0)
    want, bound = p.want()
    check(get(out, torch.bfloat16, want.shape), want, bound, BF16)
    b.free()


def test_same_bits_every_time(engine):
    p = Problem(BF16, BF16, [(5, 3000), (60, 60)], 8, 2, 128, 64, seed=13)
    first = p.run(engine)
    for _ in range(3):
        assert torch.equal(first, p.run(engine))


def test_refusals(engine):
    b = engine.alloc(1 << 16)
    kv = engine.kv_desc(F16, 2, 64, 16, 2)
    good = dict(ggml_type=F16, tokens=4, seqs=1, q_heads=4, scale=0.125, table_stride=2)

    def call(kv=kv, starts=b, **changes):
        engine.attn_prompt_dev(engine.attn_prompt_desc(**{**good, **changes}), kv, b, 0, b, 0, starts, 0, b, 0, b, 0, b, 0)

    small = engine.alloc(4)
    for status, changes in [(3, dict(ggml_type=2)), (3, dict(ggml_type=BF16)), (2, dict(scale=0.0)), (2, dict(scale=float("nan"))),
                            (2, dict(scale=float("inf"))), (2, dict(q_heads=3)), (2, dict(q_heads=0)), (2, dict(q_heads=130)),
                            (2, dict(tokens=1 << 12)), (2, dict(q_stride=255)), (2, dict(out_stride=255)), (2, dict(seqs=1 << 20)),
                            (2, dict(table_stride=1 << 33)), (2, dict(tokens=1 << 40)), (2, dict(starts=small)),
                            (3, dict(kv=engine.kv_desc(8, 2, 64, 16, 2))), (2, dict(kv=engine.kv_desc(F16, 0, 64, 16, 2))),
                            (2, dict(kv=engine.kv_desc(F16, 2, 63, 16, 2))), (2, dict(kv=engine.kv_desc(F16, 2, 264, 16, 2))),
                            (2, dict(kv=engine.kv_desc(F16, 2, 64, 24, 2))), (2, dict(kv=engine.kv_desc(F16, 2, 64, 8, 2))),
                            (2, dict(kv=engine.kv_desc(F16, 2, 64, 512, 2))), (2, dict(kv=engine.kv_desc(F16, 2, 64, 16, 0))),
                            (2, dict(kv=engine.kv_desc(F16, 2, 64, 16, 1 << 28))), (2, dict(kv=engine.kv_desc(F16, 2, 64, 16, 9))),
                            (2, dict(kv=engine.kv_desc(F16, 2, 64, 16, 2, 4095))), (2, dict(kv=engine.kv_desc(F16, 2, 64, 16, 2, 4100)))]:
        with pytest.raises(HipError) as err:
            call(**changes)
        assert err.value.status == status, changes
    with pytest.raises(HipError):
        engine.attn_prompt_dev(engine.attn_prompt_desc(**good), kv, b, 0, b, 8, b, 0, b, 0, b, 0, b, 0)


@pytest.mark.parametrize("ty,cty", TYPES)
def test_scores_of_minus_infinity(engine, ty, cty):
    """The first `low` keys score minus infinity: weights of 0 in rows that see another key, NaN (0 / 0) in rows that see these
    alone, zeros in rows that see none."""
    for i, (seqs, low, heads, kvh, dim, page) in enumerate([([(40, 40)], [20], 4, 2, 64, 16), ([(3, 2500), (5, 3)], [2498, 3], 8, 2, 128, 64),
                                                            ([(200, 1200)], [1000 + 64], 8, 1, 128, 32), ([(30, 30), (3, 90)], [30, 0], 3, 1, 72, 32),
                                                            ([(60, 40)], [33], 1, 1, 64, 64)]):
        p = Problem(ty, cty, seqs, heads, kvh, dim, page, seed=40 + i)
        p.q[:, ::dim] = p.q[:, ::dim].abs() + 0.5
        finite = p.cache.clone()
        keys = p.cache[:, :kvh * page * dim].view(-1, kvh, page, dim)
        for s, n in enumerate(low):
            for t in range(n):
                keys[p.tables[s, t // page], :, t % page, 0] = -float("inf")
        got = p.run(engine)[:p.tokens].reshape(-1, heads, dim)
        q = p.q.double().numpy().reshape(-1, heads, dim)
        for s, (n, length) in enumerate(seqs):
            rows, seen = slice(p.starts[s], p.starts[s] + n), length - n + 1 + np.arange(n)
            k, v = gather(finite, p.tables[s], length, kvh, dim, page)
            want, bound = attend(q[rows], k[low[s]:], v[low[s]:], seen - low[s], p.scale, ty, cty)
            blind, lost = seen <= 0, (seen > 0) & (seen <= low[s])
            assert torch.all(got[rows][blind] == 0), (i, s)
            assert torch.all(torch.isnan(got[rows][lost])), (i, s)
            rest = ~blind & ~lost
            check(got[rows][rest], want[rest], bound[rest], ty)
