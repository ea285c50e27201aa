"""GPU tests of a decode batch's attention over pages (attn_decode), with and without shared tokens, against
its definition in 64 bits; the bounds' derivation stands in attn_reference.py."""
import os

import numpy as np
import pytest
import torch

from attn_reference import DT, attend, check, gather, page_elements
from hayai_amd import BF16, F16, F32, HipEngine, HipError
from test_gpu_attn_pages import get, ints, normal, put

pytestmark = pytest.mark.gpu

TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]


class Batch:
    """Sequences of lens cached tokens, the first `prefix` of each the same: whole pages shared, the page that the
    prefix ends in copied."""

    def __init__(self, ty, cty, lens, prefix, heads, kvh, dim, page, seed=0, pad=0, scale=None, width=None):
        self.ty, self.cty, self.prefix, self.heads, self.kvh, self.dim, self.page, self.pad = ty, cty, prefix, heads, kvh, dim, page, pad
        self.lens = np.array(lens, np.int64)
        rng = np.random.default_rng(seed)
        per = page_elements(kvh, dim, page)
        whole = prefix // page
        need = [max(0, -(-int(n) // page) - whole) for n in lens]
        shared_pages = -(-prefix // page)
        self.n_pages = shared_pages + sum(need) + 2
        ids = rng.permutation(self.n_pages)
        self.shared = ids[:shared_pages].astype(np.int32)
        self.width = max([whole + n for n in need] + [1]) if width is None else width
        self.tables = np.full((len(lens), self.width), 2**31 - 1, np.int32)
        self.cache = normal(seed + 1, self.n_pages, per).to(DT[cty])
        at = shared_pages
        for s, n in enumerate(need):
            row = list(self.shared[:whole]) + list(ids[at:at + n])
            at += n
            if lens[s] <= 0:
                continue
            if lens[s] < prefix:  # a sequence of its own, where other tokens are
                row = list(ids[rng.permutation(self.n_pages)[:-(-int(lens[s]) // page)]])
            self.tables[s, :len(row)] = row[:self.width]
            end = prefix % page
            if end and n and lens[s] >= prefix:
                k, v = (c.view(-1, *shape) for c, shape in zip((self.cache[:, :per // 2], self.cache[:, per // 2:]),
                                                              ((kvh, page, dim), (kvh, dim, page))))
                k[row[whole], :, :end] = k[self.shared[-1], :, :end]
                v[row[whole], :, :, :end] = v[self.shared[-1], :, :, :end]
        self.q = normal(seed + 2, len(lens), heads * dim + pad).to(DT[ty])
        self.scale = float(np.float32(dim**-0.5 if scale is None else scale))

    def upload(self, engine):
        wide = self.heads * self.dim + self.pad
        self.kv = engine.kv_desc(self.cty, self.kvh, self.dim, self.page, self.n_pages)
        self.desc = engine.attn_decode_desc(self.ty, len(self.lens), self.heads, self.scale, self.width, self.prefix, wide, wide)
        self.buffers = {"q": put(engine, self.q), "cache": put(engine, self.cache),
                        "shared": ints(engine, self.shared.tolist()) if self.prefix else None,
                        "lens": ints(engine, self.lens.tolist()), "tables": ints(engine, self.tables.reshape(-1).tolist()),
                        "out": put(engine, torch.full((len(self.lens), wide), 5.0).to(DT[self.ty]))}

    def call(self, engine):
        b = self.buffers
        engine.attn_decode_dev(self.desc, self.kv, b["q"], 0, b["cache"], 0, b["shared"], 0, b["lens"], 0, b["tables"], 0, b["out"], 0)

    def read(self):
        return get(self.buffers["out"], DT[self.ty], (len(self.lens), self.heads * self.dim + self.pad))

    def run(self, engine):
        self.upload(engine)
        self.call(engine)
        return self.read()

    def want(self):
        q = self.q[:, :self.heads * self.dim].double().numpy().reshape(-1, self.heads, self.dim)
        out, bound = np.zeros_like(q), np.zeros_like(q)
        for s, n in enumerate(self.lens):
            n = int(min(max(n, 0), self.width * self.page))
            k, v = gather(self.cache, self.tables[s], n, self.kvh, self.dim, self.page)
            out[s:s + 1], bound[s:s + 1] = attend(q[s:s + 1], k, v, [n], self.scale, self.ty, self.cty)
        return out, bound

    def check(self, got):
        want, bound = self.want()
        check(got[:, :self.heads * self.dim].reshape(want.shape), want, bound, self.ty)
        assert torch.all(got[:, self.heads * self.dim:] == 5.0)


# lens, heads, kv heads, dim, page: one token, a unit's and a step's edges, one long sequence, ragged batches with
# empty rows, groups of 1, 3, 7, 20, 64 heads, partly filled heads
OWN = [([1], 1, 1, 64, 16), ([128, 129, 31, 32, 33], 8, 2, 128, 32), ([3001], 32, 8, 128, 64), ([5, 0, 700, -3, 64], 9, 3, 64, 16),
       ([400, 17], 7, 1, 72, 16), ([260, 1], 20, 1, 256, 256), ([90, 2000, 16], 64, 1, 64, 128), ([255], 6, 6, 96, 64),
       ([77, 513], 4, 2, 8, 16), ([300], 3, 1, 200, 32)]


@pytest.mark.parametrize("ty,cty", TYPES)
def test_own(engine, ty, cty):
    for i, (lens, heads, kvh, dim, page) in enumerate(OWN):
        print(f"[case] decode {ty} {cty} {OWN[i]}", flush=True)
        b = Batch(ty, cty, lens, 0, heads, kvh, dim, page, seed=i, pad=i % 3)
        b.check(b.run(engine))


# lens, prefix: whole tiles and pages or not, suffixes of none, sequences shorter than the prefix, empty rows, more
# rows than a tile holds
SHARED = [([300, 290, 257], 256, 8, 2, 128, 64), ([1000, 700, 699], 699, 4, 4, 64, 16), ([900, 20, 0, 650, 640], 640, 9, 3, 64, 32),
          ([600 + i for i in range(40)], 590, 8, 1, 128, 128), ([512, 512], 512, 2, 1, 72, 16), ([350, 400], 300, 20, 1, 256, 64),
          ([100, 90], 80, 4, 2, 64, 16), ([700], 600, 4, 2, 128, 32), ([270, 333, 5], 265, 6, 2, 96, 256),
          ([1300, 1290, 1290], 1281, 64, 1, 64, 64)]


@pytest.fixture(scope="module")
def sharing():
    """An engine that takes shared tokens apart however few they are."""
    os.environ["HAYAI_HIP_ATTN_SHARE_MIN"] = "0"
    try:
        e = HipEngine(0)
    finally:
        del os.environ["HAYAI_HIP_ATTN_SHARE_MIN"]
    yield e
    e.close()


@pytest.mark.parametrize("ty,cty", TYPES)
def test_shared(engine, sharing, ty, cty):
    for i, (lens, prefix, heads, kvh, dim, page) in enumerate(SHARED):
        print(f"[case] decode {ty} {cty} {SHARED[i]}", flush=True)
        b = Batch(ty, cty, lens, prefix, heads, kvh, dim, page, seed=i, pad=i % 2)
        b.check(b.run(sharing))
        b.check(b.run(engine))


@pytest.mark.parametrize("ty,cty", TYPES)
def test_shared_by_many(engine, ty, cty):
    """As many bytes as are taken apart by default."""
    lens = [700 + 3 * i for i in range(70)]
    lens[5], lens[20], lens[69] = 0, 100, 690
    b = Batch(ty, cty, lens, 690, 8, 4, 128, 64, seed=40)
    assert 69 * 690 * 8 * 128 * torch.empty(0, dtype=DT[cty]).element_size() >= 24 << 20
    b.check(b.run(engine))


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_slots_past_the_length(sharing, ty, bad):
    for lens, prefix, page in [([50, 130, 1], 0, 16), ([400, 300, 20, 265], 265, 64)]:
        b = Batch(ty, ty, lens, prefix, 4, 2, 128, page, seed=3)
        want, bound = b.want()
        per, used = page_elements(2, 128, page), set(b.shared.tolist())
        for s, n in enumerate(lens):
            used |= set(b.tables[s, :-(-n // page)].tolist())
        for other in range(b.n_pages):
            if other not in used:
                b.cache[other] = bad
        for s, n in enumerate(lens):
            if n % page and b.tables[s, n // page] not in b.shared and lens[s] >= prefix:
                b.cache[b.tables[s, n // page], :per // 2].view(2, page, 128)[:, n % page:] = bad
                b.cache[b.tables[s, n // page], per // 2:].view(2, 128, page)[:, :, n % page:] = bad
        got = b.run(sharing).reshape(want.shape)
        keep = [s for s, n in enumerate(lens) if n >= prefix]  # (the others lie in any page)
        check(got[keep], want[keep], bound[keep], ty)


def test_entries_outside_the_cache_are_zeros(sharing):
    b = Batch(BF16, BF16, [400, 300, 380], 256, 8, 2, 128, 32, seed=4)
    b.shared[3] = -1
    b.tables[:, 3] = -9
    b.tables[0, 10], b.tables[2, 9] = b.n_pages, -2**31
    b.check(b.run(sharing))
    b = Batch(F32, F32, [40, 300], 0, 4, 2, 72, 16, seed=5)
    b.tables[0, 1], b.tables[1, 0] = -1, b.n_pages
    b.check(b.run(sharing))


def test_lengths_past_the_table(sharing):
    for prefix in (0, 256):
        b = Batch(F16, F16, [320, 320], prefix, 4, 2, 64, 16, seed=6)
        b.lens[0] = 2**31 - 1  # as 320
        b.check(b.run(sharing))
        b.width, b.tables = 0, np.zeros((2, 0), np.int32)
        assert torch.all(b.run(sharing) == 0)


def test_more_sequences_than_threads(sharing):
    rng = np.random.default_rng(7)
    for prefix in (0, 320):
        lens = [int(n) if i % 5 else int(n) // 60 for i, n in enumerate(prefix + rng.integers(0, 90, 600))]
        b = Batch(F32, F32, lens, prefix, 2, 1, 64, 16, seed=7)
        b.check(b.run(sharing))


def test_one_long_among_short(engine):
    b = Batch(BF16, BF16, [9000] + [30] * 20, 0, 8, 2, 64, 64, seed=8)
    b.check(b.run(engine))


def test_large_scores(sharing):
    for ty in (F32, F16, BF16):
        b = Batch(ty, ty, [900, 650], 600, 2, 1, 64, 16, seed=9, scale=1.0)
        keys = b.cache[:, :16 * 64].view(-1, 16, 64)
        for t in range(600):
            keys[b.shared[t // 16], t % 16] *= 0.2 + t / 100
        for s in range(2):  # the copies of the page that the prefix ends in, if any, hold the same
            assert 600 % 16 == 8
            keys[b.tables[s, 37], :8] = keys[b.shared[37], :8]
        b.check(b.run(sharing))


def far_smaller(b, likely, rest):
    """One token with a weight of 1 and a value of 0, the others with a weight of exp(-rest) and values of 1."""
    b.q[:] = 0
    b.q[:, ::b.dim] = 8.0
    per = b.cache.shape[1] // 2
    b.cache[:, :per], b.cache[:, per:] = 0, 1.0
    page, at = divmod(likely, b.page)
    for table in b.tables:
        b.cache[table[page], :per].view(b.kvh, b.page, b.dim)[:, at, 0] = rest / b.scale / 8
        b.cache[table[page], per:].view(b.kvh, b.dim, b.page)[:, :, at] = 0


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("prefix,likely", [(0, 3), (0, 30000), (29952, 7), (29952, 29990)])
def test_many_small_weights(sharing, ty, prefix, likely):
    """30000 tokens of e^-17.5: 8e-4 together, each below f16's smallest number."""
    b = Batch(ty, ty, [30001, 30005], prefix, 2, 1, 64, 64, seed=17)
    far_smaller(b, likely, 17.5)
    b.check(b.run(sharing))


def test_prefix_is_as_good_as_none(sharing):
    """The same batch with and without the hint: equal up to the order of sums and one rounding."""
    b = Batch(F16, F16, [2100, 2055, 2060, 2200], 2050, 8, 2, 128, 64, seed=10)
    with_prefix = b.run(sharing)
    b.check(with_prefix)
    b.prefix = 0
    b.check(b.run(sharing))


def test_far_pages(engine):
    kvh, dim, page = 2, 128, 64
    per, stride = page_elements(kvh, dim, page), 3 << 29
    b = Batch(BF16, BF16, [200, 130], 0, 8, kvh, dim, page, seed=12)
    b.n_pages = 6
    b.tables = np.array([[5, 0, 3, 1], [2, 4, 1, -1]], np.int32)[:, :b.width]
    cache = engine.alloc((5 * stride + per) * 2)
    b.cache = normal(3, 6, per).to(torch.bfloat16)
    for i in range(6):
        cache.write(b.cache[i].view(torch.uint8).numpy(), i * stride * 2)
    out = engine.alloc(2 * 1024 * 2)
    engine.attn_decode_dev(engine.attn_decode_desc(BF16, 2, 8, b.scale, b.width), engine.kv_desc(BF16, kvh, dim, page, 6, stride),
                           put(engine, b.q), 0, cache, 0, None, 0, ints(engine, [200, 130]), 0,
                           ints(engine, b.tables.reshape(-1).tolist()), 0, out, 0)
    want, bound = b.want()
    check(get(out, torch.bfloat16, want.shape), want, bound, BF16)
    cache.free()


@pytest.mark.parametrize("apart", [True, False])
def test_captured(engine, sharing, apart):
    """A captured step follows the lengths, pages and queries of each replay; another graph and eager calls use the same
    workspace between the replays."""
    engine = sharing if apart else engine
    b = Batch(BF16, BF16, [700, 330, 400], 320, 8, 2, 128, 32, seed=13, width=40)
    c = Batch(F32, F32, [1000, 90], 0, 4, 2, 64, 16, seed=14)
    graphs = []
    for x in (b, c):
        x.check(x.run(engine))
        graphs.append(engine.capture(lambda: x.call(engine)))
    big = Batch(F16, F16, [3000] * 30, 1024, 32, 4, 128, 64, seed=15)
    for step in range(4):
        b.lens[:] = [320 + 31 * step, 0 if step == 2 else 1100, 321]
        b.tables[:, 10:] = np.random.default_rng(step).integers(0, b.n_pages, (3, 30))
        b.q = normal(step + 50, *b.q.shape).to(torch.bfloat16)
        b.buffers["lens"].write(b.lens.astype(np.int32))
        b.buffers["tables"].write(b.tables)
        b.buffers["q"].write(b.q.view(torch.uint8).numpy())
        graphs[0].launch()
        graphs[1].launch()
        if step == 1:
            big.run(engine)  # a larger workspace
        b.check(b.read())
        c.check(c.read())
        eager = b.read()
        b.call(engine)
        assert torch.equal(eager, b.read())
    for g in graphs:
        g.free()


def test_same_bits_every_time(sharing):
    b = Batch(F16, F16, [900, 800, 770], 700, 8, 2, 128, 64, seed=16)
    first = b.run(sharing)
    for _ in range(3):
        assert torch.equal(first, b.run(sharing))


def test_no_sequences(engine):
    b = engine.alloc(1 << 14)
    b.fill(0x5B)
    engine.attn_decode_dev(engine.attn_decode_desc(F16, 0, 4, 0.125, 2), engine.kv_desc(F16, 2, 64, 16, 1), b, 0, b, 0, None, 0,
                           b, 0, b, 0, b, 0)
    assert np.all(b.read(np.uint8, 1 << 14) == 0x5B)


def test_refusals(engine):
    b, small = engine.alloc(1 << 16), engine.alloc(4)
    good = dict(ggml_type=F16, seqs=4, q_heads=4, scale=0.125, table_stride=2)

    def call(kv=engine.kv_desc(F16, 2, 64, 16, 2), prefix_pages=None, lens=b, tables=b, **changes):
        engine.attn_decode_dev(engine.attn_decode_desc(**{**good, **changes}), kv, b, 0, b, 0, prefix_pages, 0, lens, 0, tables, 0,
                               b, 0)

    for status, changes in [(3, dict(ggml_type=2)), (3, dict(ggml_type=BF16)), (2, dict(scale=-1.0)), (2, dict(scale=float("nan"))),
                            (2, dict(q_heads=3)), (2, dict(q_heads=130)), (2, dict(seqs=1 << 12)), (2, dict(seqs=1 << 40)),
                            (2, dict(q_stride=255)), (2, dict(out_stride=255)), (2, dict(table_stride=1 << 33)),
                            (2, dict(prefix=32)), (2, dict(prefix=32, prefix_pages=small)), (2, dict(prefix=1 << 40, prefix_pages=b)),
                            (2, dict(lens=small)), (2, dict(tables=small)), (2, dict(kv=engine.kv_desc(F16, 2, 64, 24, 2))),
                            (2, dict(kv=engine.kv_desc(F16, 2, 64, 16, 9))), (3, dict(kv=engine.kv_desc(2, 2, 64, 16, 2)))]:
        with pytest.raises(HipError) as err:
            call(**changes)
        assert err.value.status == status, changes


# prefix, heads, kv heads, dim, page: no multiples of 64, so that what is taken apart is less than what is shared; one under 64
NEARLY = [(699, 4, 4, 64, 16), (690, 8, 2, 128, 64), (590, 8, 1, 128, 128), (265, 6, 2, 96, 256), (1281, 64, 1, 64, 64), (65, 9, 3, 72, 16),
          (63, 4, 2, 64, 32)]


def around(prefix):
    """Lengths on both sides of the prefix and of the whole 64 tokens in it."""
    whole = prefix // 64 * 64
    return [prefix + 90, whole - 1, whole, whole + 1, (whole + prefix) // 2, prefix - 1, prefix, prefix + 1]


@pytest.mark.parametrize("ty,cty", TYPES)
def test_nearly_the_prefix(sharing, ty, cty):
    """Sequences of a few tokens less than the prefix have tokens of their own, in their own tables alone."""
    for i, (prefix, heads, kvh, dim, page) in enumerate(NEARLY):
        print(f"[case] decode {ty} {cty} {NEARLY[i]}", flush=True)
        b = Batch(ty, cty, around(prefix), prefix, heads, kvh, dim, page, seed=50 + i)
        b.check(b.run(sharing))


@pytest.mark.parametrize("ty,cty", TYPES)
def test_nearly_the_prefix_by_many(engine, ty, cty):
    """The same with as many bytes as are taken apart by default."""
    lens = [700 + 3 * i for i in range(70)]
    lens[1], lens[7], lens[30], lens[31], lens[69] = 640, 689, 641, 639, 665
    b = Batch(ty, cty, lens, 690, 8, 4, 128, 64, seed=60)
    b.check(b.run(engine))


def test_nearly_the_prefix_captured(sharing):
    """Lengths that pass the prefix in both directions from replay to replay."""
    b = Batch(BF16, BF16, [900, 689, 689, 760, 689], 690, 8, 2, 128, 32, seed=61)
    b.check(b.run(sharing))
    graph = sharing.capture(lambda: b.call(sharing))
    for step, lens in enumerate([[700, 640, 641, 690, 689], [640, 639, 689, 689, 300], [900, 0, 645, 650, 688], [690, 689, 640, 760, 1]]):
        b.lens[:] = lens
        b.q = normal(step + 62, *b.q.shape).to(torch.bfloat16)
        b.buffers["lens"].write(b.lens.astype(np.int32))
        b.buffers["q"].write(b.q.view(torch.uint8).numpy())
        graph.launch()
        got = b.read()
        b.check(got)
        b.call(sharing)
        assert torch.equal(got, b.read())
    graph.free()


@pytest.mark.parametrize("ty,cty", TYPES)
def test_scores_of_minus_infinity(sharing, ty, cty):
    """The first `low` keys of each sequence score minus infinity: weights of 0 where another key is seen, else NaN (0 / 0)."""
    for i, (lens, low, prefix, heads, kvh, dim, page) in enumerate([
            ([50, 50, 1, 0], [20, 50, 1, 0], 0, 4, 2, 64, 16), ([3000, 3000, 200], [2500, 3000, 190], 0, 8, 2, 128, 64),
            ([700, 750, 640], [660, 750, 640], 640, 8, 2, 128, 32), ([40, 300], [40, 131], 0, 3, 1, 72, 32)]):
        b = Batch(ty, cty, lens, prefix, heads, kvh, dim, page, seed=70 + i)
        b.q[:, ::dim] = b.q[:, ::dim].abs() + 0.5
        keys = b.cache[:, :kvh * page * dim].view(-1, kvh, page, dim)
        finite = keys.clone()
        for s, n in enumerate(low):
            for t in range(n):
                keys[b.tables[s, t // page], :, t % page, 0] = -float("inf")
        for t in range(min(low) if prefix else 0, prefix):  # (shared pages: what one sequence changes holds for all)
            assert keys[b.shared[t // page], 0, t % page, 0] == -float("inf")
        got = b.run(sharing)[:, :heads * dim].reshape(-1, heads, dim)
        q = b.q.double().numpy().reshape(-1, heads, dim)
        for s, n in enumerate(lens):
            if n and low[s] == n:
                assert torch.all(torch.isnan(got[s])), (i, s)
                continue
            k, v = gather(torch.cat([finite.flatten(1), b.cache[:, kvh * page * dim:]], 1), b.tables[s], n, kvh, dim, page)
            want, bound = attend(q[s:s + 1], k[low[s]:], v[low[s]:], [n - low[s]], b.scale, ty, cty)
            check(got[s:s + 1], want, bound, ty)
