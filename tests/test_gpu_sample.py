"""GPU tests of the choice of the next token (hh_sample_dev) against its definition in 64 bits.

Ids have to equal the oracle's wherever its decisions are not within 1e-9 of a border (weights are
whole multiples of 2^-42 on the GPU, so a share of the weight is up to vocab * 2^-42 off there).
Probabilities: that, and one f32 rounding.
"""
import numpy as np
import pytest
import torch

import hayai_amd
from hayai_amd import BF16, F16, F32

pytestmark = pytest.mark.gpu

DT = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}


def oracle(logits, temperature, top_k, top_p, min_p, u):
    """(id, probability, how near a decision was to going the other way)."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, 1.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(x == top, 1.0, 0.0 if top == np.inf else np.exp((x - top) / np.float64(temperature)))
    near, s = 1.0, w[order]
    length = int(np.count_nonzero(x > -np.inf))
    if top_k > 0:
        length = min(length, top_k)
    if top_p < 1:
        run = np.cumsum(s[:length])
        before = np.concatenate([[0.0], run[:-1]])
        want = np.float64(top_p) * run[-1]
        near = min(near, float(np.min(np.abs(before[1:] - want))) / run[-1] if length > 1 else 1.0)
        length = max(1, int(np.count_nonzero(before < want)))
    if min_p > 0:
        near = min(near, float(np.min(np.abs(s[1:] - min_p) + (s[1:] == 1.0))) if len(s) > 1 else 1.0)
        length = max(1, min(length, int(np.count_nonzero(s >= min_p))))
    kept = np.zeros_like(w)
    kept[order[:length]] = s[:length]
    run = np.cumsum(kept)
    want = (min(max(float(u), 0.0), 1.0) if u == u else 0.0) * run[-1]
    edges = run[kept > 0][:-1]
    near = min(near, float(np.min(np.abs(edges - want))) / run[-1] if len(edges) else 1.0)
    at = int(np.argmax(run > want)) if want < run[-1] else int(np.flatnonzero(kept > 0)[-1])
    return at, kept[at] / run[-1], near


def sample(engine, ty, logits, params, u, pad=0, lead=0, probs=True):
    rows, vocab = logits.shape
    size = logits.element_size()
    x = torch.full((rows, vocab + pad), 1e4, dtype=DT[ty])  # what lies between rows outweighs them
    x[:, :vocab] = logits
    bx = engine.alloc(lead + x.numel() * size)
    bx.write(x.view(torch.uint8).numpy().reshape(-1), lead)
    ids, pr = engine.alloc(4 * rows + 4), engine.alloc(4 * rows + 4)
    ids.fill(0x5B)
    pr.fill(0x5B)
    d = engine.sample_desc(ty, rows, vocab, vocab + pad if pad else 0)
    engine.sample_dev(d, bx, lead, engine.upload(params), 0, engine.upload(np.asarray(u, np.float32)), 0, ids, 0,
                      pr if probs else None, 0)
    assert ids.read(np.uint8, 4, 4 * rows).tolist() == [0x5B] * 4
    assert pr.read(np.uint8, 4, 4 * rows).tolist() == [0x5B] * 4
    return ids.read(np.int32, rows), pr.read(np.float32, rows)


def check(engine, ty, logits, params, u, **kw):
    ids, probs = sample(engine, ty, logits, params, u, **kw)
    vocab = logits.shape[1]
    skipped = 0
    for r, row in enumerate(logits.float().numpy()):
        p = params[r]
        want, prob, near = oracle(row, p["temperature"], int(p["top_k"]), p["top_p"], p["min_p"], np.float32(u[r]))
        if near < 1e-9:
            skipped += 1
            continue
        assert ids[r] == want, f"row {r} {p} u={u[r]}: {ids[r]} for {want}"
        assert abs(probs[r] - prob) <= prob * (2.0**-24 + (vocab + 1) * 2.0**-42) * (1 + 1e-6), (r, probs[r], prob)
    assert skipped <= len(ids) // 8


MIX = [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 5, 1.0, 0.0),
       (0.8, 50, 0.9, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 0.999, 0.0), (1.0, 0, 0.05, 0.0), (1.0, 0, 1.0, 0.02),
       (1.5, 300, 0.95, 0.01), (1.0, 1 << 30, 0.5, 0.0), (2.5, 0, 0.98, 1e-4), (1.0, 700, 1.0, 0.0), (0.05, 40, 0.9, 0.1)]


def mixed(engine, rows, first=0):
    rows = [MIX[(first + i) % len(MIX)] for i in range(rows)]
    return engine.sample_params(*[np.array(c) for c in zip(*rows)])


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_mixed_requests(engine, ty):
    """Each row its own request; half-width logits hold many equal values."""
    rng = np.random.default_rng(3)
    for rows, vocab, pad, lead in [(15, 1, 0, 0), (15, 2, 0, 4), (30, 63, 1, 0), (30, 1000, 0, 0), (15, 4099, 3, 4),
                                   (45, 32000, 0, 0), (15, 128256, 0, 0), (1, 128256, 0, 0), (7, 151936, 8, 4)]:
        print(f"[case] sample type={ty} {rows}x{vocab}", flush=True)
        x = 2.0 * rng.standard_normal((rows, vocab))
        x[:, rng.integers(0, vocab, 20)] += 6.0
        check(engine, ty, torch.from_numpy(x).to(DT[ty]), mixed(engine, rows, vocab), rng.random(rows), pad=pad, lead=lead)


def test_flat_and_steep_rows(engine):
    """Every logit equal (ties everywhere), a plateau, one token above all, an even slope."""
    rng = np.random.default_rng(4)
    vocab = 20011
    flat = np.full(vocab, -3.25)
    plateau = np.where(np.arange(vocab) % 3 == 0, 1.0, -1.0)
    lone = np.full(vocab, -20.0)
    lone[777] = 20.0
    slope = -np.arange(vocab)[::-1] * 1e-3
    fine = -np.arange(vocab) * 1e-7
    for x in (flat, plateau, lone, slope, fine):
        logits = torch.from_numpy(np.tile(x, (len(MIX), 1))).float()
        check(engine, F32, logits, mixed(engine, len(MIX)), rng.random(len(MIX)))


def test_masks_infinities_and_nan(engine):
    rng = np.random.default_rng(5)
    vocab, n = 3001, len(MIX)
    base = 2.0 * rng.standard_normal((n, vocab))
    lowest = float(np.finfo(np.float32).min)
    for name, change in [("all but one masked", lambda x: np.where(np.arange(vocab) == 1234, x, -np.inf)),
                         ("all masked", lambda x: np.full_like(x, -np.inf)),
                         ("all nan", lambda x: np.full_like(x, np.nan)),
                         ("nan and -inf", lambda x: np.where(np.arange(vocab) % 2, x, np.nan)),
                         ("half -inf", lambda x: np.where(np.arange(vocab) % 2, x, -np.inf)),
                         ("lowest of the type", lambda x: np.where(np.arange(vocab) % 5 == 1, x, lowest)),
                         ("all lowest", lambda x: np.full_like(x, lowest)),
                         ("+inf twice", lambda x: np.where((np.arange(vocab) == 7) | (np.arange(vocab) == 2999), np.inf, x)),
                         ("signed zeros", lambda x: np.where(np.arange(vocab) % 2, 0.0, -0.0)),
                         ("far apart", lambda x: x * 1e37)]:
        print(f"[case] {name}", flush=True)
        check(engine, F32, torch.from_numpy(np.broadcast_to(change(base), base.shape).copy()).float(), mixed(engine, n), rng.random(n))


def test_ends_of_u_and_odd_parameters(engine):
    rng = np.random.default_rng(6)
    x = 2.0 * rng.standard_normal((1, 5003))
    nan, inf = float("nan"), float("inf")
    cases = [(1.0, 0, 1.0, 0.0, u) for u in (0.0, -1.0, nan, 1.0, 7.0, inf, np.nextafter(np.float32(1), np.float32(0)))]
    cases += [(1.0, 30, 0.9, 0.0, u) for u in (0.0, 1.0)]
    cases += [(nan, 0, 1.0, 0.0, 0.9), (-1.0, 0, 1.0, 0.0, 0.9), (inf, 0, 1.0, 0.0, 0.4), (1e-30, 0, 1.0, 0.0, 0.9),
              (1e30, 0, 0.5, 0.0, 0.9), (1.0, -5, 1.0, 0.0, 0.3), (1.0, 0, nan, 0.0, 0.3), (1.0, 0, 0.0, 0.0, 0.3),
              (1.0, 0, -1.0, 0.0, 0.3), (1.0, 0, 2.0, 0.0, 0.3), (1.0, 0, 1.0, nan, 0.3), (1.0, 0, 1.0, 2.0, 0.3),
              (1.0, 0, 1.0, 1.0, 0.3), (1.0, 0, 1.0, -1.0, 0.3)]
    t, k, p, m, u = (np.array(c) for c in zip(*cases))
    check(engine, F32, torch.from_numpy(np.tile(x, (len(cases), 1))).float(), engine.sample_params(t, k, p, m), u)
    tied = torch.zeros(4, 900)
    check(engine, F32, tied, engine.sample_params([1.0] * 4, [0, 7, 0, 0], [1.0, 1.0, 0.51, 1.0], [0, 0, 0, 2.0]),
          [0.9] * 4)


def test_every_kept_token_is_drawn_with_its_share(engine):
    """u over a fine grid: each token's count is its share of the grid, to one at either end."""
    vocab, n = 40, 4000
    x = torch.from_numpy(np.random.default_rng(7).standard_normal(vocab)).float()
    u = (np.arange(n) + 0.5) / n
    ids, probs = sample(engine, F32, x.repeat(n, 1), engine.sample_params(0.9, 12, 0.95, 0.0, rows=n), u)
    p = np.array([oracle(x.numpy(), np.float32(0.9), 12, np.float32(0.95), 0.0, v)[:2] for v in u])
    assert np.array_equal(ids, p[:, 0])
    count = np.bincount(ids, minlength=vocab)
    for i in range(vocab):
        if count[i]:
            assert abs(count[i] - n * probs[ids == i][0]) <= 1.001


def test_largest_vocabulary_and_many_rows(engine):
    vocab = 2097152
    x = torch.from_numpy(np.random.default_rng(8).standard_normal((2, vocab))).float()
    x[1] = 0.0
    check(engine, F32, x, engine.sample_params([1.0, 1.0], [0, 0], [0.9, 1.0], [0.0, 0.0]), [0.61, 0.999999])
    rows = 3000
    x = torch.from_numpy(np.random.default_rng(9).standard_normal((rows, 257))).bfloat16()
    check(engine, BF16, x, mixed(engine, rows), np.random.default_rng(10).random(rows))


def test_without_probabilities_and_no_rows(engine):
    x = torch.from_numpy(np.random.default_rng(11).standard_normal((3, 100))).float()
    u = [0.2, 0.5, 0.8]
    a, _ = sample(engine, F32, x, mixed(engine, 3), u)
    b, pr = sample(engine, F32, x, mixed(engine, 3), u, probs=False)
    assert np.array_equal(a, b) and np.all(pr.view(np.uint32) == 0x5B5B5B5B)
    z = engine.alloc(0)
    engine.sample_dev(engine.sample_desc(F32, 0, 100), z, 0, z, 0, z, 0, z, 0)
    engine.sync()


def test_refusals(engine):
    b = engine.alloc(4096)

    def call(ty=F32, rows=4, vocab=100, stride=0, x_off=0, p_off=0, u_off=0, i_off=0, probs=None):
        engine.sample_dev(engine.sample_desc(ty, rows, vocab, stride), b, x_off, b, p_off, b, u_off, b, i_off, probs, 0)

    for kw, status, word in [
            ({"ty": hayai_amd.Q6_K}, "HH_ERR_KERNEL_MISSING", "GGML type 14"),
            ({"vocab": 0}, "HH_ERR_INVALID", "no columns"),
            ({"vocab": 2097153}, "HH_ERR_INVALID", "vocab"),
            ({"rows": 11}, "HH_ERR_INVALID", "outside"),
            ({"stride": 99}, "HH_ERR_INVALID", "stride 99"),
            ({"stride": 2000}, "HH_ERR_INVALID", "outside"),
            ({"rows": 1 << 33}, "HH_ERR_INVALID", "31-bit"),
            ({"x_off": 2}, "HH_ERR_INVALID", "splits"),
            ({"p_off": 4096 - 60}, "HH_ERR_INVALID", "outside"),
            ({"u_off": 4084}, "HH_ERR_INVALID", "outside"),
            ({"i_off": 6}, "HH_ERR_INVALID", "splits"),
            ({"probs": engine.alloc(8)}, "HH_ERR_INVALID", "outside")]:
        with pytest.raises(hayai_amd.HipError) as err:
            call(**kw)
        assert err.value.status_name == status and word in str(err.value), (kw, err.value)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_lists_past_a_part(engine, ty):
    """Rows whose filters end among 1025 to 8192 tokens of one part: equal logits, and logits a little
    apart, alone and above a body of others."""
    rng = np.random.default_rng(12)
    for vocab, rows in ((1500, 12), (2500, 12), (4096, 12), (8000, 512), (8192, 512), (8193, 512)):
        print(f"[case] lists type={ty} {rows}x{vocab}", flush=True)
        flat = np.zeros(vocab)
        near = rng.standard_normal(vocab) * 1e-3 - 1e-2
        body = np.where(rng.random(vocab) < 0.9, -0.004 * rng.random(vocab), -3.0 - rng.random(vocab))
        params = [(1.0, vocab // 2, 1.0, 0.0), (1.0, 0, 0.83, 0.0), (1.0, vocab * 2 // 3, 0.6, 0.0), (0.5, 1100, 0.999, 0.001)]
        x = np.stack([(flat, near, body)[i % 3] for i in range(rows)])
        p = [params[i // 3 % 4] for i in range(rows)]
        check(engine, ty, torch.from_numpy(x).to(DT[ty]), engine.sample_params(*[np.array(c) for c in zip(*p)]),
              rng.random(rows))


def test_ends_of_u_in_rows_of_one_workgroup(engine):
    """Rows that one workgroup does (all tokens nearly equal under top-p, an infinite temperature, an
    infinite largest logit), with u at and past its ends."""
    vocab = 20011
    flat = -np.arange(vocab) * 1e-7
    tall = np.where(np.arange(vocab) % 9973 == 5, np.inf, flat)
    us = [0.0, -1.0, float("nan"), np.nextafter(np.float32(1), np.float32(0)), 1.0, 7.0, 1e30, 3e38, float("inf"), -float("inf")]
    cases = [(x, t, k, p, u) for x, t, k, p in [(flat, 1.0, 0, 0.9), (flat, 1.0, 9000, 1.0), (flat, float("inf"), 0, 1.0),
                                                (flat, 2e30, 9000, 0.7), (tall, 1.0, 0, 1.0), (tall, 1.0, 2, 0.5)]
             for u in us]
    x, t, k, p, u = (np.array(c) for c in zip(*cases))
    logits, params, n = torch.from_numpy(x).float(), engine.sample_params(t, k, p, 0.0), len(cases) - len(us)
    check(engine, F32, logits[:n], params[:n], u[:n])
    # the last ten: two tokens of weight 1 and half of their weight wanted.  The weight before the second is 1 and
    # the weight wanted 0.5 * 2 = 1, whole numbers on either side: not below it, so the first alone is kept.
    ids, probs = sample(engine, F32, logits[n:], params[n:], u[n:])
    assert np.all(ids == 5) and np.all(probs == 1.0)


def test_rows_four_gigabytes_apart(engine):
    vocab, far, rows = 5000, (1 << 31) + 8, 4
    x = torch.from_numpy(2.0 * np.random.default_rng(13).standard_normal((rows, vocab))).half()
    x[3] = 0.0
    b = engine.alloc(2 * ((rows - 1) * far + vocab))
    for i in range(rows):
        b.write(x[i].view(torch.uint8).numpy(), 2 * i * far)
    params, u = engine.sample_params([1.0, 0.0, 0.7, float("inf")], [0, 0, 40, 0], [0.9, 1.0, 0.9, 0.99]), [0.3, 0.5, 0.9, 0.77]
    ids, pr = engine.alloc(4 * rows), engine.alloc(4 * rows)
    engine.sample_dev(engine.sample_desc(F16, rows, vocab, far), b, 0, engine.upload(params), 0,
                      engine.upload(np.asarray(u, np.float32)), 0, ids, 0, pr, 0)
    want, probs = sample(engine, F16, x, params, u)
    assert np.array_equal(ids.read(np.int32, rows), want) and np.array_equal(pr.read(np.float32, rows), probs)
    check(engine, F16, x, params, u)
