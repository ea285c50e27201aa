"""Attention over a cache of pages in 64 bits, and how far a kernel's outputs may be from it.

For a row with weights w_j (of sum 1) and A_d = sum_j w_j |v_jd|, in units u = 2^-24 (an f32 rounding):
  scores: products of f32 operands (16-bit ones are exact in f32) summed over dim elements in f32, the
    scale and the base: |error| <= (dim + 8) u S, S = max_j scale sum_i |q_i k_ji|, plus that of the base, which
    is as large as the largest score; f32 queries over a 16-bit cache round first: c S more, c = eps / 2 of
    the cache's type
  so a weight is off by a factor of 1 +- delta, delta = 2 (score error) + 8 u (exp2), and by c more where it is
    rounded for the second product; the sum of weights by delta + n u
  output: |error_d| <= A_d (2 delta + c + (2 n + 32) u) + eps / 2 |o_d| of its own type
(n keys; 2 n: sums of weights and of products; joins of parts are among the 32).
"""
import numpy as np
import torch

import hayai_amd

DT = {hayai_amd.F32: torch.float32, hayai_amd.F16: torch.float16, hayai_amd.BF16: torch.bfloat16}


def half_step(ty):
    return {hayai_amd.F32: 2.0**-24, hayai_amd.F16: 2.0**-11, hayai_amd.BF16: 2.0**-8}[ty]


def page_elements(kvh, dim, page):
    return 2 * kvh * dim * page


def gather(cache, table, length, kvh, dim, page):
    """(keys, values) of a sequence's first `length` tokens, (length, kvh, dim) in 64 bits; pages outside are zeros."""
    n, per = cache.shape[0], page_elements(kvh, dim, page)
    keys, values = np.zeros((length, kvh, dim)), np.zeros((length, kvh, dim))
    for first in range(0, length, page):
        p, m = int(table[first // page]), min(page, length - first)
        if 0 <= p < n:
            row = cache[p, :per].double().numpy()
            keys[first:first + m] = row[:per // 2].reshape(kvh, page, dim)[:, :m].transpose(1, 0, 2)
            values[first:first + m] = row[per // 2:].reshape(kvh, dim, page)[:, :, :m].transpose(2, 0, 1)
    return keys, values


def attend(q, keys, values, seen, scale, ty, cty):
    """q (rows, heads, dim), seen[row] tokens of keys and values: outputs and their bounds."""
    rows, heads, dim = q.shape
    group = heads // keys.shape[1]
    out, bound = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    u, c = 2.0**-24, 0.0 if cty == hayai_amd.F32 else half_step(cty)
    for t in range(rows):
        n = min(int(seen[t]), len(keys))
        if n <= 0:
            continue
        for h in range(heads):
            k, v = keys[:n, h // group], values[:n, h // group]
            s = scale * (k @ q[t, h])
            size = float(np.max(scale * (np.abs(k) @ np.abs(q[t, h]))))
            w = np.exp(s - s.max())
            w /= w.sum()
            out[t, h] = w @ v
            delta = 2 * ((dim + 8) * u + (c if ty != cty else 0.0)) * size + 8 * u
            bound[t, h] = (w @ np.abs(v)) * (2 * delta + c + (2 * n + 32) * u) + half_step(ty) * np.abs(out[t, h])
    return out, bound


def check(got, want, bound, ty):
    got = got.double().numpy()
    tiny = float(torch.finfo(DT[ty]).smallest_normal) * float(torch.finfo(DT[ty]).eps)
    assert np.all(np.isfinite(got)), "outputs that are no finite numbers"
    err = np.abs(got - want)
    worst = np.max(err / (bound + tiny), initial=0.0)
    assert worst <= 1.0 + 1e-3, f"off by {worst:.2f} times the bound"
