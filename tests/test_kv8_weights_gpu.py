"""Attention over the 8-bit cache where small weights carry the result: a key far above the others whose
value is zero (as the first token of a sequence behaves in many models), and a block of large values
that next to no weight falls on.  Both leave the other keys weights many powers of two below the
largest one, in front of the largest v scale.

Tolerance, relative to A = sum w |v| / sum w (u = 2^-24, s the largest score in powers of two).  Only one
element of a query is not zero, so a score is an exact product times a scale.
 * a weight: the score's three roundings, the maximum's, the difference's and log2(e)'s rounded value are
   below 10 u s; the exponential 2^-21; the product with the scales' ratio 4 u;
 * its rounding to fp16: 2^-11 for 16-bit queries, 2^-22 for the two terms of fp32 queries;
 * sums in binary32: 64 steps of 2 u, and 8 u for the merge and the division.
What lies below fp16's normal numbers is off by half their spacing, 2^-25, before the factor that the weights
carry: 2^15 for up to 8 and 16 pairs (with a second term: 2^26), 2^11 for prompts (fp32 queries: 2^14).
That is floor_of() times the largest |v| for every key.  Outputs are rounded once to their type (fp16 below
2^-14: 2^-25)."""
import numpy as np
import pytest

from tests.quant8_util import decode

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_quant8_gpu import U, Cache, ctx, dev, half_step  # noqa: E402

__all__ = ["ctx"]

# heads, kv heads, rows: up to 8 pairs a tile, 16 pairs a tile, 128 (32 tiles of half a tile at least); with
# 448 tiles the keys are not split, so that every warp walks several steps of them
FORMS = {"pairs8": (8, 1, 1), "pairs8_heads": (4, 4, 2), "pairs16": (8, 1, 3), "prompt": (32, 32, 64),
         "pairs8_whole": (448, 448, 1), "pairs16_whole": (448, 448, 9)}
S, BLOCK = 700, 64


def floor_of(form, dtype):
    if form == "prompt":
        return 2.0 ** -39 if dtype == "f32" else 2.0 ** -36
    return 2.0 ** -51 if dtype == "f32" else 2.0 ** -40


def check(ctx, form, dtype, code, D, scores, values):
    """scores [S], values [S][D]: keys are (score, 0, 0, ..), queries about (1, 0, 0, ..)."""
    heads, G, n = FORMS[form]
    c = Cache(ctx, code, 1, G, D, S, BLOCK, 7)
    k = np.zeros((S, G, D), np.float32)
    k[:, :, 0] = scores[:, None]
    v = np.repeat(values[:, None], G, 1)
    c.append(dev(k.reshape(S, -1), dtype), dev(v.reshape(S, -1), dtype), [S], [0], dtype)
    q = np.zeros((n, heads, D), np.float32)
    q[:, :, 0] = 1.0 - 0.125 * (np.arange(n * heads) % 3).reshape(n, heads)
    out = c.attend(dev(q.reshape(n, -1), dtype), heads, [n], [S - n], dtype, 1.0)
    got = out.double().cpu().numpy().reshape(n, heads, D)
    val = {}                                            # (every kv head holds the same)
    for nm in "kv":
        codes, sc = c.host(nm)
        val[nm] = decode(codes[0, 0], code) * np.repeat(sc[0, 0].astype(np.float64), BLOCK)[:S, None]
    score = q[:, :, 0, None].astype(np.float64) * val["k"][:, 0]               # [n][heads][S]
    seen = np.arange(S)[None] <= S - n + np.arange(n)[:, None]
    w = np.where(seen[:, None], np.exp(score - score.max(-1, keepdims=True)), 0.0)
    w /= w.sum(-1, keepdims=True)
    ref, mag = w @ val["v"], w @ np.abs(val["v"])
    s2 = 1.4427 * scores.max() * 2
    rel = 10 * U * s2 + 2.0 ** -21 + 4 * U + (2.0 ** -22 if dtype == "f32" else 2.0 ** -11) + (128 + 8) * U
    tol = np.abs(ref) * half_step(dtype) + rel * mag + S * floor_of(form, dtype) * np.abs(val["v"]).max()
    if dtype == "f16":
        tol = tol + 2.0 ** -25
    off = np.abs(got - ref)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
def test_a_key_far_above_the_others_without_a_value(ctx, form, D, code, dtype):
    rng = np.random.default_rng(D)
    for gap in (8.0, 12.0, 16.0, 20.0):
        scores = rng.normal(0, 0.3, S).astype(np.float32)
        scores[0] = gap
        values = (1000 * (1 + 0.3 * rng.normal(0, 1, (S, D)))).astype(np.float32)
        values[0] = 0.0
        check(ctx, form, dtype, code, D, scores, values)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
def test_a_block_of_large_values_with_no_weight(ctx, form, D, code, dtype):
    rng = np.random.default_rng(D + 1)
    scores = rng.normal(0, 0.3, S).astype(np.float32)
    values = (1 + 0.3 * rng.normal(0, 1, (S, D))).astype(np.float32)
    scores[0], values[0] = 9.0, 0.0
    big = slice(2 * BLOCK, 3 * BLOCK)
    scores[big] = -60.0
    values[big] = 32768.0 * rng.choice([-1.0, 1.0], (BLOCK, D))
    check(ctx, form, dtype, code, D, scores, values)
