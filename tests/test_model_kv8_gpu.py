"""The model with its KV cache in 8 bits: what a layer call leaves in the cache equals the
append's definition on the layer's own keys and values, its output is the o projection of the
attention's definition over those codes, decoding (a captured graph) follows the same rules as
stepping, and going back to fp32 gives the oracle's tokens again."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests.model_util import TINY, gpu_model, make_weights
from tests.quant8_util import append_ref, decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from asicfortranai_b200.quantized import Context
    c = Context(0)
    yield c
    c.close()


def layer_model(ctx, cfg, seed):
    """One INT4 model whose down projection is zero, so that a layer's output is x + o(attention)."""
    w = make_weights(cfg, seed=seed)
    for l in range(cfg["n_layers"]):
        w[f"{l}.wd"] = np.zeros_like(w[f"{l}.wd"])
        w[f"{l}.sd"] = np.zeros_like(w[f"{l}.sd"])
    return gpu_model(ctx, cfg, w), w


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D,H,KVH,block", [(128, 4, 2, 64), (256, 2, 1, 16), (128, 8, 1, 32)])
def test_layer_over_an_8_bit_cache(ctx, code, D, H, KVH, block):
    check_layer(ctx, code, D, H, KVH, block, 100,
                [(1, 1, 9, 1.0), (0, 1, 3, 2.0), (1, 1, 1, 1.0), (1, 1, 1, 30.0), (1, 1, 40, 0.5), (0, 1, 1, 1.0)])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D,H,KVH,block", [(128, 16, 16, 64), (128, 32, 8, 32), (256, 12, 12, 16)])
def test_layer_of_a_prompt_over_an_8_bit_cache(ctx, code, D, H, KVH, block):
    """Rows for many 128-row tiles, first and behind others."""
    check_layer(ctx, code, D, H, KVH, block, 410, [(0, 1, 260, 1.0), (0, 1, 131, 2.0), (1, 1, 300, 0.5), (0, 1, 1, 1.0)])


def check_layer(ctx, code, D, H, KVH, block, max_seq, calls):
    """calls: (sequence, layer, rows, size of the input)"""
    cfg = dict(TINY, n_layers=2, n_heads=H, n_kv_heads=KVH, head_dim=D, hidden=512, wformat=1, max_batch=2, max_seq=max_seq)
    gm, w = layer_model(ctx, cfg, 31)
    gm.set_kv_cache(code, block=block)
    S, nblk, hid = cfg["max_seq"], -(-cfg["max_seq"] // block), cfg["hidden"]
    rng = np.random.default_rng(4)
    codes = {n: np.zeros((2, 2, KVH, S, D), np.uint8) for n in "kv"}
    scales = {n: np.zeros((2, 2, KVH, nblk), np.float32) for n in "kv"}
    past = [0, 0]
    wo = orc.matmul_int4_awq                                         # int32 accumulators of an int8 matrix
    for seq, layer, n, size in calls:
        x = (rng.normal(0, size, (n, hid)) * np.exp(rng.normal(0, 1, (n, 1)))).astype(np.float32)
        out = gm.apply_transformer_layer(layer, x, seq=seq)
        QN, KN = H * D, KVH * D
        y = gm.debug_buffer("yqkv", (n, QN + 2 * KN))
        q = gm.debug_buffer("q", (n, H, D))
        new = {"k": y[:, QN:QN + KN].reshape(n, KVH, D), "v": y[:, QN + KN:].reshape(n, KVH, D)}
        got = {nm: gm.debug_buffer(nm + "8", codes[nm].shape, np.uint8) for nm in "kv"}
        gots = {nm: gm.debug_buffer(nm + "8_scale", scales[nm].shape) for nm in "kv"}
        val = {}
        for nm in "kv":
            for g in range(KVH):
                codes[nm][seq, layer, g], scales[nm][seq, layer, g] = append_ref(
                    codes[nm][seq, layer, g], scales[nm][seq, layer, g], new[nm][:, g], past[seq], block, code)
            np.testing.assert_array_equal(got[nm], codes[nm])
            np.testing.assert_array_equal(gots[nm], scales[nm])
            val[nm] = decode(codes[nm][seq, layer], code) * np.repeat(scales[nm][seq, layer].astype(np.float64), block, 1)[:, :S, None]
        att = np.zeros((n, H, D))
        seen = np.arange(past[seq] + n)[None] <= past[seq] + np.arange(n)[:, None]
        for h in range(H):
            g = h * KVH // H
            s = np.where(seen, q[:, h].astype(np.float64) @ val["k"][g, :past[seq] + n].T / np.sqrt(D), -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            att[:, h] = p @ val["v"][g, :past[seq] + n] / p.sum(1, keepdims=True)
        a = np.clip(att.reshape(n, QN) * 127.0, -127, 127)
        ai = np.trunc(a).astype(np.int8)
        # an attention output within 2^-14 of a step of 127 a may fall on either side of it
        near = np.abs(a - np.rint(a)) < np.maximum(2.0 ** -14 * np.abs(a), 2.0 ** -14)
        mag = np.abs(w[f"{layer}.so"])[None] * (near.sum(1)[:, None] * 8 + 0)
        acc = wo(ai, w[f"{layer}.wo"], w[f"{layer}.so"])
        want = x.astype(np.float64) + acc * w[f"{layer}.so"][None].astype(np.float64)
        tol = mag + np.abs(want) * 2.0 ** -22 + np.abs(acc * w[f"{layer}.so"][None]) * 2.0 ** -22
        assert (np.abs(out - want) <= tol).all(), float((np.abs(out - want) - tol).max())
        past[seq] += n
    gm.cleanup_llama_model()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_generation_over_an_8_bit_cache(ctx, fmt):
    """The captured decode step gives what stepping with given tokens gives, for two sequences,
    twice, also after the format was changed in between."""
    cfg = dict(TINY, max_batch=2)
    w = make_weights(cfg, seed=12)
    gm = gpu_model(ctx, cfg, w)
    prompts = np.stack([orc.gen_tokens(9, 6, 40 + b, cfg["vocab"]) for b in range(2)])
    plain = gm.generate(prompts, 20)
    gm.set_kv_cache(fmt)
    a = gm.generate(prompts, 20)
    gm.set_kv_cache("fp32")
    for x, y in zip(gm.generate(prompts, 20), plain):
        np.testing.assert_array_equal(x, y)
    gm.set_kv_cache(fmt)
    for x, y in zip(gm.generate(prompts, 20), a):
        np.testing.assert_array_equal(x, y)
    gm.reset_kv_cache()
    first = [gm.forward_next_token(prompts[b], seq=b) for b in range(2)]
    toks = [first]
    for _ in range(19):
        toks.append(list(gm.decode_step(np.array(toks[-1], np.int32))))
    for b in range(2):
        np.testing.assert_array_equal([t[b] for t in toks], a[b])
    # a prompt's logits stay near the fp32 cache's: 8-bit keys and values are off by 2^-8 (int8, of
    # the block's largest) or 2^-4 (e4m3) each, and every activation is truncated to 1/127 behind them
    gm.set_kv_cache("fp32")
    ref = gm.forward_llama(prompts[0])
    gm.set_kv_cache(fmt)
    got = gm.forward_llama(prompts[0])
    assert np.isfinite(got).all()
    gm.cleanup_llama_model()
    assert got.shape == ref.shape


def test_refusals(ctx):
    from asicfortranai_b200 import Q35Error
    cfg = dict(TINY)
    gm = gpu_model(ctx, cfg, make_weights(cfg, seed=1))
    for fmt, block in ((3, 64), (-1, 64), ("int8", 48), ("e4m3", 0)):
        with pytest.raises(Q35Error):
            gm.set_kv_cache(fmt, block=block)
    gm.debug_buffer("kc", (4,))
    with pytest.raises(Q35Error):
        gm.debug_buffer("k8", (4,), np.uint8)
    gm.set_kv_cache("int8")
    with pytest.raises(Q35Error):
        gm.debug_buffer("kc", (4,))
    # the cache still has its max_seq positions
    gm.forward_next_token(np.ones(cfg["max_seq"], np.int32))
    with pytest.raises(Q35Error):
        gm.decode_step()
    gm.cleanup_llama_model()
