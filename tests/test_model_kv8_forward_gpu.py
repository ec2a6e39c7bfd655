"""A whole forward over the 8-bit cache, prompts and decode steps of two sequences, against its layers
called one at a time on a second model (tests/test_model_kv8_gpu.py holds a layer call to the definition
on the cache's own codes) and the final norm and LM head in 64 bits.

Tolerance (u = 2^-24): the mean square is a sum of `hidden` terms in chains of at most 64 + 10 additions, the root and
the products add 4 roundings, the LM head's sum of `hidden` products at most `hidden` additions, each off by a step
(2 u) of the magnitudes' sum: (2 hidden + 160) u times sum |xn| |w|."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests.model_util import TINY, gpu_model, make_weights

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from asicfortranai_b200.quantized import Context
    c = Context(0)
    yield c
    c.close()


class Layers:
    """A model stepped layer by layer."""

    def __init__(self, ctx, cfg, w, fmt, block):
        self.cfg, self.w = cfg, w
        self.m = gpu_model(ctx, cfg, w)
        self.m.set_kv_cache(fmt, block=block)

    def logits(self, ids, seq):
        """64-bit logits and the sums of magnitudes"""
        x = np.asfortranarray(self.w["embed"][np.asarray(ids) - 1])
        for l in range(self.cfg["n_layers"]):
            x = self.m.apply_transformer_layer(l, x, seq=seq, advance=l + 1 == self.cfg["n_layers"])
        x = x.astype(np.float64)
        xn = x / np.sqrt((x ** 2).mean(1, keepdims=True) + self.cfg["rms_eps"]) * self.w["final_norm"].astype(np.float64)
        h = self.w["lm_head"].astype(np.float64)
        return xn @ h, np.abs(xn) @ np.abs(h)


def near(got, want, mag, hidden):
    return bool((np.abs(got.astype(np.float64) - want) <= (2 * hidden + 160) * U * mag).all())


@pytest.mark.parametrize("fmt,block,rope_mode,wformat", [("int8", 16, 1, 0), ("e4m3", 64, 0, 0), ("int8", 32, 0, 1),
                                                        ("e4m3", 16, 1, 1)])
def test_forward_equals_its_layers(ctx, fmt, block, rope_mode, wformat):
    cfg = dict(TINY, n_layers=3, max_batch=2, rope_mode=rope_mode, wformat=wformat)
    w = make_weights(cfg, seed=21)
    gm = gpu_model(ctx, cfg, w)
    gm.set_kv_cache(fmt, block=block)
    by_layer = Layers(ctx, cfg, w, fmt, block)
    prompts = [orc.gen_tokens(n, 21, 3 + n, cfg["vocab"]) for n in (37, 12)]
    for part in (slice(0, 9), slice(9, None)):                  # each prompt in two calls, the sequences in turn
        for seq in (1, 0):
            ids = prompts[seq][part]
            got = gm.forward_llama(ids, seq=seq)
            want, mag = by_layer.logits(ids, seq)
            assert near(got, want, mag, cfg["hidden"])
    for step in range(20):                                      # decode: all sequences in one step
        ids = orc.gen_tokens(2, 21, 50 + step, cfg["vocab"])
        _, got = gm.decode_step(ids, want_logits=True)
        for seq in range(2):
            want, mag = by_layer.logits(ids[seq:seq + 1], seq)
            assert near(got[seq:seq + 1], want, mag, cfg["hidden"]), (step, seq)
    gm.cleanup_llama_model()
    by_layer.m.cleanup_llama_model()


def test_the_bound_sees_a_wrong_history(ctx):
    """The last token's logits behind two prompts that differ in their other tokens are apart."""
    cfg = dict(TINY, n_layers=3, max_batch=1, rope_mode=1)
    w = make_weights(cfg, seed=21)
    by_layer = Layers(ctx, cfg, w, "int8", 16)
    last = orc.gen_tokens(1, 21, 99, cfg["vocab"])
    out = []
    for tid in (5, 6):
        by_layer.m.reset_kv_cache()
        by_layer.logits(orc.gen_tokens(30, 21, tid, cfg["vocab"]), 0)
        out.append(by_layer.logits(last, 0))
    assert not near(out[0][0], *out[1], 100 * cfg["hidden"])
    by_layer.m.cleanup_llama_model()
