"""fp32 attention over many keys of like weight and like values, where every addition to the running sums is
off in the same direction if it does not round to nearest (the tensor cores' additions do not).

Tolerance, relative to sum w |v| / sum w: a weight as in tests/test_kv8_weights_gpu.py (exact scores up to 3);
sums: at most one rounding a step of 64 keys for the outputs and two for the weights' sum; inside a step 32
additions of weights, inside two steps 16 tensor-core products of 16 terms with a step (2 u) each: 64 u more."""
import numpy as np
import pytest

from tests.quant8_util import decode

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_quant8_gpu import U, Cache, ctx, dev  # noqa: E402

__all__ = ["ctx"]

# heads, kv heads, rows: up to 8 pairs a tile, 16, 128, keys of a tile not split
FORMS = {"pairs8": (448, 448, 1), "pairs16": (448, 448, 9), "prompt": (32, 32, 64)}


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(FORMS))
def test_many_keys_of_like_weight(ctx, form, D, code):
    heads, G, n = FORMS[form]
    S, block = (20000 if form == "prompt" else 5000), 64
    rng = np.random.default_rng(D)
    scores = rng.normal(0, 0.3, S).astype(np.float32)
    scores[0] = 3.0                                            # (the reference from the first step on)
    values = (1 + 0.1 * rng.normal(0, 1, (S, D))).astype(np.float32)
    c = Cache(ctx, code, 1, G, D, S, block, 7)
    k = torch.zeros(S, G, D, device="cuda")
    k[:, :, 0] = dev(scores)[:, None]
    v = dev(values)[:, None].expand(S, G, D).contiguous()
    c.append(k.view(S, -1), v.view(S, -1), [S], [0], "f32")
    q = torch.zeros(n, heads, D, device="cuda")
    q[:, :, 0] = 1.0
    out = c.attend(q.view(n, -1), heads, [n], [S - n], "f32", 1.0).view(n, heads, D)
    nb = -(-S // block)
    val = {}
    for nm in "kv":                                            # (every kv head holds the same)
        codes = c.codes[nm][:S * D].cpu().numpy().reshape(S, D)
        val[nm] = decode(codes, code) * np.repeat(c.scales[nm][:nb].cpu().numpy().astype(np.float64), block)[:S, None]
    w = np.exp(val["k"][:, 0] - val["k"][:, 0].max())
    run_w, run_o = np.cumsum(w)[S - n:], np.cumsum(w[:, None] * val["v"], 0)[S - n:]
    ref = torch.from_numpy(run_o / run_w[:, None]).cuda()[:, None]
    assert (val["v"] > 0).all()
    steps = -(-S // 64)
    rel = 10 * U * 2 * 1.4427 * 3 + 2.0 ** -21 + 4 * U + 2.0 ** -22 + (3 * steps + 64) * U
    off = ((out.double() - ref).abs() / ref).max()
    assert off <= rel, (float(off), rel)
