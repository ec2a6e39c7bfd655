"""The 8-bit operators run together, as a serving step uses them, each stage against the 64-bit
reference of its own inputs; the same step captured, replayed and on two contexts at once; and
prompts, ragged and unaligned, through the attention's 128-row form.  Tolerances are those of
tests/test_quant8_gpu.py."""
import numpy as np
import pytest

from tests.quant8_util import sample_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_quant8_gpu import (  # noqa: E402
    DT, F, Cache, attention_ref, check_attention, check_norm, check_product, ctx, dev, product_ref)

__all__ = ["ctx"]


class Step:
    """norm -> q|k|v product -> append, attention -> codes -> o product -> norm with the residual ->
    head product -> sampling, of `rows` rows of a small layer."""

    HID, H, G, D, S, BLK, V = 640, 5, 1, 128, 400, 64, 5003

    def __init__(self, ctx, counts, past, seed):
        from asicfortranai_b200.quant8 import KV8Cache
        self.ctx, self.counts, self.past = ctx, counts, past
        self.rows = rows = sum(counts)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        B, HID, H, G, D = len(counts), self.HID, self.H, self.G, self.D
        self.N = (H + 2 * G) * D

        def weight(n, k):
            w = (rand(n, k) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            return w, torch.rand(-(-n // 128), -(-k // 128), generator=g, device="cuda") * 2e-4 + 2e-4
        self.wqkv, self.wo, self.wh = weight(self.N, HID), weight(HID, H * D), weight(self.V, HID)
        self.n1, self.n2, self.one = 1 + 0.1 * rand(HID), 1 + 0.1 * rand(HID), torch.ones(H * D, device="cuda")
        self.x = rand(rows, HID).bfloat16()
        self.cache = Cache(ctx, "e4m3", B, G, D, self.S, self.BLK, seed)
        if sum(past):
            hist = {n: rand(sum(past), G * D).bfloat16() for n in "kv"}
            self.cache.append(hist["k"], hist["v"], past, [0] * B, "bf16")
        self.state = {n: (self.cache.codes[n].clone(), self.cache.scales[n].clone()) for n in "kv"}
        self.rs = dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        self.pt = dev(np.array(past, np.int32))
        e8 = lambda n, k: (torch.zeros(n, k, dtype=torch.uint8, device="cuda"),  # noqa: E731
                           torch.zeros(n, -(-k // 128), device="cuda"))
        self.c1, self.c2, self.c3 = e8(rows, HID), e8(rows, H * D), e8(rows, HID)
        b16 = lambda n: torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.qkv, self.att, self.o, self.h = b16(self.N), b16(H * D), b16(HID), b16(HID)
        self.logits = torch.zeros(rows, self.V, device="cuda")
        self.u = torch.rand(rows, generator=g, device="cuda")
        self.T = torch.full((rows,), 0.8, device="cuda")
        self.p = torch.full((rows,), 0.9, device="cuda")
        self.tok = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.prob = torch.zeros(rows, device="cuda")
        self.kv = KV8Cache(ctx, self.cache.codes["k"].data_ptr(), self.cache.codes["v"].data_ptr(),
                           self.cache.scales["k"].data_ptr(), self.cache.scales["v"].data_ptr(), B, G, D, self.S, self.BLK)
        n = self.kv.attention_workspace(H, rows, max(counts))
        self.ws = torch.full((n + 16,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def run(self):
        from asicfortranai_b200 import quant8, sampling
        a = lambda t: t.data_ptr()  # noqa: E731
        c, rows, HID, H, G, D = self.ctx, self.rows, self.HID, self.H, self.G, self.D
        quant8.rms_norm_quant(c, a(self.x), a(self.n1), a(self.c1[0]), a(self.c1[1]), rows, HID)
        quant8.fp8_gemm(c, a(self.c1[0]), a(self.c1[1]), a(self.wqkv[0]), a(self.wqkv[1]), a(self.qkv), rows, self.N, HID)
        kp = a(self.qkv) + 2 * H * D
        mr = max(self.counts)
        self.kv.append(kp, kp + 2 * G * D, a(self.rs), a(self.pt), rows, mr, ld=self.N)
        self.kv.attention(a(self.qkv), a(self.att), H, a(self.rs), a(self.pt), rows, mr, D ** -0.5, ldq=self.N,
                          workspace=a(self.ws), workspace_bytes=self.ws.numel())
        quant8.rms_norm_quant(c, a(self.att), a(self.one), a(self.c2[0]), a(self.c2[1]), rows, H * D)
        quant8.fp8_gemm(c, a(self.c2[0]), a(self.c2[1]), a(self.wo[0]), a(self.wo[1]), a(self.o), rows, HID, H * D)
        quant8.rms_norm_quant(c, a(self.o), a(self.n2), a(self.c3[0]), a(self.c3[1]), rows, HID, residual=a(self.x),
                              residual_out=a(self.h))
        quant8.fp8_gemm(c, a(self.c3[0]), a(self.c3[1]), a(self.wh[0]), a(self.wh[1]), a(self.logits), rows, self.V, HID,
                        dtype="f32")
        sampling.sample_filtered_rows(c, a(self.logits), rows, self.V, a(self.u), a(self.tok), temperature=a(self.T),
                                      top_p=a(self.p), probs=a(self.prob))

    def restore(self):
        """The cache as before the step, and nothing of its outputs."""
        for n in "kv":
            self.cache.codes[n].copy_(self.state[n][0])
            self.cache.scales[n].copy_(self.state[n][1])
        for t in (*self.c1, *self.c2, *self.c3, self.qkv, self.att, self.o, self.h, self.logits, self.tok, self.prob):
            t.zero_()
        torch.cuda.synchronize()

    def results(self):
        self.ctx.synchronize()
        return [t.clone() for t in (*self.c1, self.qkv, self.att, *self.c2, self.o, self.h, *self.c3, self.logits, self.tok,
                                    self.prob, *self.cache.codes.values())]


STEPS = [([1, 1, 1], [0, 130, 399]), ([1], [200]), ([70, 0, 3], [33, 5, 64]), ([200, 129], [0, 77])]


@pytest.mark.parametrize("counts,past", STEPS, ids=[str(i) for i in range(len(STEPS))])
def test_step_stage_by_stage(ctx, counts, past):
    s = Step(ctx, counts, past, 3)
    s.run()
    ctx.device_error()
    check_norm(s.x, None, s.n1, s.x, s.c1[0].cpu().numpy(), s.c1[1], "bf16", "e4m3", 128)
    check_product(s.qkv, *product_ref(*s.c1, *s.wqkv, s.N, s.HID), s.HID, "bf16")
    ref, mag, vmax = attention_ref(s.cache, s.qkv[:, :s.H * s.D].float().cpu().numpy(), s.H, counts, past, s.D ** -0.5)
    check_attention(s.att.double().cpu().numpy().reshape(ref.shape), ref, mag, vmax, s.D, "bf16")
    check_norm(s.att, None, s.one, s.att, s.c2[0].cpu().numpy(), s.c2[1], "bf16", "e4m3", 128)
    check_product(s.o, *product_ref(*s.c2, *s.wo, s.HID, s.H * s.D), s.H * s.D, "bf16")
    # (the norm's input is the binary32 sum; the stored one is rounded)
    check_norm(s.o, s.x, s.n2, s.h, s.c3[0].cpu().numpy(), s.c3[1], "bf16", "e4m3", 128)
    check_product(s.logits, *product_ref(*s.c3, *s.wh, s.V, s.HID), s.HID, "f32")
    lg, u = s.logits.double().cpu().numpy(), s.u.cpu().numpy()
    for r in range(s.rows):
        tok, prob = sample_ref(lg[r], float(F(0.8)), 0, float(F(0.9)), 0.0, float(u[r]))
        assert int(s.tok[r]) == tok
        assert abs(float(s.prob[r]) - prob) <= prob * 2.0 ** -23 + 2.0 ** -30


@pytest.mark.parametrize("counts,past", STEPS[1:], ids=[str(i) for i in range(1, len(STEPS))])
def test_step_captured_and_replayed(ctx, counts, past):
    s = Step(ctx, counts, past, 4)
    s.run()
    want = s.results()
    s.restore()
    graph = ctx.capture(s.run)
    for _ in range(2):
        s.restore()
        graph.launch()
        for a, b in zip(want, s.results()):
            assert torch.equal(a, b)
    # other inputs under the same pointers, the history's length among them
    x2 = torch.randn_like(s.x) * 2
    past2 = [max(p - 20, 0) for p in past]
    outs = []
    for go in (s.run, graph.launch):
        s.restore()
        s.x.copy_(x2)
        s.pt.copy_(dev(np.array(past2, np.int32)))
        torch.cuda.synchronize()
        go()
        outs.append(s.results())
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert not torch.equal(outs[0][2], want[2])
    ctx.device_error()
    graph.close()


def test_two_contexts_at_once():
    """Two steps on two streams, their calls in turn, give what each gives alone."""
    from asicfortranai_b200.quantized import Context
    cs = [Context(0), Context(0)]
    steps = [Step(cs[0], [1, 1], [333, 40], 5), Step(cs[1], [150], [100], 6)]
    want = []
    for s in steps:
        s.run()
        want.append(s.results())
        s.restore()
    for _ in range(5):
        for s in steps:
            s.restore()
        for s in steps:
            s.run()
        for s, w in zip(steps, want):
            for a, b in zip(w, s.results()):
                assert torch.equal(a, b)
    for c in cs:
        c.device_error()
        c.close()


PROMPTS = [  # heads, kv heads, D, block, max_seq, counts, past, scale, columns behind a row
    (2, 2, 128, 64, 700, [64, 300, 0], [0, 333, 9], 0.09, 0),
    (8, 1, 128, 16, 300, [33, 1, 129], [7, 299, 171], -0.09, 1),          # negative: the smallest product wins
    (12, 4, 64, 128, 1000, [500, 0, 64], [500, 0, 65], 0.125, 8),
    (5, 1, 64, 32, 400, [400], [0], 0.3, 3),
    (1, 1, 128, 64, 1300, [129], [1171], 0.0, 0),                         # 0: the mean of what a row sees
    (3, 1, 64, 16, 65, [64, 65, 1], [1, 0, 64], 0.125, 0),
    (16, 2, 128, 128, 2500, [9], [2491], 0.0884, 16),
    # below: tiles of 128 rows for many SMs
    (24, 24, 128, 64, 700, [64, 300, 0], [0, 333, 9], 0.09, 0),
    (64, 16, 64, 16, 300, [33, 1, 129], [7, 299, 171], -0.09, 1),
    (16, 16, 128, 64, 1300, [129], [1171], 0.0, 0),
    (48, 16, 128, 16, 65, [64, 65, 1], [1, 0, 64], 0.125, 0),
    (3, 3, 256, 64, 500, [190, 0, 70], [310, 40, 5], 0.0625, 0),
    (8, 2, 256, 16, 300, [17, 33], [200, 0], -0.0625, 5),
    (16, 16, 128, 64, 900, [140, 129, 131, 150], [700, 0, 3, 64], 0.0884, 0),
    (40, 20, 64, 64, 1100, [300], [777], 0.125, 4),
    (6, 6, 256, 128, 1000, [140, 257, 300, 128, 65, 129, 150, 200], [800, 0, 3, 64, 9, 129, 640, 1], 0.0625, 4),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
def test_attention_of_prompts(ctx, dtype, code, case):
    heads, G, D, block, S, counts, past, scale, pad = case
    rng = np.random.default_rng(31 * heads + D + S)
    B, rows = len(counts), sum(counts)
    c = Cache(ctx, code, B, G, D, S, block, 7)
    if sum(past):
        hist = {n: dev(rng.normal(0, 1, (sum(past), G * D)), dtype) for n in "kv"}
        hist["k"] *= dev(np.exp(rng.normal(0, 1, (sum(past), 1))), dtype)
        hist["v"] *= dev(np.exp(rng.normal(0, 2, (sum(past), 1))), dtype)
        hist["v"][: sum(past) // 3] = 0.0                    # blocks whose v scale is 0
        c.append(hist["k"], hist["v"], past, [0] * B, dtype)
    new = {n: dev(rng.normal(0, 1, (rows, G * D)), dtype) for n in "kv"}
    c.append(new["k"], new["v"], counts, past, dtype)
    # two rows more than the tables name: they stay as they are
    q = torch.full((rows + 2, heads * D + pad), float("nan"), dtype=DT[dtype], device="cuda")
    size = np.exp(rng.normal(0, 1.5, (rows, 1)))             # from nearly flat weights to a single key
    q[:rows, :heads * D] = dev(rng.normal(0, 1, (rows, heads * D)) * size, dtype)
    q[0, :D] = 0.0
    out = c.attend(q, heads, counts, past, dtype, scale)
    assert (out[:, heads * D:] == 3).all() and (out[rows:] == 3).all()
    got = out[:rows, :heads * D].double().cpu().numpy().reshape(rows, heads, D)
    ref, mag, vmax = attention_ref(c, q[:rows, :heads * D].float().cpu().numpy(), heads, counts, past, scale)
    check_attention(got, ref, mag, vmax, D, dtype)
    assert torch.equal(out, c.attend(q, heads, counts, past, dtype, scale))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,G,D,past,rows", [(1, 1, 128, 13, 6), (1, 1, 128, 5, 40), (2, 1, 64, 5, 123), (1, 1, 256, 7, 20),
                                                 (40, 40, 128, 5, 123), (64, 32, 64, 5, 100), (32, 32, 256, 7, 80)])
def test_later_values_take_no_bits_from_earlier_rows(ctx, dtype, heads, G, D, past, rows):
    """Values that grow by 2^7 from block to block: a row is as exact as what it sees is large."""
    rng = np.random.default_rng(heads * D + rows)
    S = past + rows
    c = Cache(ctx, "int8", 1, G, D, S, 16, 3)
    grow = 2.0 ** (-100 + 7 * (np.arange(S) // 16))[:, None] if dtype != "f16" else 2.0 ** (-14 + 3 * (np.arange(S) // 16))[:, None]
    k, v = dev(rng.normal(0, 1, (S, G * D)), dtype), dev(rng.normal(0, 1, (S, G * D)) * grow, dtype)
    c.append(k, v, [S], [0], dtype)
    q = dev(rng.normal(0, 1, (rows, heads * D)), dtype)
    out = c.attend(q, heads, [rows], [past], dtype, D ** -0.5)
    ref, mag, vmax = attention_ref(c, q.float().cpu().numpy(), heads, [rows], [past], D ** -0.5)
    if dtype == "f16":                                       # its numbers end at 2^-25: values above that
        keep = np.abs(ref) > 2.0 ** -12
        ref, got = np.where(keep, ref, 0), np.where(keep, out.double().cpu().numpy().reshape(ref.shape), 0)
    else:
        got = out.double().cpu().numpy().reshape(ref.shape)
    check_attention(got, ref, mag, vmax, D, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G", [1, 20])
def test_values_of_the_smallest_numbers(ctx, G, dtype):
    """Block scales that are subnormal: no division by one makes an infinity."""
    D, S = 128, 200
    rng = np.random.default_rng(3)
    for rows in (1, 20, S):
        c = Cache(ctx, "e4m3", 1, G, D, S, 16, 4)
        size = np.choose(np.arange(S) // 16 % 3, [0.0, 1e-38, 3e-37])[:, None]
        k, v = dev(rng.normal(0, 1, (S, G * D)), dtype), dev(rng.normal(0, 1, (S, G * D)) * size, dtype)
        c.append(k, v, [S], [0], dtype)
        q = dev(rng.normal(0, 1, (rows, G * D)), dtype)
        out = c.attend(q, G, [rows], [S - rows], dtype, 0.09)
        assert torch.isfinite(out).all() and float(out.abs().max()) <= 1.5e-36


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G", [1, 16])
def test_prompt_rows_that_are_not_numbers_stay_alone(ctx, G, dtype):
    heads, D, S = 2 * G, 128, 200
    rng = np.random.default_rng(17)
    c = Cache(ctx, "int8", 1, G, D, S, 64, 8)
    kv = {n: dev(rng.normal(0, 1, (S, G * D)), dtype) for n in "kv"}
    c.append(kv["k"], kv["v"], [S], [0], dtype)
    q = dev(rng.normal(0, 1, (S, heads * D)), dtype)
    clean = c.attend(q, heads, [S], [0], dtype, 0.09)
    q[50, 3] = float("nan")
    out = c.attend(q, heads, [S], [0], dtype, 0.09)
    assert torch.isnan(out[50, :D]).all()
    out[50, :D] = clean[50, :D]
    assert torch.equal(out, clean)


def test_append_quotients_at_and_near_rounding_boundaries(ctx):
    """Values whose quotient by the scale falls on or beside the middle between two codes."""
    from tests.quant8_util import E4M3, QMAX, append_ref
    D, block = 64, 64
    for code in ("int8", "e4m3"):
        top = float(QMAX[code])
        codes = np.arange(0, 127) if code == "int8" else E4M3[:126]
        after = np.arange(1, 128) if code == "int8" else E4M3[1:127]
        mid = (codes + after) / 2
        for amax in (top, 1.0, 3.7, 1e-20, 1e-37, 2.0 ** 100):
            s = F(F(amax) / QMAX[code])
            x = (mid * float(s)).astype(F)
            x = np.concatenate([np.nextafter(x, F(0)), x, np.nextafter(x, F(np.inf)), [F(amax)]])
            x = np.resize(np.concatenate([x, -x]), (block, D)).astype(F)
            c = Cache(ctx, code, 1, 1, D, block, block, 1)
            before = c.host("k")
            t = dev(x)
            c.append(t, t, [block], [0], "f32")
            want = append_ref(before[0][0, 0], before[1][0, 0], x, 0, block, code)
            got = c.host("k")
            np.testing.assert_array_equal(got[1][0, 0], want[1])
            np.testing.assert_array_equal(got[0][0, 0], want[0], err_msg=f"{code} {amax}")


@pytest.mark.parametrize("V", [100277, 401408])
def test_sampler_long_rows_of_equal_and_of_few_values(ctx, V):
    """More equal logits at the cut than any list of the selected ones holds."""
    from tests.test_quant8_gpu import ONE_MINUS, check_sampler
    rng = np.random.default_rng(V)
    lg = np.zeros((6, V))
    lg[1] = rng.integers(0, 2, V)
    lg[2] = rng.integers(0, 5, V) * 0.25
    lg[3, ::2] = np.inf
    lg[4] = rng.integers(0, 2, V) * 1e-3
    lg[5] = 30.0 * (np.arange(V) == V - 1)
    u = np.array([0.5, ONE_MINUS, 0.25, 0.75, 0.5, 0.0], F)
    check_sampler(ctx, lg, "f32", None, None, np.full(6, 0.75), None, u)
    check_sampler(ctx, lg, "f32", None, np.array([V // 2, 40, V // 3, 7, 50000, 3]), None, None, u)
    check_sampler(ctx, lg, "f32", np.full(6, 2.0), np.full(6, V // 2), np.full(6, 0.5), np.full(6, 1e-3), u)
