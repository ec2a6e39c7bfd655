"""The 8-bit operators on the GPU against 64-bit references written from their definitions
(tests/quant8_util.py).

Tolerances.  u = 2^-24 is half a step of binary32.
 * norm: the mean square is a sum of n terms in chains of at most 32 + 10 additions, the root,
   the quotient and the two products add 4 roundings: y is within 64 u of the exact value, a
   scale within 66 u, and a code's value within half a code step of y beyond that.
 * product: a block's 128 exact products are summed in binary32 by the tensor cores (at most 128
   additions, each off by a step, 2u), the scale product and the fused multiply-add are 2 more
   roundings, and ceil(K/128) partial sums add up: (130 + KB) 2u times the sum of the magnitudes,
   plus half a step of y's type.
 * attention: scores are binary32 tensor-core sums (D/16 steps, twice for fp32 queries, each off
   by a step of the magnitudes' sum), so a weight is off by that much plus 2^-21 (the exponential
   and the scale factors); 16-bit queries round weights to fp16 (2^-12), fp32 ones to 2^-23;
   adding weights and outputs in binary32 costs (keys / 16) steps at worst, over the splits and
   warps far less: 64 are allowed.  All relative to the largest |v|, plus half a step of the type.
"""
import numpy as np
import pytest

from tests.quant8_util import QMAX, append_ref, decode, sample_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F = np.float32
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(DT[dtype]).eps / 2


@pytest.fixture(scope="module")
def ctx():
    from asicfortranai_b200.quantized import Context
    c = Context(0)
    yield c
    c.device_error()          # no kernel recorded an inconsistency
    c.close()


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(DT[dtype])


def done(ctx):
    ctx.synchronize()


# ---- norm -------------------------------------------------------------------------------

def run_norm(ctx, x, r, w, dtype, code, group, pad=0, in_place=False):
    from asicfortranai_b200 import quant8
    rows, dim = x.shape
    ld = dim + pad
    def padded(a):
        t = torch.full((rows, ld), 7.0, dtype=DT[dtype], device="cuda")
        t[:, :dim] = a
        return t
    tx = padded(x)
    tr = padded(r) if r is not None else None
    to = tr if in_place else torch.full((rows, ld), 7.0, dtype=DT[dtype], device="cuda")
    groups = -(-dim // group) if group else 1
    q = torch.full((rows, ld), 99, dtype=torch.uint8, device="cuda")
    s = torch.full((rows, groups), -1.0, device="cuda")
    torch.cuda.synchronize()
    quant8.rms_norm_quant(ctx, tx.data_ptr(), w.data_ptr(), q.data_ptr(), s.data_ptr(), rows, dim, dtype=dtype,
                          code=code, group=group, residual=tr.data_ptr() if tr is not None else None,
                          residual_out=to.data_ptr(), eps=1e-5, ldx=ld, ldr=ld, ldo=ld, ldq=ld)
    done(ctx)
    assert (q[:, dim:] == 99).all() and (to[:, dim:] == 7).all()
    return to[:, :dim], q[:, :dim].cpu().numpy(), s


def check_norm(x, r, w, h_out, q, s, dtype, code, group, eps=1e-5):
    rows, dim = x.shape
    h = x.double() + (r.double() if r is not None else 0.0)
    # the stored sum: one rounding to the type of the binary32 sum
    assert ((h_out.double() - h).abs() <= h.abs() * (half_step(dtype) + U) + 2.0 ** -150).all()
    y = (h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()).cpu().numpy()
    s = s.double().cpu().numpy()
    g = group or dim
    val = np.zeros_like(y)
    d = decode(np.ascontiguousarray(q), code).reshape(rows, dim)
    for b in range(s.shape[1]):
        part = slice(b * g, min(dim, (b + 1) * g))
        top = np.abs(y[:, part]).max(1)
        want = top / float(QMAX[code])
        assert (np.abs(s[:, b] - want) <= 66 * U * want).all()
        val[:, part] = d[:, part] * s[:, b:b + 1]
        step = s[:, b:b + 1] / 2 if code == "int8" else np.maximum(np.abs(y[:, part]) * 2.0 ** -4, s[:, b:b + 1] * 2.0 ** -10)
        off = np.abs(val[:, part] - y[:, part])
        assert (off <= step * (1 + 140 * U) + 140 * U * np.abs(y[:, part])).all(), (off / step).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code,group", [("e4m3", 128), ("int8", 128), ("e4m3", 0), ("int8", 0)])
@pytest.mark.parametrize("rows,dim,pad", [(1, 1, 0), (3, 7, 1), (2, 128, 0), (5, 129, 3), (1, 8192, 0), (4, 5120, 8),
                                          (2, 13824, 0), (3, 16392, 0), (2, 32768, 0), (33, 933, 0)])
def test_norm(ctx, dtype, code, group, rows, dim, pad):
    g = torch.Generator(device="cuda").manual_seed(rows * 100003 + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(DT[dtype])
    r = (torch.randn(rows, dim, generator=g, device="cuda") * 3).to(DT[dtype])
    w = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    for res, in_place in ((r, False), (r, True), (None, False)):
        h, q, s = run_norm(ctx, x, res, w, dtype, code, group, pad, in_place)
        check_norm(x, res, w, h, q, s, dtype, code, group)


def test_norm_zero_rows_and_non_finite_rows(ctx):
    x = torch.zeros(4, 256, device="cuda")
    x[1] = 1.0
    x[2, 5] = float("nan")
    x[3, 200] = float("inf")
    w = torch.ones(256, device="cuda")
    for code in ("e4m3", "int8"):
        h, q, s = run_norm(ctx, x, None, w, "f32", code, 128)
        assert (q[0] == 0).all() and (s[0] == 0).all()
        assert torch.isfinite(s[1]).all() and np.isfinite(decode(q[1], code)).all()
        assert torch.isnan(s[2]).all() and torch.isnan(s[3]).any()


def test_norm_result_does_not_depend_on_alignment(ctx):
    """The vector and the element-wise loads give the same bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(7, 2048, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.ones(2048, device="cuda")
    a = run_norm(ctx, x, x, w, "bf16", "e4m3", 128, 0)
    b = run_norm(ctx, x, x, w, "bf16", "e4m3", 128, 1)
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all() and (a[2] == b[2]).all()


# ---- product -----------------------------------------------------------------------------

def make_product(M, N, K, seed, spread=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = -(-K // 16) * 16
    kb, nb = -(-K // 128), -(-N // 128)
    def codes(rows):
        t = torch.full((rows, ld), 0x7F, dtype=torch.uint8, device="cuda")      # NaN in the padding
        t[:, :K] = (torch.randn(rows, K, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return t
    x, w = codes(M), codes(N)
    xs = torch.rand(M, kb, generator=g, device="cuda") * 0.01 + 1e-4
    ws = torch.rand(nb, kb, generator=g, device="cuda") * 0.001 + 1e-5
    if spread:
        xs *= torch.exp2(torch.round(torch.randn(M, kb, generator=g, device="cuda") * spread))
    return x, xs, w, ws, ld


def product_ref(x, xs, w, ws, N, K):
    a = x[:, :K].view(torch.float8_e4m3fn).double() * xs.double().repeat_interleave(128, 1)[:, :K]
    b = w[:, :K].view(torch.float8_e4m3fn).double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return a @ b.t(), a.abs() @ b.abs().t()


def run_product(ctx, x, xs, w, ws, ld, M, N, K, dtype, pad=0):
    from asicfortranai_b200 import quant8
    y = torch.full((M + 1, N + pad), 5.0, dtype=DT[dtype], device="cuda")
    torch.cuda.synchronize()
    quant8.fp8_gemm(ctx, x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), M, N, K, dtype=dtype,
                    ldx=ld, ldw=ld, ldy=N + pad)
    done(ctx)
    assert (y[M] == 5).all() and (y[:M, N:] == 5).all()
    return y[:M, :N]


def check_product(y, ref, mag, K, dtype):
    kb = -(-K // 128)
    tol = ref.abs() * half_step(dtype) * 1.001 + (130 + kb) * 2 * U * mag
    if dtype == "f16":
        tol = tol + 2.0 ** -25                  # half a step of fp16's subnormal numbers
    off = (y.double() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 64, 100), (3, 130, 129), (16, 256, 1024), (17, 300, 257), (33, 129, 4096),
          (64, 1000, 640), (100, 257, 1111), (129, 384, 512), (200, 1280, 896), (256, 128, 2048), (257, 200, 300),
          (1, 5120, 13824), (5, 40000, 256), (700, 1024, 1024), (1000, 19200, 256)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(ctx, dtype, M, N, K):
    x, xs, w, ws, ld = make_product(M, N, K, M + 7 * N + 13 * K)
    ref, mag = product_ref(x, xs, w, ws, N, K)
    y = run_product(ctx, x, xs, w, ws, ld, M, N, K, dtype, pad=(M + N) % 3)
    check_product(y, ref, mag, K, dtype)
    again = run_product(ctx, x, xs, w, ws, ld, M, N, K, dtype, pad=(M + N) % 3)
    assert torch.equal(y, again)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(129, 19001, 300), (513, 9500, 1000), (2048, 8192, 1024), (300, 10240, 130), (256, 28672, 16),
                                   (1025, 5120, 512), (12, 128, 65536), (197, 5120, 1500), (40, 20000, 512), (90, 640, 9000)])
def test_product_of_many_tiles_and_of_split_ones(ctx, dtype, M, N, K):
    """Two CTAs per tile (a tile for every pair of SMs), persistent grids, and clusters along k."""
    x, xs, w, ws, ld = make_product(M, N, K, M + 3 * N + K)
    ref, mag = product_ref(x, xs, w, ws, N, K)
    for pad in (0, 1, 8):
        check_product(run_product(ctx, x, xs, w, ws, ld, M, N, K, dtype, pad=pad), ref, mag, K, dtype)


def test_product_scales_of_very_different_size(ctx):
    M, N, K = 40, 512, 2048
    x, xs, w, ws, ld = make_product(M, N, K, 9, spread=20)
    ref, mag = product_ref(x, xs, w, ws, N, K)
    check_product(run_product(ctx, x, xs, w, ws, ld, M, N, K, "f32"), ref, mag, K, "f32")


def test_product_nan_stays_in_its_row_and_column(ctx):
    M, N, K = 20, 300, 384
    x, xs, w, ws, ld = make_product(M, N, K, 10)
    x[3, 200] = 0x7F
    w[290, 5] = 0xFF
    y = run_product(ctx, x, xs, w, ws, ld, M, N, K, "f32")
    nan = torch.isnan(y)
    assert nan[3].all() and nan[:, 290].all()
    nan[3] = False
    nan[:, 290] = False
    assert not nan.any()


# ---- cache -------------------------------------------------------------------------------

class Cache:
    """A cache with arbitrary bytes (NaN codes and scales among them) behind every sequence."""

    def __init__(self, ctx, code, B, G, D, S, block, seed, gap=0):
        from asicfortranai_b200.quant8 import KV8Cache
        rng = np.random.default_rng(seed)
        nb = -(-S // block)
        self.code, self.B, self.G, self.D, self.S, self.block = code, B, G, D, S, block
        self.stride, self.sstride = G * S * D + 16 * gap, G * nb + gap
        self.codes = {n: dev(rng.integers(0, 256, B * self.stride, dtype=np.uint8)) for n in "kv"}
        sc = rng.choice(np.array([np.nan, np.inf, 1e30, -1.0], F), (2, B * self.sstride))
        self.scales = {n: dev(sc[i]) for i, n in enumerate("kv")}
        self.h = KV8Cache(ctx, self.codes["k"].data_ptr(), self.codes["v"].data_ptr(), self.scales["k"].data_ptr(),
                          self.scales["v"].data_ptr(), B, G, D, S, block, code, self.stride if gap else 0,
                          self.sstride if gap else 0)
        self.ctx = ctx

    def host(self, n):
        nb = -(-self.S // self.block)
        c = self.codes[n].cpu().numpy().reshape(self.B, self.stride)[:, :self.G * self.S * self.D]
        s = self.scales[n].cpu().numpy().reshape(self.B, self.sstride)[:, :self.G * nb]
        return c.reshape(self.B, self.G, self.S, self.D), s.reshape(self.B, self.G, nb)

    def append(self, k, v, counts, past, dtype, max_rows=None):
        rows = sum(counts)
        rs = dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        pt = dev(np.array(past, np.int32))
        torch.cuda.synchronize()
        self.h.append(k.data_ptr(), v.data_ptr(), rs.data_ptr(), pt.data_ptr(), rows, max_rows or max(counts), dtype=dtype,
                      ld=k.shape[1])
        done(self.ctx)

    def attend(self, q, heads, counts, past, dtype, scale, max_rows=None, out=None):
        rows = sum(counts)
        rs = dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        pt = dev(np.array(past, np.int32))
        mr = max_rows or max(counts)
        ws = torch.full((self.h.attention_workspace(heads, rows, mr) + 16,), 255, dtype=torch.uint8, device="cuda")
        out = torch.full_like(q, 3.0) if out is None else out
        torch.cuda.synchronize()
        self.h.attention(q.data_ptr(), out.data_ptr(), heads, rs.data_ptr(), pt.data_ptr(), rows, mr, scale, dtype=dtype,
                         ldq=q.shape[1], ldo=q.shape[1], workspace=ws.data_ptr(), workspace_bytes=ws.numel())
        done(self.ctx)
        return out


def rounded(a, dtype):
    """numpy values in the type's precision, as float32"""
    return torch.from_numpy(np.asarray(a, F)).to(DT[dtype]).float().numpy()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D,block,S", [(64, 16, 70), (128, 64, 200), (256, 128, 300), (128, 32, 33)])
def test_append_equals_the_definition(ctx, dtype, code, D, block, S):
    B, G = 3, 2
    c = Cache(ctx, code, B, G, D, S, block, 11, gap=2)
    rng = np.random.default_rng(12)
    past = [0, 0, 0]
    # several calls, each a different number of tokens per sequence, growing and shrinking values
    for step, counts in enumerate([[1, 5, 0], [S // 3, 0, 2], [1, 1, 1], [3, block, 1], [1, 1, S - 4 - 0], [0, 2, 0]]):
        counts = [min(n, S - p) for n, p in zip(counts, past)]
        if sum(counts) == 0:
            continue
        rows = sum(counts)
        size = [1.0, 0.1, 20.0, 1e-3, 3.0, 1e4][step]
        new = {n: rounded(rng.normal(0, size, (rows, G * D)), dtype) for n in "kv"}
        if step == 2:
            new["k"][0, :3] = [np.inf, -np.inf, np.nan]
            new["v"][1, 7] = np.nan
        if step == 1:
            new["v"][-1] = 0.0
        before = {n: c.host(n) for n in "kv"}
        pad = 5
        t = {n: torch.full((rows, G * D + pad), 9.0, dtype=DT[dtype], device="cuda") for n in "kv"}
        for n in "kv":
            t[n][:, :G * D] = dev(new[n], dtype)
        c.append(t["k"], t["v"], counts, past, dtype)
        for n in "kv":
            codes, scales = before[n]
            codes, scales = codes.copy(), scales.copy()
            r = 0
            for b in range(B):
                for g in range(G):
                    if counts[b]:
                        x = new[n][r:r + counts[b], g * D:(g + 1) * D]
                        codes[b, g], scales[b, g] = append_ref(codes[b, g], scales[b, g], x, past[b], block, code)
                r += counts[b]
            got_c, got_s = c.host(n)
            np.testing.assert_array_equal(got_s.view(np.uint32), scales.view(np.uint32), err_msg=f"{n} {step}")
            np.testing.assert_array_equal(got_c, codes, err_msg=f"{n} {step}")
        past = [p + n for p, n in zip(past, counts)]


def attention_ref(c, q, heads, counts, past, scale):
    """float64 outputs, the weights' score magnitudes and the largest |v|, per row and head"""
    G, D, block = c.G, c.D, c.block
    out = np.zeros((sum(counts), heads, D))
    mag, vmax = np.zeros((sum(counts), heads)), np.zeros((sum(counts), heads))
    vals = {}
    for n in "kv":
        codes, scales = c.host(n)
        with np.errstate(invalid="ignore", over="ignore"):
            vals[n] = decode(codes, c.code) * np.repeat(scales.astype(np.float64), block, 2)[:, :, :c.S, None]
    r = 0
    for b, cnt in enumerate(counts):
        if cnt == 0:
            continue
        L = past[b] + cnt
        k = torch.from_numpy(vals["k"][b, :, :L].copy()).cuda()
        v = torch.from_numpy(vals["v"][b, :, :L].copy()).cuda()
        qs = torch.from_numpy(q[r:r + cnt].reshape(cnt, heads, D).astype(np.float64)).cuda()
        seen = torch.arange(L, device="cuda")[None] <= past[b] + torch.arange(cnt, device="cuda")[:, None]
        for h in range(heads):
            g = h // (heads // G)
            s = (qs[:, h] @ k[g].t()) * scale
            w = torch.softmax(s.masked_fill(~seen, -torch.inf), 1)
            out[r:r + cnt, h] = (w @ v[g]).cpu().numpy()
            mag[r:r + cnt, h] = ((qs[:, h].abs() @ k[g].abs().t()) * abs(scale) * seen).amax(1).cpu().numpy()
            vmax[r:r + cnt, h] = [float(v[g, :past[b] + i + 1].abs().max()) for i in range(cnt)]
        r += cnt
    return out, mag, vmax


def check_attention(got, ref, mag, vmax, D, dtype):
    terms = 2 if dtype == "f32" else 1
    weight = (D // 16 * terms + 4) * 2 * U * mag * 2 + 2.0 ** -21 + (2.0 ** -23 if dtype == "f32" else 2.0 ** -12)
    tol = np.abs(ref) * half_step(dtype) + (weight + 64 * 2 * U)[..., None] * vmax[..., None] * (1 + 2.0 ** -8)
    off = np.abs(got - ref)
    assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())


ATTN = [  # heads, kv heads, D, block, max_seq, counts, past
    (1, 1, 64, 16, 1, [1], [0]),
    (2, 2, 128, 64, 40, [1, 1], [0, 39]),
    (8, 1, 128, 64, 700, [1, 1, 1], [699, 1, 300]),
    (6, 2, 64, 32, 1500, [1, 0, 1], [1400, 5, 17]),
    (4, 4, 256, 16, 333, [1, 1], [332, 16]),
    (64, 8, 128, 64, 2048, [1], [2000]),
    (5, 1, 128, 128, 5000, [1, 1], [4999, 129]),
    (20, 1, 64, 64, 900, [1], [800]),                    # more than 16 heads on one kv head
    (4, 2, 128, 64, 300, [7, 1, 33], [0, 250, 60]),
    (3, 1, 128, 16, 400, [130, 0, 2], [3, 9, 397]),
    (8, 2, 64, 32, 600, [257], [300]),
    (2, 1, 256, 64, 200, [17, 64], [100, 0]),
    (1, 1, 128, 64, 70, [70], [0]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", ATTN, ids=[str(i) for i in range(len(ATTN))])
def test_append_then_attention(ctx, dtype, code, case):
    heads, G, D, block, S, counts, past = case
    rng = np.random.default_rng(abs(hash((heads, D, S))) % 1000)
    B = len(counts)
    c = Cache(ctx, code, B, G, D, S, block, 5, gap=1)
    # history in one append, then the rows of the call
    if sum(past):
        hist = {n: dev(rng.normal(0, 1, (sum(past), G * D)), dtype) for n in "kv"}
        hist["k"] *= dev(np.exp(rng.normal(0, 1, (sum(past), 1))), dtype)
        hist["v"] *= dev(np.exp(rng.normal(0, 2, (sum(past), 1))), dtype)       # v scales far apart
        c.append(hist["k"], hist["v"], past, [0] * B, dtype)
    rows = sum(counts)
    new = {n: dev(rng.normal(0, 1, (rows, G * D)), dtype) for n in "kv"}
    c.append(new["k"], new["v"], counts, past, dtype)
    q = torch.full((rows, heads * D + 3), 4.0, dtype=DT[dtype], device="cuda")
    q[:, :heads * D] = dev(rng.normal(0, 1, (rows, heads * D)), dtype)
    scale = D ** -0.5
    out = c.attend(q, heads, counts, past, dtype, scale)
    assert (out[:, heads * D:] == 3).all()
    got = out[:, :heads * D].double().cpu().numpy().reshape(rows, heads, D)
    ref, mag, vmax = attention_ref(c, q[:, :heads * D].float().cpu().numpy(), heads, counts, past, scale)
    check_attention(got, ref, mag, vmax, D, dtype)
    assert torch.equal(out, c.attend(q, heads, counts, past, dtype, scale))
    # a larger max_rows than needed changes nothing but the split
    if max(counts) < rows:
        more = c.attend(q, heads, counts, past, dtype, scale, max_rows=min(rows, S))
        got = more[:, :heads * D].double().cpu().numpy().reshape(rows, heads, D)
        check_attention(got, ref, mag, vmax, D, dtype)


def test_attention_large_scores_and_tiny_queries(ctx):
    """Scores of hundreds (one key takes all the weight) and queries near the smallest numbers."""
    rng = np.random.default_rng(8)
    S, D, heads = 500, 128, 4
    c = Cache(ctx, "int8", 1, 1, D, S, 64, 2)
    kv = {n: dev(rng.normal(0, 1, (S, D)), "f32") for n in "kv"}
    c.append(kv["k"], kv["v"], [S], [0], "f32")
    for size in (100.0, 1e-30, 0.0):
        q = dev(rng.normal(0, 1, (1, heads * D)) * size, "f32")
        out = c.attend(q, heads, [1], [S - 1], "f32", 0.3)
        ref, mag, vmax = attention_ref(c, q.cpu().numpy(), heads, [1], [S - 1], 0.3)
        check_attention(out.double().cpu().numpy().reshape(1, heads, D), ref, mag, vmax, D, "f32")


def test_attention_zero_and_tiny_value_blocks(ctx):
    rng = np.random.default_rng(9)
    S, D = 256, 64
    c = Cache(ctx, "e4m3", 1, 1, D, S, 16, 2)
    k = rng.normal(0, 1, (S, D))
    v = rng.normal(0, 1, (S, D))
    v[:64] = 0.0
    v[64:128] *= 1e-25
    v[200:] = 0.0
    tk, tv = dev(k, "f32"), dev(v, "f32")
    c.append(tk, tv, [S], [0], "f32")
    q = dev(rng.normal(0, 1, (S, D)), "f32")
    out = c.attend(q, 1, [S], [0], "f32", 0.125)
    ref, mag, vmax = attention_ref(c, q.cpu().numpy(), 1, [S], [0], 0.125)
    check_attention(out.double().cpu().numpy().reshape(S, 1, D), ref, mag, vmax, D, "f32")


def test_inconsistent_rows_are_left_out_and_reported():
    from asicfortranai_b200 import Q35Error
    from asicfortranai_b200.quantized import Context
    own = Context(0)
    c = Cache(own, "int8", 2, 1, 64, 32, 16, 3)
    kv = dev(np.ones((4, 64)), "f32")
    c.append(kv, kv, [2, 2], [0, 0], "f32")
    own.device_error()
    before = c.host("k")
    q = dev(np.ones((4, 64)), "f32")
    # sequence 1 would pass max_seq; sequence 0 goes on as usual
    c.append(kv, kv, [2, 2], [2, 31], "f32")
    out = c.attend(q, 1, [2, 2], [2, 31], "f32", 0.1)
    with pytest.raises(Q35Error):
        own.device_error()
    after = c.host("k")
    np.testing.assert_array_equal(before[0][1], after[0][1])
    assert (out[2:] == 3).all() and (out[:2] != 3).all()
    # negative history, more rows than max_rows
    for counts, past, mr in (([2, 2], [-1, 2], 2), ([1, 3], [2, 2], 1)):
        c.append(kv, kv, counts, past, "f32", max_rows=mr)
        with pytest.raises(Q35Error):
            own.device_error()
    own.device_error()
    own.close()


def test_long_offsets():
    """Codes beyond 2^31 bytes into the arrays (one sequence of a strided cache)."""
    from asicfortranai_b200.quant8 import KV8Cache
    from asicfortranai_b200.quantized import Context
    ctx = Context(0)
    G, D, S, block = 3, 256, 3_000_000, 128          # 768 MB a head: head 2 starts past 2^31
    k = torch.zeros(G * S * D, dtype=torch.uint8, device="cuda")
    v = torch.zeros(G * S * D, dtype=torch.uint8, device="cuda")
    nb = -(-S // block)
    ks, vs = (torch.zeros(G * nb, device="cuda") for _ in "kv")
    c = KV8Cache(ctx, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), 1, G, D, S, block, "int8")
    past = S - 1
    rs, pt = dev(np.array([0, 1], np.int32)), dev(np.array([past], np.int32))
    rng = np.random.default_rng(1)
    nk, nv, q = (dev(rng.normal(0, 1, (1, G * D)), "bf16") for _ in range(3))
    ws = torch.zeros(c.attention_workspace(G, 1, 1) + 16, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    c.append(nk.data_ptr(), nv.data_ptr(), rs.data_ptr(), pt.data_ptr(), 1, 1, dtype="bf16")
    c.attention(q.data_ptr(), out.data_ptr(), G, rs.data_ptr(), pt.data_ptr(), 1, 1, 1.0, dtype="bf16",
                workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    ctx.device_error()
    for g in range(G):
        row = slice(g * D, (g + 1) * D)
        at = (g * S + past) * D
        s = float(vs[(g + 1) * nb - 1])
        got = v[at:at + D].view(torch.int8).double() * s
        assert (got - nv[0, row].double()).abs().max() <= s * 0.5001
        sk = float(ks[(g + 1) * nb - 1])
        score = float((q[0, row].double() * k[at:at + D].view(torch.int8).double() * sk).sum())
        # every other key is zero: score 0, value 0
        w = 1.0 / (1.0 + past * np.exp(-score))
        want = got * w
        assert (out[0, row].double() - want).abs().max() <= want.abs().max() * (2.0 ** -8 + 2.0 ** -10)
    ctx.close()


# ---- sampling ----------------------------------------------------------------------------

def run_sampler(ctx, lg, dtype, T=None, k=None, p=None, m=None, u=None, ld=None):
    from asicfortranai_b200 import sampling
    R, V = lg.shape
    ld = V if ld is None else ld
    t = torch.full((R, ld), 50.0, dtype=DT[dtype], device="cuda")
    t[:, :V] = dev(lg.astype(F), dtype)
    f = [None if a is None else dev(np.asarray(a, F)) for a in (T, p, m, u)]
    tk = None if k is None else dev(np.asarray(k, np.int32))
    tok = torch.full((R + 1,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((R + 1,), -7.0, device="cuda")
    ptr = lambda a: None if a is None else a.data_ptr()  # noqa: E731
    torch.cuda.synchronize()
    sampling.sample_filtered_rows(ctx, t.data_ptr(), R, V, ptr(f[3]), tok.data_ptr(), temperature=ptr(f[0]), top_k=ptr(tk),
                                  top_p=ptr(f[1]), min_p=ptr(f[2]), probs=pr.data_ptr(), dtype=dtype, ld=ld)
    done(ctx)
    assert tok[R] == -7 and pr[R] == -7
    return tok[:R].cpu().numpy(), pr[:R].cpu().numpy(), t[:, :V].double().cpu().numpy()


def check_sampler(ctx, lg, dtype, T, k, p, m, u, ld=None):
    R = len(lg)
    tok, pr, lgd = run_sampler(ctx, lg, dtype, T, k, p, m, u, ld)
    one = lambda a, r, d: d if a is None else float(F(a[r]))  # noqa: E731
    for r in range(R):
        want, prob = sample_ref(lgd[r], one(T, r, 1.0), 0 if k is None else int(k[r]), one(p, r, 1.0), one(m, r, 0.0),
                                one(u, r, 0.0))
        assert tok[r] == want, (r, tok[r], want, one(T, r, 1.0), None if k is None else k[r], one(p, r, 1.0),
                                one(m, r, 0.0), one(u, r, 0.0))
        # weights are integers of 2^-40 (2^-20 of a weight of 2^-20), the result binary32
        assert abs(pr[r] - prob) <= prob * 2.0 ** -23 + 2.0 ** -30, (r, pr[r], prob)


ONE_MINUS = float(np.nextafter(F(1), F(0)))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,R", [(1, 48), (2, 48), (31, 48), (33, 48), (1000, 48), (4097, 48), (32000, 48), (100277, 48),
                                 (9000, 200), (131072, 5), (400001, 5), (401408, 5)])
def test_sampler(ctx, dtype, V, R):
    rng = np.random.default_rng(V)
    lg = rng.normal(0, 2.5, (R, V))
    lg[::5] = np.round(lg[::5] * 2) / 2                        # ties
    lg[1::7] = rng.normal(0, 0.01, (len(lg[1::7]), V))         # flat
    lg[3, : V // 2] = -np.inf
    lg[4, V // 3:] = np.nan
    lg[4, 0] = 0.5
    T = rng.choice([0.3, 0.7, 1.0, 1.5, 0.0], R)
    k = rng.choice([0, -1, 1, 2, 5, 40, 999, V - 1, V, V + 5], R)
    p = rng.choice([1.0, 0.99, 0.9, 0.5, 0.01, 0.0, 1.5], R)
    m = rng.choice([0.0, 0.0, 0.01, 0.1, 1.0, 1.5], R)
    u = rng.random(R).astype(F)
    u[:4] = [0.0, ONE_MINUS, 0.5, 0.0]
    check_sampler(ctx, lg, dtype, T, k, p, m, u)
    check_sampler(ctx, lg, dtype, None, None, None, None, u, ld=V + 3)
    check_sampler(ctx, lg, dtype, T, None, p, None, u)
    check_sampler(ctx, lg, dtype, None, k, None, m, u)


def test_sampler_equal_logits_take_the_lowest_indices(ctx):
    V = 3000
    lg = np.zeros((6, V))
    lg[3:, 100] = 1.0
    lg[5, :] = -0.0
    lg[5, ::2] = 0.0
    u = np.full(6, ONE_MINUS)
    check_sampler(ctx, lg, "f32", None, [10, 0, 0, 10, 0, 10], [1, 0.25, 1, 1, 0.25, 1], [0, 0, 1, 0, 0, 0], u)


def test_sampler_masked_rows_and_infinities(ctx):
    V = 700
    lg = np.full((5, V), -np.inf)
    lg[1] = np.nan
    lg[2, 333] = -1e30
    lg[3] = np.random.default_rng(0).normal(0, 1, V)
    lg[3, [5, 77]] = np.inf
    lg[4] = np.finfo(F).min                                    # a mask of the type's lowest value
    lg[4, 42] = 1.0
    u = np.array([0.3, 0.3, 0.9, 0.7, 0.99])
    tok, pr, _ = run_sampler(ctx, lg, "f32", u=u)
    np.testing.assert_array_equal(tok, [0, 0, 334, 78, 43])
    np.testing.assert_array_equal(pr, np.array([0, 0, 1, 0.5, 1], F))
    check_sampler(ctx, lg[2:], "f32", None, [3, 0, 50], [0.9, 1, 0.9], None, u[2:])
