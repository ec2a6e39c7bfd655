"""RMSNorm with 8-bit output at the edges of binary32: rows with elements that are no numbers, rows whose
squares leave the range.  Tolerances are those of tests/test_quant8_gpu.py."""
import threading

import numpy as np
import pytest

from tests.quant8_util import decode

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_quant8_gpu import DT, check_norm, ctx  # noqa: E402

__all__ = ["ctx"]


def norm(ctx, x, r, w, dtype, code, group, eps=1e-5):
    """h, codes, scales of contiguous rows"""
    from asicfortranai_b200 import quant8
    rows, dim = x.shape
    h = torch.full((rows, dim), 7.0, dtype=DT[dtype], device="cuda")
    q = torch.full((rows, dim), 99, dtype=torch.uint8, device="cuda")
    s = torch.full((rows, -(-dim // group) if group else 1), -1.0, device="cuda")
    torch.cuda.synchronize()
    quant8.rms_norm_quant(ctx, x.data_ptr(), w.data_ptr(), q.data_ptr(), s.data_ptr(), rows, dim, dtype=dtype, code=code,
                          group=group, residual=None if r is None else r.data_ptr(), residual_out=h.data_ptr(), eps=eps)
    ctx.synchronize()
    return h, q, s


# one row a CTA, several rows a CTA, rows that are no whole vectors
SHAPES = [(12, 1000), (12, 5120), (700, 640), (700, 1001), (450, 13824)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("code,group", [("e4m3", 128), ("int8", 128), ("e4m3", 0), ("int8", 0)])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_a_row_with_an_element_that_is_no_number(ctx, rows, dim, code, group, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(DT[dtype])
    r = torch.randn(rows, dim, generator=g, device="cuda").to(DT[dtype])
    w = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    w[: dim // 2 : 7] = 0.0
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i, (t, at, v) in enumerate([(x, 5, "nan"), (x, dim - 1, "inf"), (r, 0, "-inf"), (r, 300, "nan"), (x, 7, "inf")]):
        t[2 * i, at] = float(v)
        bad[2 * i] = True
    for at, v in ((40, "inf"), (41, "-inf")):            # a sum of opposite infinities
        x[2, at], r[2, at] = float(v), -float(v)
    bad[rows - 1] = True
    x[rows - 1, dim // 2] = float("nan")
    h, q, s = norm(ctx, x, r, w, dtype, code, group)
    assert torch.isnan(s[bad]).all()
    ok = ~bad
    check_norm(x[ok], r[ok], w, h[ok], q[ok].cpu().numpy(), s[ok], dtype, code, group)
    want = (x.float() + r.float()).to(DT[dtype])
    assert torch.equal(h.nan_to_num(1.0, 2.0, 3.0), want.nan_to_num(1.0, 2.0, 3.0))


@pytest.mark.parametrize("code,group", [("e4m3", 128), ("int8", 0)])
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_whose_squares_leave_the_range(ctx, dtype, rows, dim, code, group):
    """Magnitudes from 2^-140 to 2^127, each row of one size, ordinary rows between them."""
    g = torch.Generator(device="cuda").manual_seed(dim + 1)
    w = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    # (at most 2^-10 of a row's largest element away from it: every element a normal number, or exact)
    base = (1 + torch.rand(rows, dim, generator=g, device="cuda")) * (1 - 2 * torch.randint(0, 2, (rows, dim), generator=g, device="cuda"))
    for eps, powers in ((0.0, [-120, -100, -70, -60, 0, 50, 64, 100, 126]), (1e-38, [-140, -100, -63, -61, 3, 70]),
                        (1e-5, [0, 60, 65, 90, 126, -120, -30])):
        e = torch.tensor([powers[i % len(powers)] for i in range(rows)], device="cuda")
        # (normal numbers alone: what lies below 2^-126 is not rounded as the type's half step says)
        x = torch.ldexp(base.double(), e[:, None]).float()
        x = torch.where(x.abs() < 2.0 ** -126, torch.sign(x) * 2.0 ** -126, x).to(DT[dtype])
        h, q, s = norm(ctx, x, None, w, dtype, code, group, eps)
        normal = (e > -120) | (eps == 0.0)               # (scales of the others lie below binary32's normal numbers)
        assert torch.isfinite(s).all()
        eps32 = float(np.float32(eps))
        check_norm(x[normal], None, w, h[normal], q[normal].cpu().numpy(), s[normal], dtype, code, group, eps32)


def test_sums_that_pass_the_range_are_infinite(ctx):
    x = torch.full((3, 256), 3e38, device="cuda")
    x[1] = 1.0
    x[2, 1:] = -1.0
    w = torch.ones(256, device="cuda")
    h, q, s = norm(ctx, x, x, w, "f32", "int8", 128)
    assert torch.isnan(s[[0, 2]]).all() and (s[1] > 0).all()
    assert (decode(q[1].cpu().numpy(), "int8") == 127).all()


def test_two_threads_with_rows_of_different_length():
    """Two contexts of one process, rows whose weights take 64 and 52 KB of shared memory."""
    from asicfortranai_b200 import quant8
    from asicfortranai_b200.quantized import Context
    rows = 152
    jobs = []
    for dim in (16384, 13312):
        c = Context(0)
        x = torch.randn(rows, dim, device="cuda").bfloat16()
        w = torch.ones(dim, device="cuda")
        q = torch.zeros(rows, dim, dtype=torch.uint8, device="cuda")
        s = torch.zeros(rows, dim // 128, device="cuda")
        jobs.append((c, x, w, q, s, dim))
    torch.cuda.synchronize()
    failed = []

    def go(c, x, w, q, s, dim):
        try:
            for i in range(3000):
                quant8.rms_norm_quant(c, x.data_ptr(), w.data_ptr(), q.data_ptr(), s.data_ptr(), rows, dim)
                if i % 100 == 99:
                    c.synchronize()
        except Exception as e:      # noqa: BLE001  (raised in the thread: reported by the test)
            failed.append((dim, i, str(e)))

    threads = [threading.Thread(target=go, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for c, x, w, q, s, dim in jobs:
        c.synchronize()
        check_norm(x, None, w, x, q.cpu().numpy(), s, "bf16", "e4m3", 128)
        c.close()


def test_one_row_in_place_whatever_the_strides(ctx):
    """A single row has no stride that could make the sum's buffer another one than its input."""
    from asicfortranai_b200 import quant8
    dim = 640
    x, r = (torch.randn(1, dim, device="cuda").bfloat16() for _ in "xr")
    w = torch.ones(dim, device="cuda")
    h, q, s = norm(ctx, x, r, w, "bf16", "e4m3", 128)
    q2, s2 = torch.zeros_like(q), torch.zeros_like(s)
    torch.cuda.synchronize()
    quant8.rms_norm_quant(ctx, x.data_ptr(), w.data_ptr(), q2.data_ptr(), s2.data_ptr(), 1, dim, residual=r.data_ptr(),
                          residual_out=r.data_ptr(), ldr=dim, ldo=4 * dim)
    ctx.synchronize()
    assert torch.equal(r, h) and torch.equal(q, q2) and torch.equal(s, s2)
