"""Attention of more rows than 65535 tiles of 16 (row, head) pairs hold, without a workspace.  Rows are
compared with 64 bits, with tests/test_quant8_gpu.py's tolerance."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_quant8_gpu import check_attention, ctx, dev  # noqa: E402

__all__ = ["ctx"]


@pytest.mark.parametrize("heads,n", [(16, 65537), (64, 16500)])
def test_a_prompt_of_many_rows(ctx, heads, n):
    from asicfortranai_b200.quant8 import KV8Cache
    D, block, S = 64, 128, n + 3
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = (torch.randint(-127, 128, (S, D), generator=g, device="cuda", dtype=torch.int8) for _ in "kv")
    ks, vs = (torch.rand(-(-S // block), generator=g, device="cuda") * 0.01 + 0.005 for _ in "kv")
    c = KV8Cache(ctx, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), 1, 1, D, S, block, "int8")
    q = torch.randn(n, heads * D, generator=g, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    rs, pt = dev(np.array([0, n], np.int32)), dev(np.array([3], np.int32))
    assert c.attention_workspace(heads, n, n) == 0
    torch.cuda.synchronize()
    c.attention(q.data_ptr(), out.data_ptr(), heads, rs.data_ptr(), pt.data_ptr(), n, n, D ** -0.5)
    ctx.device_error()
    kd = k.double() * ks.double().repeat_interleave(block)[:S, None]
    vd = v.double() * vs.double().repeat_interleave(block)[:S, None]
    for row in (0, 1, 4095, n // 2, n - 2, n - 1):
        L = row + 4
        qr = q[row].view(heads, D).double()
        s = qr @ kd[:L].t() * D ** -0.5
        ref = torch.softmax(s, 1) @ vd[:L]
        mag = (qr.abs() @ kd[:L].abs().t() * D ** -0.5).amax(1)
        vmax = vd[:L].abs().max().expand(heads)
        check_attention(out[row].view(heads, D).double().cpu().numpy(), ref.cpu().numpy(), mag.cpu().numpy(),
                        vmax.cpu().numpy(), D, "bf16")
