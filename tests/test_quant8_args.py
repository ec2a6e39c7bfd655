"""The 8-bit operators refuse bad arguments before any device work, and their references'
rounding agrees with torch's (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

from asicfortranai_b200 import _lib
from asicfortranai_b200.quant8 import KV8CacheStruct
from tests.quant8_util import E4M3, decode, encode, sample_ref

INVALID = 1
CTX = C.create_string_buffer(4096)          # a context that no refused call may look into
P = 0x1000                                  # an aligned address that no refused call may touch


def _ctx():
    return C.addressof(CTX)


def norm(**kw):
    a = dict(ctx=_ctx(), dtype=1, x=P, ldx=256, r=P, ldr=256, ro=P, ldo=256, w=P, eps=1e-5, rows=2, dim=256, code=1,
             group=128, q=P, ldq=256, s=P)
    a.update(kw)
    return _lib.load().q35_rms_norm_quant_dev(*a.values())


@pytest.mark.parametrize("kw", [
    dict(ctx=None), dict(dtype=3), dict(dtype=-1), dict(code=2), dict(rows=-1), dict(dim=0), dict(dim=32769),
    dict(group=64), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(w=None), dict(q=None), dict(s=None),
    dict(ldx=255), dict(ldr=255), dict(ldo=255), dict(ldq=255), dict(x=P + 1), dict(w=P + 2), dict(s=P + 2),
    dict(ro=P + 2), dict(ldo=512), dict(r=P + 512)])
def test_norm_refuses(kw):
    assert norm(**kw) == INVALID
    assert _lib.last_error()


def gemm(**kw):
    a = dict(ctx=_ctx(), x=P, ldx=256, xs=P, w=P, ldw=256, ws=P, dtype=1, y=P, ldy=64, M=2, N=64, K=256)
    a.update(kw)
    return _lib.load().q35_fp8_gemm_dev(*a.values())


@pytest.mark.parametrize("kw", [
    dict(ctx=None), dict(dtype=3), dict(M=-1), dict(M=65537), dict(N=-1), dict(N=(1 << 24) + 1), dict(K=0),
    dict(K=131073), dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(ldx=240),
    dict(ldw=240), dict(ldy=63), dict(ldx=264), dict(ldw=264), dict(x=P + 8), dict(w=P + 8), dict(xs=P + 2),
    dict(ws=P + 1), dict(y=P + 1)])
def test_gemm_refuses(kw):
    assert gemm(**kw) == INVALID
    assert _lib.last_error()


def cache(**kw):
    a = dict(code=0, seqs=2, kv_heads=2, head_dim=128, max_seq=100, block=64, k=P, v=P, k_scale=P, v_scale=P,
             seq_stride=0, scale_seq_stride=0)
    a.update(kw)
    return C.byref(KV8CacheStruct(*a.values()))


BAD_CACHE = [dict(code=2), dict(seqs=0), dict(kv_heads=0), dict(head_dim=96), dict(max_seq=0), dict(block=8),
             dict(block=48), dict(k=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 4), dict(k_scale=P + 2),
             dict(seq_stride=100), dict(seq_stride=16), dict(scale_seq_stride=3), dict(seqs=40000),
             dict(max_seq=(1 << 30) + 1)]


def append(c=None, **kw):
    a = dict(ctx=_ctx(), c=c if c is not None else cache(), dtype=1, k=P, v=P, ld=256, rs=P, past=P, rows=2, max_rows=1)
    a.update(kw)
    return _lib.load().q35_kv8_append_dev(*a.values())


def attend(c=None, **kw):
    a = dict(ctx=_ctx(), c=c if c is not None else cache(), dtype=1, q=P, ldq=512, heads=4, out=P, ldo=512, rs=P,
             past=P, rows=2, max_rows=1, scale=0.1, ws=P, wsb=1 << 30)
    a.update(kw)
    return _lib.load().q35_kv8_attention_dev(*a.values())


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_cache_refused(kw):
    assert append(cache(**kw)) == INVALID
    assert attend(cache(**kw)) == INVALID
    assert _lib.load().q35_kv8_attention_workspace(cache(**kw), 4, 2, 1) == -1


ROWS = [dict(rows=-1), dict(max_rows=-1), dict(max_rows=3), dict(max_rows=0), dict(rows=200, max_rows=101),
        dict(rs=None), dict(past=None)]


@pytest.mark.parametrize("kw", ROWS + [dict(ctx=None), dict(c=None, ctx=None), dict(dtype=5), dict(k=None),
                                       dict(v=None), dict(ld=255), dict(k=P + 1)])
def test_append_refuses(kw):
    assert append(**kw) == INVALID
    assert _lib.last_error()


@pytest.mark.parametrize("kw", ROWS + [
    dict(ctx=None), dict(dtype=5), dict(q=None), dict(out=None), dict(heads=0), dict(heads=3), dict(ldq=511),
    dict(ldo=511), dict(q=P + 1), dict(out=P + 1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(ws=None), dict(wsb=8), dict(ws=P + 8)])
def test_attention_refuses(kw):
    if any(k in kw for k in ("ws", "wsb")):
        kw["c"] = cache(max_seq=100000)     # long enough to be split, so a workspace is needed
        assert _lib.load().q35_kv8_attention_workspace(kw["c"], 4, 2, 1) > 0
    assert attend(**kw) == INVALID
    assert _lib.last_error()


def test_null_cache_refused():
    lib = _lib.load()
    assert lib.q35_kv8_append_dev(_ctx(), None, 1, P, P, 256, P, P, 2, 1) == INVALID
    assert lib.q35_kv8_attention_workspace(None, 4, 2, 1) == -1


def sample(**kw):
    a = dict(ctx=_ctx(), dtype=0, lg=P, ld=100, rows=2, V=100, T=P, k=P, p=P, m=P, u=P, tok=P, probs=P)
    a.update(kw)
    return _lib.load().q35_sample_filtered_dev(*a.values())


@pytest.mark.parametrize("kw", [dict(ctx=None), dict(dtype=4), dict(rows=-1), dict(V=0), dict(V=(1 << 22) + 1),
                                dict(lg=None), dict(u=None), dict(tok=None), dict(ld=99), dict(lg=P + 2),
                                dict(T=P + 1), dict(k=P + 2), dict(u=P + 1), dict(probs=P + 3)])
def test_sampler_refuses(kw):
    assert sample(**kw) == INVALID
    assert _lib.last_error()


def test_empty_calls_do_nothing():
    assert norm(rows=0, x=None, w=None) == 0
    assert gemm(M=0, x=None) == 0 and gemm(N=0, ldy=0, w=None) == 0
    assert append(rows=0, max_rows=0, k=None) == 0 and attend(rows=0, max_rows=0, q=None) == 0
    assert sample(rows=0, lg=None) == 0
    assert _lib.load().q35_kv8_attention_workspace(cache(), 4, 0, 0) == 0


def test_cache_struct_matches_the_header(tmp_path):
    import json
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "l.c"
    names = [f for f, _ in KV8CacheStruct._fields_]
    body = "".join(f'printf("\\"{f}\\": %zu, ", offsetof(q35_kv8_cache, {f}));' for f in names)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "q35.h"\nint main(void) { printf("{"); ' + body +
                   'printf("\\"size\\": %zu}", sizeof(q35_kv8_cache)); return 0; }\n')
    exe = tmp_path / "l"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = json.loads(subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout)
    assert got == {**{f: getattr(KV8CacheStruct, f).offset for f in names}, "size": C.sizeof(KV8CacheStruct)}


def test_reference_codes_round_as_torch_does():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(3)
    mid = (E4M3[:126] + E4M3[1:127]) / 2
    v = np.concatenate([rng.normal(0, 60, 4000), rng.normal(0, 0.01, 4000), mid, -mid, E4M3[:127], [448, -448, 0]])
    v = np.clip(v.astype(np.float32), -448, 448)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(encode(v, "e4m3"), want)
    all_codes = np.arange(256, dtype=np.uint8)
    np.testing.assert_array_equal(decode(all_codes, "e4m3"),
                                  torch.from_numpy(all_codes).view(torch.float8_e4m3fn).double().numpy())


def test_reference_sampler_on_known_rows():
    lg = np.log(np.array([0.1, 0.4, 0.3, 0.2]))
    assert sample_ref(lg, 1.0, 0, 1.0, 0.0, 0.05)[0] == 1
    assert sample_ref(lg, 1.0, 0, 1.0, 0.0, 0.5)[0] == 3 or sample_ref(lg, 1.0, 0, 1.0, 0.0, 0.49)[0] == 2
    assert sample_ref(lg, 0.0, 0, 1.0, 0.0, 0.9) == (2, 1.0)
    tok, prob = sample_ref(lg, 1.0, 2, 1.0, 0.0, 0.99)          # keeps 0.4 and 0.3
    assert tok == 3 and abs(prob - 0.3 / 0.7) < 1e-12
    assert sample_ref(lg, 1.0, 0, 0.5, 0.0, 0.99)[0] == 3       # 0.4 does not reach 0.5, 0.7 does
    assert sample_ref(lg, 1.0, 0, 1.0, 0.6, 0.99)[0] == 3       # at least 0.24
    assert sample_ref(np.full(4, -np.inf), 1.0, 0, 1.0, 0.0, 0.5) == (0, 0.0)


def test_the_program_takes_a_cache_format():
    import os
    import subprocess

    from asicfortranai_b200 import build
    build.build()
    cli = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asicfortranai_b200", "bin", "llama_generate")
    assert "--kv-cache" in subprocess.run([cli, "--help"], capture_output=True, text=True).stdout
    for bad in (["--kv-cache", "int7"], ["--kv-cache"]):
        assert subprocess.run([cli, *bad], capture_output=True).returncode == 2
