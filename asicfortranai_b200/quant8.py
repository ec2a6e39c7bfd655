"""The 8-bit operators of a serving step over libq35.so, on device arrays (pointers such as
torch tensors' data_ptr()), enqueued on the context's stream:

    rms_norm_quant(ctx, x, weight, q, scales, rows, dim, residual=r, residual_out=r)   # norm -> codes
    fp8_gemm(ctx, q, scales, w, w_scales, y, M, N, K)                                  # e4m3 product
    cache = KV8Cache(ctx, k, v, k_scale, v_scale, seqs=8, kv_heads=8, head_dim=128, max_seq=8192)
    cache.append(k_new, v_new, row_start, past, rows, max_rows)                        # fills the cache
    cache.attention(q, out, heads, row_start, past, rows, max_rows, scale=128 ** -0.5,
                    workspace=ws, workspace_bytes=cache.attention_workspace(heads, rows, max_rows))

The sampler of such a step is sampling.sample_filtered_rows.  Element types are "f32", "bf16"
or "f16"; 8-bit codes are "int8" or "e4m3".
"""
from __future__ import annotations

import ctypes as C

from . import _lib


def rms_norm_quant(ctx, x: int, weight: int, q: int, scales: int, rows: int, dim: int, dtype: str = "bf16",
                   code: str = "e4m3", group: int = 128, residual: int | None = None,
                   residual_out: int | None = None, eps: float = 1e-5, ldx: int | None = None,
                   ldr: int | None = None, ldo: int | None = None, ldq: int | None = None) -> None:
    """RMSNorm of x + residual with codes and scales as output (q35_rms_norm_quant_dev): group
    128 (one scale per 128 elements) or 0 (one per row); residual_out gets x + residual."""
    _lib.check(_lib.load().q35_rms_norm_quant_dev(
        ctx.h, _lib.dtype_code(dtype), x, dim if ldx is None else ldx, residual, dim if ldr is None else ldr,
        residual_out, dim if ldo is None else ldo, weight, eps, rows, dim, _lib.code_of(code), group, q,
        dim if ldq is None else ldq, scales), "q35_rms_norm_quant_dev")


def fp8_gemm(ctx, x: int, x_scales: int, w: int, w_scales: int, y: int, M: int, N: int, K: int,
             dtype: str = "bf16", ldx: int | None = None, ldw: int | None = None, ldy: int | None = None) -> None:
    """y = x w^T in e4m3 with a scale for each block of 128 (q35_fp8_gemm_dev): x [M][K] with
    x_scales [M][ceil(K/128)], w [N][K] with w_scales [ceil(N/128)][ceil(K/128)]; rows of x and
    w start on 16-byte boundaries (pass ldx / ldw, multiples of 16, where K is not one)."""
    _lib.check(_lib.load().q35_fp8_gemm_dev(ctx.h, x, K if ldx is None else ldx, x_scales, w,
                                            K if ldw is None else ldw, w_scales, _lib.dtype_code(dtype), y,
                                            N if ldy is None else ldy, M, N, K), "q35_fp8_gemm_dev")


class KV8CacheStruct(C.Structure):
    _fields_ = [("code", C.c_int32), ("seqs", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("max_seq", C.c_int32), ("block", C.c_int32), ("k", C.c_void_p), ("v", C.c_void_p),
                ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("seq_stride", C.c_int64),
                ("scale_seq_stride", C.c_int64)]


class KV8Cache:
    """A KV cache held in 8 bits with a scale for each block of tokens and head
    (q35_kv8_cache).  The arrays are the caller's device memory: codes k, v
    [seqs][kv_heads][max_seq][head_dim], scales [seqs][kv_heads][ceil(max_seq/block)]; keep
    them alive while the cache is used."""

    def __init__(self, ctx, k: int, v: int, k_scale: int, v_scale: int, seqs: int, kv_heads: int, head_dim: int,
                 max_seq: int, block: int = 64, code: str = "e4m3", seq_stride: int = 0, scale_seq_stride: int = 0):
        self.ctx = ctx
        self.kv_heads, self.head_dim = kv_heads, head_dim
        lib = _lib.load()
        self._append, self._attention = lib.q35_kv8_append_dev, lib.q35_kv8_attention_dev
        self._c = KV8CacheStruct(_lib.code_of(code), seqs, kv_heads, head_dim, max_seq, block, k, v, k_scale, v_scale,
                                 seq_stride, scale_seq_stride)
        self._ref = C.byref(self._c)

    def append(self, k: int, v: int, row_start: int, past: int, rows: int, max_rows: int, dtype: str = "bf16",
               ld: int | None = None) -> None:
        """Rows row_start[s] .. row_start[s+1]-1 of k and v become sequence s's tokens at
        positions past[s] .. (int32 device arrays); rows in all, at most max_rows of one."""
        st = self._append(self.ctx.h, self._ref, _lib.dtype_code(dtype), k, v,
                          self.kv_heads * self.head_dim if ld is None else ld, row_start, past, rows, max_rows)
        if st:
            _lib.check(st, "q35_kv8_append_dev")

    def attention(self, q: int, out: int, heads: int, row_start: int, past: int, rows: int, max_rows: int,
                  scale: float, dtype: str = "bf16", ldq: int | None = None, ldo: int | None = None,
                  workspace: int | None = None, workspace_bytes: int = 0) -> None:
        """Causal attention of the rows' queries over the cache, their own tokens included."""
        width = heads * self.head_dim
        st = self._attention(self.ctx.h, self._ref, _lib.dtype_code(dtype), q, width if ldq is None else ldq, heads, out,
                             width if ldo is None else ldo, row_start, past, rows, max_rows, scale, workspace,
                             workspace_bytes)
        if st:
            _lib.check(st, "q35_kv8_attention_dev")

    def attention_workspace(self, heads: int, rows: int, max_rows: int) -> int:
        """Bytes of device workspace an attention call of this size needs."""
        n = _lib.load().q35_kv8_attention_workspace(self._ref, heads, rows, max_rows)
        if n < 0:
            raise _lib.Q35Error(f"q35_kv8_attention_workspace: {_lib.last_error()}")
        return int(n)
