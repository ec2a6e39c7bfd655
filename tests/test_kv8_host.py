"""Host side of the 8-bit cache's attention: the limits of a call and its workspace, and what the kernels'
source has to keep to (no GPU needed)."""
import ctypes as C
import glob
import os
import re

import pytest

from asicfortranai_b200 import _lib
from asicfortranai_b200.quant8 import KV8CacheStruct

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x1000
INT32_MAX = 2 ** 31 - 1


def cache(kv_heads, head_dim=128, seqs=1, max_seq=1 << 28):
    return C.byref(KV8CacheStruct(0, seqs, kv_heads, head_dim, max_seq, 64, P, P, P, P, 0, 0))


def workspace(c, heads, rows, max_rows):
    return _lib.load().q35_kv8_attention_workspace(c, heads, rows, max_rows)


@pytest.mark.parametrize("heads,kv_heads,rows", [(8, 1, 131072), (64, 8, 131073), (64, 1, 16384), (16, 1, 65537),
                                                 (40, 40, 2048), (32, 32, 64), (8, 1, 512)])
def test_prompts_take_no_workspace(heads, kv_heads, rows):
    """The 128-row form does not split a tile's keys."""
    assert workspace(cache(kv_heads), heads, rows, rows) == 0


def test_few_rows_take_one():
    assert workspace(cache(8), 64, 1, 1) > 0
    assert workspace(cache(1), 8, 100, 100) > 0             # 7 tiles of 128 pairs: split over the SMs


def test_pairs_past_32_bits_are_refused():
    lib = _lib.load()
    ctx = C.create_string_buffer(4096)
    for heads, rows, ok in ((64, INT32_MAX // 64 - 2, True), (64, INT32_MAX // 64 + 1, False), (1 << 20, 1 << 12, False)):
        c = cache(1, 64)
        assert (workspace(c, heads, rows, rows) >= 0) == ok
        if not ok:
            width = heads * 64
            assert lib.q35_kv8_attention_dev(C.addressof(ctx), c, 1, P, width, heads, P, width, P, P, rows, rows, 0.1,
                                             None, 0) == 1
            assert "heads / kv_heads" in _lib.last_error()


def test_kernels_that_start_early_use_no_read_only_loads():
    """A grid launched ahead of the previous one's end lives while that one writes: ld.global.nc and __ldg,
    which want memory that nobody writes meanwhile, are not for its inputs."""
    early = []
    for path in sorted(glob.glob(os.path.join(ROOT, "asicfortranai_b200", "csrc", "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        if "dependency_wait" in text or os.path.basename(path).startswith("q35_kv8"):
            early.append(os.path.basename(path))
            assert not re.search(r"ld\.global\.nc|\b__ldg\b|\b__ldcv?\b", text), path
    assert {"q35_kv8.cu", "q35_kv8.cuh", "q35_kv8_prompt.cu", "q35_norm8.cu", "q35_fp8.cu"} <= set(early)
