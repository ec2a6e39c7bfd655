"""What the source of the 8-bit cache's kernels has to keep to (no GPU needed)."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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
