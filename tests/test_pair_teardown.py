"""CPU check of how kernels of CTA pairs end: a CTA that left its SM before its partner had released the
pair's TMEM could make room for another kernel's CTA, which allocates TMEM there."""
import re

from conftest import PKG

CSRC = sorted((PKG / "csrc").glob("*.cu*"))


def test_every_pair_kernel_ends_with_both_ctas_released():
    users = []
    for path in CSRC:
        code = re.sub(r"//[^\n]*", "", path.read_text())
        if path.name == "moe_common.cuh":
            body = re.search(r"void pair_teardown\([^)]*\) \{(.*?)\n\}", code, re.S).group(1)
            steps = re.findall(r"cluster_sync|tmem_dealloc_pair|__syncthreads", body)
            assert steps == ["__syncthreads", "cluster_sync", "tmem_dealloc_pair", "cluster_sync"]
            continue
        assert "tmem_dealloc_pair" not in code, path.name
        assert code.count("tmem_alloc_pair(") == code.count("pair_teardown("), path.name
        if "tmem_alloc_pair(" in code:
            users.append(path.stem)
    assert users == ["fp8_gemm", "grouped_gemm", "grouped_wgrad", "router_gemm"]
