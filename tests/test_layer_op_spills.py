"""Kernels of the layer operators that keep a part of their registers in memory: which, and at most how many bytes a lane.  All
others keep none.  They are the head dimensions above 64 at rows that are not whole 16-byte pieces, the sinks' launch of the
attention's backward at those dimensions, float32 at 128 keys a workgroup, and the norm's backward beyond 8192 float32
elements."""
import re

from test_kernel_resources import kernels  # noqa: F401

# what the built library holds, by kernel (mangled names: DF16b bfloat16, DF16_ float16, f float32; b1 / b0 whole 16-byte rows)
MOST = {
    "bk_attn_dq_kernelIDF16bLi128ELb0ELi2E": 16, "bk_attn_dq_kernelIDF16_Li128ELb0ELi2E": 24,
    "bk_attn_dkv_kernelIDF16bLi128ELb0ELb0ELi2E": 24, "bk_attn_dkv_kernelIDF16_Li128ELb0ELb0ELi2E": 164,
    "bk_attn_dkv_kernelIDF16bLi128ELb0ELb1ELi1E": 180, "bk_attn_dkv_kernelIDF16_Li128ELb0ELb1ELi1E": 204,
    "bk_attn_dkv_kernelIDF16bLi128ELb0ELb1ELi2E": 60, "bk_attn_dkv_kernelIDF16_Li128ELb0ELb1ELi2E": 104,
    "bk_attn_dkv_kernelIDF16bLi128ELb1ELb1ELi1E": 8, "bk_attn_dkv_kernelIDF16_Li128ELb1ELb1ELi1E": 8,
    "bk_attn_dkv_kernelIfLi128ELb0ELb0ELi2E": 28, "bk_attn_dkv_kernelIfLi128ELb1ELb0ELi2E": 8,
    "bk_attn_dkv_kernelIfLi128ELb0ELb1ELi2E": 456, "bk_attn_dkv_kernelIfLi128ELb1ELb1ELi2E": 292,
    "bk_layer_norm_backward_kernelIfLi512ELi32ELb0E": 164, "bk_layer_norm_backward_kernelIfLi512ELi32ELb1E": 88,
}


def test_no_kernel_keeps_more_in_memory_than_listed(kernels):  # noqa: F811
    mine = {k: r["private_segment_fixed_size"] for k, r in kernels.items()
            if re.search(r"bk_(attn|layer_norm_(kernel|backward)|scan_(kernel|adjoint|backward|step|sum)|conv|sum_parts)", k)}
    assert len(mine) > 150
    for name in MOST:
        assert sum(name in k for k in mine) == 1, name
    for k, size in mine.items():
        most = next((m for name, m in MOST.items() if name in k), 0)
        assert size <= most, (k, size, most)
