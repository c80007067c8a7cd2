"""Registers of the layer operators' hot kernels, read from the code objects inside libbkcore.so (no GPU needed).  A spilled
register in their loops costs more than its own access: its reload waits for the rows under way (dk, dv of the attention
450 -> 525 us for 52 bytes, the scan's backward 158 -> 313 us for 292)."""
from test_kernel_resources import _find, kernels  # noqa: F401


def test_hot_loops_do_not_spill(kernels):  # noqa: F811
    names = ["bk_scan_kernel", "bk_scan_adjoint_agg_kernel", "bk_scan_backward_kernel", "bk_scan_step_kernel", "bk_conv_kernel",
             "bk_conv_step_kernel", "bk_layer_norm_kernel", "bk_attn_kernelIDF16", "bk_attn_step_kernel"]
    for name in names:
        for k in _find(kernels, name):
            assert kernels[k]["private_segment_fixed_size"] == 0, (k, kernels[k])
    # the backward at whole 16-byte rows, apart from the sinks' own launch
    for name, variant in (("bk_attn_dq_kernelIDF16", "ELb1ELi"), ("bk_attn_dkv_kernelIDF16", "ELb1ELb0ELi")):
        for k in _find(kernels, name, variant):
            assert kernels[k]["private_segment_fixed_size"] == 0, (k, kernels[k])


def test_two_workgroups_a_compute_unit(kernels):  # noqa: F811
    for name in ("bk_attn_kernel", "bk_attn_dq_kernel", "bk_scan_backward_kernel"):
        for k in _find(kernels, name):
            assert 2 * kernels[k]["group_segment_fixed_size"] <= 160 * 1024, (k, kernels[k])
