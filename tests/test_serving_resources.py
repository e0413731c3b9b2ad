"""The kernels for the choice of experts, 4-bit weights and adjusted logits keep their values in registers."""
import re

from test_kernel_resources import kernels  # noqa: F401

NAMES = r"q4_few_kernel|q4_dx_kernel|q4_tile_kernel|quant_i4_kernel|pack_i4_kernel|dequant_i4_kernel|route_experts_kernel|route_backward_kernel|logits_kernel"


def test_no_spills(kernels):  # noqa: F811
    """No stack; the choice among 32 experts a lane (33 groups and more) moves one value to an accumulation register and back."""
    found = {}
    for n, k in kernels.items():
        m = re.search(NAMES, n)
        if m is None:
            continue
        found.setdefault(m.group(), []).append(n)
        wide = m.group() == "route_experts_kernel" and re.search(r"64, 32, true|Li64ELi32ELb1E", n)
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] <= (1 if wide else 0), (n, k[".vgpr_count"])
    assert len(found) == 9, sorted(found)
