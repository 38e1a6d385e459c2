"""The scale of tree_attention, on the CPU: the kernels work with scale x log2(e) in 32 bits."""

from __future__ import annotations

import pytest

from kernelcode_generate_amd import native
from tests.test_serving_refusals import refused, tree_args


@pytest.mark.parametrize("scale,text", [(2.3e38, "not a device pointer"), (2.4e38, "scale must be finite"), (-2.4e38, "scale must be finite"),
                                        (3.4e38, "scale must be finite"), (0.0, "not a device pointer"), (-1e-300, "not a device pointer"),
                                        (float("inf"), "scale must be finite")])
def test_scales(scale, text):
    refused("tree", tree_args, -1, text, scale=scale)
    assert native.last_error()
