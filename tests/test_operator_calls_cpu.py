"""Calls at the edge of what the operators take, as far as they can be checked without a
GPU: what is refused, and which pointers, strides and masks reach the kernels."""

import pytest
import torch

from auspex_soup_demo_b200 import _lib, kernels


# ------------------------------------------------------------- host tensors ----
@pytest.mark.parametrize("call", [
    lambda t: _lib.stream_of(t),
    lambda t: kernels.fast_swiglu(t, t),
    lambda t: kernels.fast_rms_norm(t, t[0], 1e-6),
], ids=["stream_of", "fast_swiglu", "fast_rms_norm"])
def test_host_tensors_are_refused_before_a_launch(call):
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        call(torch.zeros(4, 8))
