"""Every kernel at the token end of a step waits for the launches in front of it before it reads what they wrote."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashoptim_jax_b200", "csrc")


@pytest.mark.parametrize("source", ["fo_dropout.cu", "fo_embed.cu", "fo_embed_grad.cu"])
def test_kernels_wait_first(source):
    """A launch that may start early sees the writes of earlier ones only behind its own griddepcontrol.wait."""
    with open(os.path.join(CSRC, source)) as f:
        text = f.read()
    kernels = re.findall(r"__global__ void[^;{]*?(\w+_kernel)\([^{;]*\) \{\s*(\w+)\(", text)
    assert len(kernels) == text.count("__global__ void")
    assert {name: first for name, first in kernels if first != "chain_wait"} == {}
