"""Calls of the block operators at the edge of what they take, on the GPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import block_ops_oracle as oracle
import test_block_ops_edges as cpu
from ditserve_b200 import ops

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


def _dev():
    return torch.device("cuda", 0)


def _randn(*shape, seed=0, dtype=FL, std=1.0):
    g = torch.Generator(device=_dev()).manual_seed(seed)
    return (torch.randn(*shape, device=_dev(), generator=g) * std).to(dtype)


@pytest.mark.parametrize("case", range(4))
def test_rms_norm_quant_outputs_share_no_memory(case):
    with pytest.raises(ValueError):
        cpu.scale_on_other_outputs(_dev())[0][case]()


def test_rms_norm_quant_scale_beside_the_codes():
    x = _randn(8, 64, dtype=BF)
    oracle.check_norm_quant(cpu.scale_on_other_outputs(_dev())[1](x), x, None, None, 1e-6)
