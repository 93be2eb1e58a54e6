"""Calls of the block operators at the edge of what they take, on the CPU: outputs on other tensors, values that
leave a type's range."""
import math

import pytest
import torch

import block_ops_oracle as oracle
from ditserve_b200 import ops
from ditserve_b200.ops._memory import shares_memory

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


def test_shares_memory_against_the_bytes():
    """Every pair of views of one buffer against the bytes that they touch; a general layout may only be refused."""
    buf = torch.zeros(96, dtype=torch.uint8)
    views = [buf, buf[:16], buf[16:], buf[8:24].view(FL), buf.view(6, 16)[:, :8], buf.view(6, 16)[:, 8:],
             buf.view(6, 16)[:, 12:].view(FL), buf.view(6, 16)[2:, 4:12], buf.view(6, 16)[1:3], buf.view(2, 3, 16)[..., 4:8],
             buf.view(6, 16)[::2, :8], buf.view(6, 16)[1::2], buf[4:84].view(5, 16)[:, 8:], buf[95:], buf[:0],
             buf.view(FL).view(6, 4)[:, 3], buf.view(FL)[3::4][:2], buf[:1].expand(7)]
    exact = list(range(len(views)))

    def touched(v):
        mark = torch.zeros(96, dtype=torch.bool)
        at = torch.zeros(v.shape, dtype=torch.int64) + v.data_ptr() - buf.data_ptr()
        for i, (n, st) in enumerate(zip(v.shape, v.stride())):
            at = at + (torch.arange(n) * st * v.element_size()).reshape([-1 if j == i else 1 for j in range(v.dim())])
        for e in range(v.element_size()):
            mark[(at + e).flatten()] = True
        return mark
    for i in exact:
        for j in exact:
            meet = bool((touched(views[i]) & touched(views[j])).any())
            got = shares_memory(views[i], views[j])
            assert got or not meet, (i, j)
    # the layouts that calls use: exactly
    for i in (1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 13, 14, 15):
        for j in (1, 2, 4, 5, 6, 9, 13, 14, 15):
            assert shares_memory(views[i], views[j]) == bool((touched(views[i]) & touched(views[j])).any()), (i, j)


def scale_on_other_outputs(dev):
    """rms_norm_quant calls whose outputs share bytes, and one whose outputs are columns of one buffer."""
    x = torch.ones(8, 64, dtype=BF, device=dev)
    codes = torch.zeros(8, 64, dtype=torch.uint8, device=dev)
    h = torch.zeros(8, 64, dtype=BF, device=dev)
    refused = [lambda: ops.rms_norm_quant(x, out=codes.view(E4M3), scale_out=codes.view(-1)[:32].view(FL)),
               lambda: ops.rms_norm_quant(x, out=codes.view(E4M3), scale_out=codes.view(FL)[:, 3]),
               lambda: ops.rms_norm_quant(x, residual=x, residual_out=h, scale_out=h.view(-1)[:16].view(FL)),
               lambda: ops.rms_norm_quant(x, residual=x, residual_out=h, out=h.view(E4M3)[:, 64:])]
    rows = torch.zeros(8, 80, dtype=torch.uint8, device=dev)  # a row's codes, then its scale
    return refused, lambda v: ops.rms_norm_quant(v, out=rows[:, :64].view(E4M3), scale_out=rows.view(FL)[:, 16])


@pytest.mark.parametrize("case", range(4))
def test_rms_norm_quant_outputs_share_no_memory(case):
    with pytest.raises(ValueError):
        scale_on_other_outputs("cpu")[0][case]()


def test_rms_norm_quant_scale_beside_the_codes():
    x = torch.randn(8, 64).to(BF)
    oracle.check_norm_quant(scale_on_other_outputs("cpu")[1](x), x, None, None, 1e-6)
