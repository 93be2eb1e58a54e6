"""Calls of the block operators at the edge of what they take, on the GPU."""
import math
import os
import subprocess
import sys

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


# ---- linear_fp8 -------------------------------------------------------------------------------
def gelu_cases(m, dtype):
    """Every row and column of the product is one pre-activation, exactly: 1 * 1 * its channel's scale."""
    t = torch.cat([torch.linspace(-12, 12, 8193), torch.linspace(-40, 40, 801),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4, 6e4, -6e4])]).to(_dev())
    one = torch.zeros(m, 64, device=_dev())
    one[:, 0] = 1
    each = torch.zeros(t.numel(), 64, device=_dev())
    each[:, 0] = 1
    return t, ops.linear_fp8(one.to(E4M3), torch.ones(m, device=_dev()), each.to(E4M3), t, act="gelu", out_dtype=dtype)


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("m", [1, 12, 100, 300])
def test_linear_fp8_gelu_keeps_its_tail(m, dtype):
    """x / (1 + exp(-a)), a = 2 sqrt(2/pi) (x + 0.044715 x^3), in the few-row form and in single and paired tiles.

    With w = 2^-24 an fp32 rounding: the exponent takes 7 roundings, which the power turns into 7 |a| w of itself; the
    power and the quotient err by 2^-22 each, the sum by w: (7 |a| + 9) w of the value.
    Then the output's rounding, half a step of the smallest number in fp16, and what a power below 2^-126 leaves."""
    t, y = gelu_cases(m, dtype)
    ops.check_status(_dev())
    x, w = t.double(), 2.0 ** -24
    a = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    want = x / (1 + torch.exp(-a))
    bound = want.abs() * ((7 * a.abs() + 9) * w + oracle.u(dtype) * 1.001) + (1 + x.abs()) * 2.0 ** -126
    if dtype == HF:
        bound = bound + 2.0 ** -25
    d = (y.double() - want).abs()
    assert (d <= bound).all(), (d / bound).max()


# ---- cross_attention --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq", [3, 520])  # few-row form, tiles
def test_cross_attention_nan_rows(sq, d, dtype):
    q, k, v, lens, mask = cpu.nan_inputs(_dev(), sq, d, dtype)
    want = ops.cross_attention_reference(q, k, v, 24, kv_lens=lens, key_mask=mask, return_lse=True)
    got = ops.cross_attention(q, k, v, 24, kv_lens=lens, key_mask=mask, return_lse=True)
    ops.check_status(_dev())
    cpu.check_nan(*got, *want, sq, d)


@pytest.mark.parametrize("sq", [3, 520])
def test_cross_attention_scales_out_of_range(sq):
    """Refused, in both forms; the smallest scale is a plain mean over the keys that are left."""
    q, k, v = (_randn(2, n, 24 * 64, seed=s, dtype=BF) for n, s in ((sq, 1), (300, 2), (300, 3)))
    lens = torch.tensor([270, 131], device=_dev(), dtype=torch.int32)
    before = ops.launch_counts()
    for scale in cpu.BAD_SCALES:
        with pytest.raises(ValueError):
            ops.cross_attention(q, k, v, 24, kv_lens=lens, scale=scale)
            pytest.fail(f"{scale} was not refused")
    assert ops.launch_counts() == before
    o, lse = ops.cross_attention(q, k, v, 24, kv_lens=lens, scale=2e-45, return_lse=True)
    ops.check_status(_dev())
    oracle.check_cross(o, lse, q, k, v, 24, allowed=torch.arange(300, device=_dev()) < lens[:, None], scale=2e-45)


@pytest.mark.parametrize("sq", [3, 520])
def test_cross_attention_rows_that_overlap(sq):
    """Sliding windows over one buffer: rows 8 elements apart, read in place by loads and by tiles."""
    flat = _randn(24 * 64 + 8 * 600, seed=5, dtype=BF)
    q, k, v = (flat[o:].as_strided((2, n, 24 * 64), (16, 8, 1)) for o, n in ((0, sq), (8, 300), (32, 300)))
    want = ops.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), 24)
    assert torch.equal(ops.cross_attention(q, k, v, 24), want)
    ops.check_status(_dev())


# ---- graphs -----------------------------------------------------------------------------------
_FIRST_CALL_IN_A_CAPTURE = """
import torch
from ditserve_b200 import ops
dev = torch.device("cuda", 0)
q, k = torch.randn(1, 300, 1536, device=dev).bfloat16(), torch.randn(1, 200, 1536, device=dev).bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.cross_attention(q, k, k, 24)
ops.check_status(dev)                  # clear before any replay
graph.replay()
assert torch.equal(out, ops.cross_attention(q, k, k, 24))
word = ops.status_word(dev)
word.fill_(1)                          # as a launch that gave up leaves it
graph.replay()
try:
    ops.check_status(dev)
except ops.KernelTimeout:
    print("kept")
ops.check_status(dev)                  # the report was taken
del graph, out
torch.cuda.empty_cache()
ops.check_status(dev)
"""


def test_status_word_made_in_a_capture_outlives_replays():
    """The first call of a process inside a capture: no replay clears what another launch reported."""
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL_IN_A_CAPTURE], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout.strip() == "kept", r.stdout + r.stderr


# ---- outputs on other tensors -----------------------------------------------------------------
@pytest.mark.parametrize("case", range(4))
def test_overlap_is_told_by_addresses(case):
    with pytest.raises(ValueError):
        cpu.outputs_through_another_storage(_dev())[case]()


def test_in_place_through_another_storage():
    x, r = _randn(8, 64, dtype=BF), _randn(8, 64, seed=1, dtype=BF)
    want = r.clone()
    got = ops.rms_norm_quant(x, residual=r, residual_out=cpu.other_storage(r))
    oracle.check_norm_quant((got[0], got[1], r), x, None, want, 1e-6)


@pytest.mark.parametrize("case", range(7))
def test_linear_fp8_out_on_parameters(case):
    with pytest.raises(ValueError):
        cpu.linear_outputs_on_parameters(_dev())[0][case]()


def test_linear_fp8_parameters_beside_out():
    cpu.linear_outputs_on_parameters(_dev())[1]()
    ops.check_status(_dev())


@pytest.mark.parametrize("case", range(3))
def test_rms_norm_quant_outputs_on_weight(case):
    with pytest.raises(ValueError):
        cpu.norm_outputs_on_weight(_dev())[0][case]()


@pytest.mark.parametrize("case", range(2))
def test_rms_norm_quant_weight_near_outputs(case):
    cpu.norm_outputs_on_weight(_dev())[1][case]()


@pytest.mark.parametrize("case", range(3))
def test_rope_axes_outputs_on_positions(case):
    with pytest.raises(ValueError):
        cpu.rope_outputs_on_positions(_dev())[0][case]()


def test_rope_axes_positions_beside_out():
    cpu.rope_outputs_on_positions(_dev())[1]()


@pytest.mark.parametrize("case", range(3))
def test_cross_attention_out_on_masks(case):
    with pytest.raises(ValueError):
        cpu.cross_outputs_on_masks(_dev(), 4)[0][case]()


@pytest.mark.parametrize("sq", [4, 300])
def test_cross_attention_masks_beside_out(sq):
    cpu.cross_outputs_on_masks(_dev(), sq)[1]()
    ops.check_status(_dev())


@pytest.mark.parametrize("sq", [4, 300])
@pytest.mark.parametrize("case", range(5))
def test_cross_attention_out_entries_apart(case, sq):
    refused, taken, call = cpu.cross_out_layouts(_dev(), sq)
    with pytest.raises(ValueError):
        call(refused[case])
    call(taken[case])
    ops.check_status(_dev())


def test_cross_attention_tiles_between_rows():
    """[S, B, width] buffers: entries between one another's rows, through tile loads and stores."""
    q, k, v = (_randn(n, 3, 24 * 64 + 8, seed=s, dtype=BF)[..., 8:].transpose(0, 1) for n, s in ((520, 1), (300, 2), (300, 3)))
    out = torch.full((521, 3, 24 * 64 + 8), 7.0, device=_dev(), dtype=BF)
    ops.cross_attention(q, k, v, 24, out=out[:520, :, :24 * 64].transpose(0, 1))
    ops.check_status(_dev())
    want = ops.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), 24)
    assert torch.equal(out[:520, :, :24 * 64].transpose(0, 1), want)
    assert (out[520] == 7).all() and (out[..., 24 * 64:] == 7).all()


# ---- errors -----------------------------------------------------------------------------------
def test_out_of_memory_is_torchs_error():
    """An allocation beyond the allocator's limit (a limit of this process, not the device's end): torch's own class."""
    x = torch.zeros(1, 64, device=_dev(), dtype=BF).expand(1 << 22, 64)  # 256 MB of codes
    xq, xs = ops.quantize_rows_fp8(torch.zeros(16, 64, device=_dev()))
    wq, ws = ops.empty_fp8(1 << 22, 64, _dev()), torch.ones(1 << 22, device=_dev())
    q = torch.zeros(1, 1, 128, device=_dev(), dtype=BF).expand(1, 1 << 20, 128)
    calls = [lambda: ops.rms_norm_quant(x), lambda: ops.linear_fp8(xq, xs, wq, ws),
             lambda: ops.rope_axes(x, torch.zeros(1, 1, device=_dev()), (64,), head_dim=64),
             lambda: ops.cross_attention(q, q[:, :3], q[:, :3], 2)]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (32 << 20)) /
                                                   torch.cuda.get_device_properties(0).total_memory)
        for call in calls:
            with pytest.raises(torch.cuda.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert ops.rms_norm_quant(x[:4])[0].shape == (4, 64)
    with pytest.raises(TypeError):
        ops._ext.launch("rms_norm_quant", 1, None, None, 1e-6, None, None, None)


@pytest.mark.parametrize("m,n,k", [(17, 2, (1 << 28) + 16), ((1 << 30) + 1, 1, 1), (1, (1 << 30) + 1, 1)])
def test_linear_fp8_refuses_sizes(m, n, k):
    cpu.test_linear_fp8_refuses_sizes(m, n, k, _dev())
