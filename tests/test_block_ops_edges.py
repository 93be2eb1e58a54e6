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
             buf.view(FL).view(6, 4)[:, 3], buf.view(FL)[3::4][:2], buf[:1].expand(7),
             buf.view(2, 3, 16)[:, :2, :8], buf.view(2, 3, 16)[:, 1:, 8:], buf.view(2, 3, 16)[:, 2, 4:8]]
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
    for i in (1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 13, 14, 15, 18, 19):
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


def nan_inputs(dev, sq, d, dtype):
    """q, k, v of two entries with 24 heads, 300 keys, lengths and a mask; a NaN query in entry 0, a NaN key that is
    left out in entry 0 and one that is not in head 5 of entry 1."""
    g = torch.Generator().manual_seed(sq)
    q, k, v = (torch.randn(2, n, 24 * d, generator=g).to(dtype) for n in (sq, 300, 300))
    q[0, sq // 2, 3 * d + 1] = math.nan
    k[0, 280] = math.nan
    k[1, 130, 5 * d:6 * d] = math.nan
    mask = torch.ones(2, 300, dtype=torch.bool)
    mask[:, 5:9] = False
    return (*(t.to(dev) for t in (q, k, v)), torch.tensor([270, 200], device=dev, dtype=torch.int32), mask.to(dev))


def check_nan(o, lse, o_want, lse_want, sq, d):
    """NaN exactly where a query, or a key that it may attend to, is NaN: outputs and log sums, in that head alone."""
    nan = torch.zeros(2, 24, sq, dtype=torch.bool)
    nan[0, 3, sq // 2] = True
    nan[1, 5] = True
    assert torch.equal(lse_want.isnan().cpu(), nan) and torch.equal(lse.isnan().cpu(), nan)
    rows = nan.transpose(1, 2)[..., None].expand(2, sq, 24, d).reshape(2, sq, 24 * d)
    assert torch.equal(o_want.isnan().cpu(), rows) and torch.equal(o.isnan().cpu(), rows)
    assert not lse.isinf().any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_cross_attention_nan_rows(dtype):
    q, k, v, lens, mask = nan_inputs("cpu", 3, 64, dtype)
    got = ops.cross_attention(q, k, v, 24, kv_lens=lens, key_mask=mask, return_lse=True)
    check_nan(*got, *got, 3, 64)


BAD_SCALES = [0.0, -0.5, 1e-50, 1e-45, 3e38, 1e39, math.inf, math.nan]


@pytest.mark.parametrize("scale", BAD_SCALES)
def test_cross_attention_scales_out_of_range(scale):
    q = torch.ones(1, 2, 64, dtype=BF)
    with pytest.raises(ValueError):
        ops.cross_attention(q, q, q, 1, scale=scale)


def test_cross_attention_smallest_scale():
    q, k, v = (torch.randn(2, n, 128).to(BF) for n in (3, 20, 20))
    lens = torch.tensor([20, 7], dtype=torch.int32)
    o, lse = ops.cross_attention(q, k, v, 2, kv_lens=lens, scale=2e-45, return_lse=True)
    oracle.check_cross(o, lse, q, k, v, 2, allowed=torch.arange(20) < lens[:, None], scale=2e-45)


def other_storage(t):
    """The same memory as a storage of its own."""
    got = torch.from_dlpack(t)
    assert got.data_ptr() == t.data_ptr() and not torch._C._is_alias_of(got, t)
    return got


def outputs_through_another_storage(dev):
    """Calls whose output lies on an operand's rows, but for one: known by address alone."""
    x, wide = torch.ones(4, 64, dtype=BF, device=dev), torch.ones(6, 64, dtype=BF, device=dev)
    pos = torch.arange(4, device=dev)
    xq, xs = ops.quantize_rows_fp8(torch.ones(4, 64, device=dev))
    wq, ws = ops.quantize_rows_fp8(torch.ones(32, 64, device=dev))
    r = torch.ones(6, 32, dtype=BF, device=dev)
    q = torch.ones(1, 6, 64, dtype=BF, device=dev)
    return [lambda: ops.rms_norm_quant(x, residual=wide[:4], residual_out=other_storage(wide[1:])[:4]),
            lambda: ops.linear_fp8(xq, xs, wq, ws, residual=r[:4], out=other_storage(r[1:])[:4]),
            lambda: ops.rope_axes(wide[:4], pos, (64,), head_dim=64, out=other_storage(wide[1:])[:4]),
            lambda: ops.cross_attention(q[:, :4], x[None], x[None], 1, out=other_storage(q[:, 1:])[:, :4])]


def test_overlap_is_told_by_addresses():
    from ditserve_b200.ops.cross import _shares_memory
    from ditserve_b200.ops.fp8 import _partial_overlap
    buf = torch.zeros(8, 96)
    for view in (buf[1:], buf[:, 16:48], buf.view(-1)[8:200]):
        far = other_storage(view)
        assert shares_memory(far, buf[:, :32]) and _shares_memory(far, buf[:, :32])
        assert not _partial_overlap(far, view) and not _partial_overlap(view, far)
    assert _partial_overlap(other_storage(buf[1:])[:, :32], buf[:-1, :32])
    assert not _partial_overlap(other_storage(buf)[:, :32], buf[:, 32:])
    with pytest.raises(ValueError):
        outputs_through_another_storage("cpu")[3]()


def linear_outputs_on_parameters(dev):
    """(calls whose out lies on a scale, the bias, the gate or row_batch; one whose parameters lie beside out's rows)"""
    xq, xs = ops.quantize_rows_fp8(torch.randn(32, 64).to(dev))
    wq, ws = ops.quantize_rows_fp8(torch.randn(32, 64).to(dev))
    o, r = torch.zeros(40, 32, device=dev), torch.zeros(32, 32, device=dev)
    one = torch.ones(2, 32, device=dev)
    refused = [lambda: ops.linear_fp8(xq, o.view(-1)[:32], wq, ws, out=o[:32]),
               lambda: ops.linear_fp8(xq, o[:32, 5], wq, ws, out=o[:32]),
               lambda: ops.linear_fp8(xq, xs, wq, o[31], out=o[:32]),
               lambda: ops.linear_fp8(xq, xs, wq, ws, o[7], out=o[:32]),
               lambda: ops.linear_fp8(xq, xs, wq, ws, residual=r, gate=o[31:33], rows_per_batch=16, out=o[:32]),
               lambda: ops.linear_fp8(xq, xs, wq, ws, residual=r, gate=o[31], out=o[:32]),
               lambda: ops.linear_fp8(xq, xs, wq, ws, residual=r, gate=one, row_batch=o[3].view(torch.int32), out=o[:32])]
    wide = torch.randn(40, 160).to(dev)
    wide[:32, 64] = xs
    wide[1, 64:96] = ws
    keep = wide.clone()

    def beside():
        """out in the first columns; residual, scale, bias and gate in others of the same rows."""
        got = ops.linear_fp8(xq, wide[:32, 64], wq, ws, wide[2, 96:128], residual=wide[:32, 32:64], gate=wide[3:5, 128:],
                             rows_per_batch=16, out=wide[:32, :32])
        assert torch.equal(wide[:, 32:], keep[:, 32:]) and torch.equal(wide[32:], keep[32:])
        gate = keep[3:5, 128:].repeat_interleave(16, 0)
        oracle.check_linear(got, *oracle.linear(xq, keep[:32, 64], wq, ws, keep[2, 96:128], residual=keep[:32, 32:64],
                                                gate_rows=gate))
    return refused, beside


@pytest.mark.parametrize("case", range(7))
def test_linear_fp8_out_on_parameters(case):
    with pytest.raises(ValueError):
        linear_outputs_on_parameters("cpu")[0][case]()


def test_linear_fp8_parameters_beside_out():
    linear_outputs_on_parameters("cpu")[1]()


def norm_outputs_on_weight(dev):
    """(calls whose out or residual_out lies on the weight; calls that are right: a scale on the weight, which is
    written last, and a weight beside the rows of residual_out)"""
    x, r = torch.randn(8, 64).to(dev, BF), torch.randn(8, 64).to(dev, BF)
    buf = torch.ones(10, 64, dtype=BF, device=dev)
    codes = torch.zeros(10, 128, dtype=torch.uint8, device=dev)
    codes.view(BF).fill_(1.0)
    refused = [lambda: ops.rms_norm_quant(x, buf[3], residual=r, residual_out=buf[:8]),
               lambda: ops.rms_norm_quant(x, buf[7], residual=r, residual_out=buf[:8]),
               lambda: ops.rms_norm_quant(x, codes.view(BF)[2], out=codes.view(E4M3)[:8, 64:])]

    def scale_on_weight():
        w = (1 + 0.2 * torch.randn(64)).to(dev, BF)
        before = w.clone()
        oracle.check_norm_quant(ops.rms_norm_quant(x, w, scale_out=w[16:32].view(FL)), x, before, None, 1e-6)

    def beside():
        wide = torch.randn(8, 136).to(dev, BF)
        w = wide[2, 72:]
        oracle.check_norm_quant(ops.rms_norm_quant(x, w, residual=r, residual_out=wide[:, :64]), x, w, r, 1e-6)
    return refused, (scale_on_weight, beside)


@pytest.mark.parametrize("case", range(3))
def test_rms_norm_quant_outputs_on_weight(case):
    with pytest.raises(ValueError):
        norm_outputs_on_weight("cpu")[0][case]()


@pytest.mark.parametrize("case", range(2))
def test_rms_norm_quant_weight_near_outputs(case):
    norm_outputs_on_weight("cpu")[1][case]()


def rope_outputs_on_positions(dev):
    """(calls whose outputs lie on the positions; positions in columns beside the rows of out)"""
    pos = torch.zeros(8, 64, dtype=torch.int64, device=dev)
    x = torch.randn(8, 128).to(dev)
    refused = [lambda: ops.rope_axes(x, pos[3, :8], (64,), out=pos.view(FL)),
               lambda: ops.rope_axes(x, pos[:, :3], (44, 42, 42), out=pos.view(FL)),
               lambda: ops.rope_axes(x, pos.t()[:8, :3], (44, 42, 42), k=x, k_out=pos.view(FL))]

    def beside():
        wide = torch.zeros(8, 136, device=dev)
        p = wide[:, 130:133]
        p.copy_(torch.arange(24).view(8, 3))
        want = p.clone()
        oracle.check_rope(ops.rope_axes(x, p, (44, 42, 42), out=wide[:, :128]), x, want, (44, 42, 42), 128, (1e4,) * 3)
        assert torch.equal(p, want)
    return refused, beside


@pytest.mark.parametrize("case", range(3))
def test_rope_axes_outputs_on_positions(case):
    with pytest.raises(ValueError):
        rope_outputs_on_positions("cpu")[0][case]()


def test_rope_axes_positions_beside_out():
    rope_outputs_on_positions("cpu")[1]()


def test_rope_axes_out_on_k():
    """On the CPU x' may go where k was: k' is of the k that came in.  x' and k' in one place are refused."""
    x, k = torch.randn(6, 64), torch.randn(6, 64)
    pos, was = torch.arange(6), k.clone()
    y, ky = ops.rope_axes(x, pos, (64,), k=k, head_dim=64, out=k)
    assert y is k
    oracle.check_rope(y, x, pos[:, None], (64,), 64, (1e4,))
    oracle.check_rope(ky, was, pos[:, None], (64,), 64, (1e4,))
    o = torch.zeros(7, 64)
    for a, b in ((o[:6], o[:6]), (o[:6], o[1:])):
        with pytest.raises(ValueError):
            ops.rope_axes(x, pos, (64,), k=was, head_dim=64, out=a, k_out=b)


def cross_outputs_on_masks(dev, sq):
    """(calls whose out lies on the lengths or the mask; lengths and mask in columns beside out's rows)"""
    q, k = torch.randn(2, sq, 128).to(dev, BF), torch.randn(2, 9, 128).to(dev, BF)
    out = torch.zeros(2, sq, 128, dtype=BF, device=dev)
    flat = out.view(-1)
    refused = [lambda: ops.cross_attention(q, k, k, 2, kv_lens=flat.view(torch.int32)[:2], out=out),
               lambda: ops.cross_attention(q, k, k, 2, kv_lens=flat[-8:].view(torch.int64), out=out),
               lambda: ops.cross_attention(q, k, k, 2, key_mask=flat.view(torch.bool)[64:82].view(2, 9), out=out)]

    def beside():
        wide = torch.zeros(2, sq, 160, dtype=BF, device=dev)
        lens = wide[:, 0, 128:130].view(torch.int32)[:, 0]
        lens.copy_(torch.tensor([9, 4]))
        mask = wide[:, 0, 132:141].view(torch.bool)[:, :9]
        mask.copy_(torch.tensor([[1, 1, 0, 1, 0, 1, 1, 1, 1], [0, 1, 1, 1, 1, 1, 1, 1, 1]]).bool())
        allowed = mask & (torch.arange(9, device=dev) < lens[:, None])
        keep = wide.clone()
        o = ops.cross_attention(q, k, k, 2, kv_lens=lens, key_mask=mask, out=wide[..., :128])
        oracle.check_cross(o, None, q, k, k, 2, allowed=allowed)
        assert torch.equal(wide[..., 128:], keep[..., 128:])
    return refused, beside


@pytest.mark.parametrize("case", range(3))
def test_cross_attention_out_on_masks(case):
    with pytest.raises(ValueError):
        cross_outputs_on_masks("cpu", 4)[0][case]()


def test_cross_attention_masks_beside_out():
    cross_outputs_on_masks("cpu", 4)[1]()


def cross_out_layouts(dev, sq):
    """(strides of out whose entries or rows meet; strides whose do not: entries behind or between one another)"""
    q, k = torch.randn(3, sq, 128).to(dev, BF), torch.randn(3, 9, 128).to(dev, BF)
    flat = torch.full((3 * 2 * sq * 256,), 7.0, dtype=BF, device=dev)

    def call(strides):
        out = flat.as_strided((3, sq, 128), (*strides, 1))
        o = ops.cross_attention(q, k, k, 2, out=out)
        oracle.check_cross(o, None, q, k, k, 2)
        mark = torch.zeros_like(flat, dtype=torch.bool)
        mark.as_strided((3, sq, 128), (*strides, 1)).fill_(True)
        assert (flat[~mark] == 7).all()
    refused = [(128, 128), (128 * (sq - 1), 128), (256, 128), (128, 256), (0, 128)]
    taken = [(128 * sq, 128), (256 * sq + 8, 256), (128, 3 * 128), (136, 3 * 136), (256, 3 * 256 - 128)]
    return refused, taken, call


@pytest.mark.parametrize("case", range(5))
def test_cross_attention_out_entries_apart(case):
    refused, taken, call = cross_out_layouts("cpu", 4)
    with pytest.raises(ValueError):
        call(refused[case])
    call(taken[case])


def test_timer_records_launches_alone(monkeypatch):
    """An entry that returns None launched nothing: no record and no count, whatever is timed."""
    from ditserve_b200.ops import _ext

    class Event:
        def __init__(self, enable_timing):
            pass

        def record(self):
            pass
    monkeypatch.setattr(torch.cuda, "Event", Event)
    answers = iter([None, "out"])
    fake = type("Ext", (), {"op": staticmethod(lambda *a: next(answers)), "other": staticmethod(lambda: None)})
    monkeypatch.setattr(_ext, "_ext", fake)
    monkeypatch.setattr(_ext, "_launches", {})
    with ops.KernelTimer() as timer:
        assert _ext.launch("op", 1) is None and _ext.launch("op", 1) == "out"
        assert _ext.kernel("other")() is None  # entries that return nothing always launch
    assert [r[0] for r in timer.records] == ["op", "other"] and ops.launch_counts() == {"op": 1, "other": 1}


@pytest.mark.parametrize("m,n,k", [(17, 2, (1 << 28) + 16), ((1 << 30) + 1, 1, 1), (1, (1 << 30) + 1, 1)])
def test_linear_fp8_refuses_sizes(m, n, k, dev="cpu"):
    """Broadcast operands: refused by their sizes, before anything of them is laid out."""
    one, s = torch.zeros(1, 1, device=dev).to(E4M3), torch.ones(1, device=dev)
    with pytest.raises(ValueError, match="up to"):
        ops.linear_fp8(one.expand(m, k), s.expand(m), one.expand(n, k), s.expand(n))
