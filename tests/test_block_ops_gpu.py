"""The block operators' kernels against plain implementations in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import block_ops_oracle as oracle
from ditserve_b200 import ops

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _dev():
    return torch.device("cuda", 0)


def _randn(*shape, seed=0, dtype=FL, std=1.0):
    g = torch.Generator(device=_dev()).manual_seed(seed)
    return (torch.randn(*shape, device=_dev(), generator=g) * std).to(dtype)


# ---- rms_norm_quant ---------------------------------------------------------------------------
# widths: one element, odd, a vector, warp form, block form with 1, 2 and 4 vectors a thread, long rows
@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("rows,dim", [(1, 1), (5, 7), (3, 8), (1300, 64), (1300, 100), (1201, 1536), (1190, 333), (7, 1536),
                                      (2, 4096), (3, 10240), (2, 20000), (2, 40000), (1, 4099), (2, 70000)])
def test_rms_norm_quant(dtype, rows, dim):
    x, r = _randn(rows, dim, seed=1, dtype=dtype), _randn(rows, dim, seed=2, dtype=dtype, std=3.0)
    w = (1 + 0.2 * _randn(dim, seed=3)).to(dtype)
    oracle.check_norm_quant(ops.rms_norm_quant(x, w, residual=r), x, w, r, 1e-6)
    oracle.check_norm_quant(ops.rms_norm_quant(x, None, eps=1e-5), x, None, None, 1e-5)


def test_rms_norm_quant_strides_and_in_place():
    buf = _randn(40, 3 * 264, seed=4, dtype=BF)
    for lo, dim in ((264, 264), (265, 200), (3, 64)):  # rows on 16 bytes, and not
        x, r = buf[:, lo:lo + dim], _randn(40, dim + 8, seed=5, dtype=BF)[:, :dim]
        w = _randn(dim, seed=6, dtype=BF)
        want = r.clone()
        q = torch.full((40, dim + 3), 7.0, device=_dev()).to(ops.fp8.E4M3)
        s = torch.zeros(40, 2, device=_dev())
        got = ops.rms_norm_quant(x, w, residual=r, residual_out=r, out=q[:, :dim])
        oracle.check_norm_quant(got, x, w, want, 1e-6)
        assert got[2] is r and (q[:, dim:].float() == 7).all()
    x3 = _randn(2, 5, 96, seed=7, dtype=HF)
    q, s, h = ops.rms_norm_quant(x3, residual=x3)
    oracle.check_norm_quant((q, s, h), x3, None, x3, 1e-6)
    assert h.shape == x3.shape
    oracle.check_norm_quant(ops.rms_norm_quant(x3.transpose(0, 1)), x3.transpose(0, 1), None, None, 1e-6)
    assert ops.rms_norm_quant(x3[:0])[0].shape == (0, 5, 96)


@pytest.mark.parametrize("rows", [3, 1200])
def test_rms_norm_quant_zero_nan_and_large_rows(rows):
    x = _randn(rows, 512, seed=8, dtype=BF)
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 9] = math.nan
    q, s, _ = ops.rms_norm_quant(x)
    assert s[0].item() == pytest.approx(1e-30) and not q[0].float().any()
    assert s[1:3].isnan().all() and q[1:3].float().isnan().all()
    assert s[3:].isfinite().all() and q[3:].float().isfinite().all()
    x = _randn(rows, 512, seed=9, dtype=FL) * 1e15
    oracle.check_norm_quant(ops.rms_norm_quant(x), x, None, None, 1e-6)
    x = x * 1e-30  # eps outweighs the row
    oracle.check_norm_quant(ops.rms_norm_quant(x), x, None, None, 1e-6)


# ---- linear_fp8 -------------------------------------------------------------------------------
def _quantised(m, n, k, seed=0):
    return (*ops.quantize_rows_fp8(_randn(m, k, seed=seed)),
            *ops.quantize_rows_fp8(_randn(n, k, seed=seed + 1, std=1 / math.sqrt(k))))


SHAPES = [(1, 1, 1), (1, 64, 4096), (2, 9216, 1536), (8, 17, 33), (9, 48, 64), (16, 100, 1000), (17, 256, 160), (33, 31, 16),
          (77, 4096, 512), (128, 256, 128), (129, 384, 129), (300, 1000, 4097), (1000, 1536, 1536), (2049, 776, 200),
          (700, 10240, 512)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_linear_fp8(m, n, k, dtype):
    xq, xs, wq, ws = _quantised(m, n, k)
    b = _randn(n, seed=5, dtype=dtype)
    oracle.check_linear(ops.linear_fp8(xq, xs, wq, ws, out_dtype=dtype), *oracle.linear(xq, xs, wq, ws))
    oracle.check_linear(ops.linear_fp8(xq, xs, wq, ws, b, act="gelu", out_dtype=dtype),
                        *oracle.linear(xq, xs, wq, ws, b, act="gelu"))
    r, gate = _randn(m, n, seed=6, dtype=dtype), _randn(3, n, seed=7)
    rows = torch.arange(m, device=_dev()) // max(1, -(-m // 3))
    oracle.check_linear(ops.linear_fp8(xq, xs, wq, ws, b, residual=r, out_dtype=dtype),
                        *oracle.linear(xq, xs, wq, ws, b, residual=r))
    want = oracle.linear(xq, xs, wq, ws, b, residual=r, gate_rows=gate[rows])
    oracle.check_linear(ops.linear_fp8(xq, xs, wq, ws, b, residual=r, gate=gate, rows_per_batch=max(1, -(-m // 3)),
                                       out_dtype=dtype), *want)
    oracle.check_linear(ops.linear_fp8(xq, xs, wq, ws, b, residual=r, gate=gate, row_batch=rows.int(), out_dtype=dtype), *want)
    out = r.clone()
    assert ops.linear_fp8(xq, xs, wq, ws, b, residual=out, gate=gate, row_batch=rows.int(), out=out) is out
    oracle.check_linear(out, *want)
    ops.check_status(_dev())


@pytest.mark.parametrize("m", [1, 20, 260])
def test_linear_fp8_strides_padding_and_alignment(m):
    n, k = 70, 100
    xq, xs, wq, ws = _quantised(m, n, k)
    want = oracle.linear(xq, xs, wq, ws)
    nan = torch.full((1,), 0x7f, dtype=torch.uint8, device=_dev()).view(ops.fp8.E4M3)
    # what lies behind K in a row, or behind the last row, is not read into a sum
    pad = nan.view(torch.uint8).expand(m + 2, 144).contiguous().view(ops.fp8.E4M3)
    pad[:m, :k] = xq
    wpad = nan.view(torch.uint8).expand(n + 2, 160).contiguous().view(ops.fp8.E4M3)
    wpad[:n, :k] = wq
    big = torch.full((m + 1, n + 5), 7.0, device=_dev(), dtype=BF)
    y = ops.linear_fp8(pad[:m, :k], xs, wpad[:n, :k], ws, out=big[:m, 2:n + 2])
    oracle.check_linear(y, *want)
    assert (big[m:] == 7).all() and (big[:, :2] == 7).all() and (big[:, n + 2:] == 7).all()
    # packed rows of 100 bytes, and columns with gaps: copied first
    oracle.check_linear(ops.linear_fp8(xq.contiguous(), xs, wq.contiguous(), ws), *want)
    scales = torch.stack([xs, xs], 1)[:, 0]
    oracle.check_linear(ops.linear_fp8(pad[:m, :k], scales, wq.t().contiguous().t(), ws), *want)
    x3 = xq.contiguous().view(1, m, k)
    assert ops.linear_fp8(x3, xs.view(1, m), wq, ws).shape == (1, m, n)
    assert ops.linear_fp8(xq[:0], xs[:0], wq, ws).shape == (0, n)
    assert ops.linear_fp8(xq, xs, wq[:0], ws[:0]).shape == (m, 0)
    ops.check_status(_dev())


# ---- rope_axes --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rows,heads,heads_k,head_dim,dims", [
    (1, 12, 12, 128, (44, 42, 42)), (77, 24, 6, 64, (32, 32)), (130, 4, 1, 96, (32, 32, 32)), (33, 3, 3, 80, (20, 30, 30)),
    (64, 2, 2, 64, (16, 16)), (9, 5, 1, 34, (2, 4)), (5, 1, 1, 2, (2,)), (6, 2, 1, 512, (128, 128, 128, 128)),
    (1001, 12, 2, 128, (128,)), (7, 3, 3, 12, (8,))])
def test_rope_axes(dtype, layout, rows, heads, heads_k, head_dim, dims):
    g = torch.Generator(device=_dev()).manual_seed(3)
    pos = torch.randint(-20, 5000, (rows, len(dims)), device=_dev(), generator=g)
    x, k = _randn(rows, heads * head_dim, seed=1, dtype=dtype), _randn(rows, heads_k * head_dim, seed=2, dtype=dtype)
    theta = tuple(10000.0 * (i + 1) for i in range(len(dims)))
    y, ky = ops.rope_axes(x, pos, dims, k=k, head_dim=head_dim, theta=theta, layout=layout)
    oracle.check_rope(y, x, pos, dims, head_dim, theta, layout)
    oracle.check_rope(ky, k, pos, dims, head_dim, theta, layout)
    z = ops.rope_axes(x, pos, dims, head_dim=head_dim, theta=theta, layout=layout, inverse=True, out=x.clone())
    oracle.check_rope(z, x, pos, dims, head_dim, theta, layout, True)


@pytest.mark.parametrize("ptype", [torch.int64, torch.int32, FL, torch.float64])
def test_rope_axes_positions(ptype):
    """Far, fractional and strided positions, shared by a batch."""
    dims, theta = (64, 64), (1e4, 1e4)
    p = torch.tensor([[0, 1], [1 << 20, -(1 << 20)], [(1 << 30) + 1, 77], [5, 1000003]], device=_dev()).to(ptype)
    if ptype.is_floating_point:
        p = p + 0.25
    wide = torch.zeros(4, 5, device=_dev(), dtype=ptype)
    wide[:, 1::2] = p
    x = _randn(3, 4, 256, seed=1)
    for q in (p, wide[:, 1::2], p.t().contiguous().t()):
        y = ops.rope_axes(x, q, dims, head_dim=128)
        assert y.shape == x.shape
        oracle.check_rope(y.view(12, 256), x.view(12, 256), p, dims, 128, theta)


def test_rope_axes_in_place_on_a_fused_buffer():
    qkv, pos = _randn(50, 3 * 256, seed=1, dtype=BF), ops.grid_positions((2, 5, 5), _dev())
    before = qkv.clone()
    q, k = qkv[:, :256], qkv[:, 256:512]
    ops.rope_axes(q, pos, (44, 42, 42), k=k, head_dim=128, out=q, k_out=k)
    for a, b in ((q, before[:, :256]), (k, before[:, 256:512])):
        oracle.check_rope(a, b, pos, (44, 42, 42), 128, (1e4,) * 3)
    assert torch.equal(qkv[:, 512:], before[:, 512:])
    odd = qkv[:, 1:257]  # rows off 16 bytes
    oracle.check_rope(ops.rope_axes(odd, pos, (44, 42, 42), head_dim=128), odd, pos, (44, 42, 42), 128, (1e4,) * 3)
    with pytest.raises(ValueError):
        ops.rope_axes(q, pos, (44, 42, 42), out=qkv[:, 8:264])
    with pytest.raises(ValueError):
        ops.rope_axes(q, pos, (44, 42, 42), k=k, out=q, k_out=q)
    assert ops.rope_axes(q[:0], pos, (44, 42, 42)).shape == (0, 256)


# ---- cross_attention --------------------------------------------------------------------------
# few queries and many, one key to many, widths that end inside a tile, shared key heads
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,sq,sk,heads,heads_kv,d", [
    (1, 1, 1, 1, 1, 64), (2, 1, 512, 12, 12, 128), (1, 1, 5000, 4, 1, 128), (3, 7, 17, 6, 2, 64), (2, 16, 130, 8, 2, 128),
    (2, 33, 77, 4, 4, 64), (1, 128, 128, 2, 2, 128), (2, 129, 257, 3, 3, 64), (2, 300, 333, 4, 2, 128),
    (1, 1000, 64, 2, 1, 64), (1, 257, 2048, 2, 2, 128), (1, 64, 3000, 2, 2, 64), (1, 700, 513, 24, 24, 128)])
def test_cross_attention(dtype, B, sq, sk, heads, heads_kv, d):
    q = _randn(B, sq, heads * d, seed=1, dtype=dtype)
    k, v = _randn(B, sk, heads_kv * d, seed=2, dtype=dtype), _randn(B, sk, heads_kv * d, seed=3, dtype=dtype)
    o, lse = ops.cross_attention(q, k, v, heads, heads_kv=heads_kv, return_lse=True)
    ops.check_status(_dev())
    oracle.check_cross(o, lse, q, k, v, heads, heads_kv)
    lens = torch.tensor([max(0, sk - i * (sk // 2) - 1) for i in range(B)], device=_dev())
    mask = torch.rand(B, sk, device=_dev(), generator=torch.Generator(device=_dev()).manual_seed(4)) < 0.6
    valid = torch.arange(sk, device=_dev()) < lens[:, None]
    for i, (kw, allowed) in enumerate(((dict(kv_lens=lens.int()), valid), (dict(key_mask=mask), mask),
                                       (dict(kv_lens=lens, key_mask=mask), valid & mask))):
        ki, vi = k.masked_fill(~allowed[..., None], math.nan), v.masked_fill(~allowed[..., None], (math.inf, math.nan)[i % 2])
        o, lse = ops.cross_attention(q, ki, vi, heads, heads_kv=heads_kv, return_lse=True, scale=0.2, **kw)
        ops.check_status(_dev())
        oracle.check_cross(o, lse, q, ki, vi, heads, heads_kv, allowed, 0.2)


@pytest.mark.parametrize("sq", [1, 40, 300])
def test_cross_attention_empty_rows(sq):
    q, k, v = (_randn(4, n, 256, seed=s, dtype=BF) for n, s in ((sq, 1), (200, 2), (200, 3)))
    lens = torch.tensor([200, 0, -3, 999], device=_dev(), dtype=torch.int32)
    mask = torch.ones(4, 200, dtype=torch.bool, device=_dev())
    mask[0, :128] = False  # a whole tile
    mask[3] = False
    out = torch.full((4, sq, 256), 7.0, device=_dev(), dtype=BF)
    o, lse = ops.cross_attention(q, k, v, 2, kv_lens=lens, key_mask=mask, return_lse=True, out=out)
    assert o is out
    allowed = mask & (torch.arange(200, device=_dev()) < lens[:, None])
    oracle.check_cross(o, lse, q, k, v, 2, allowed=allowed)
    assert not o[1:].any() and (lse[1:] == -math.inf).all()
    o, lse = ops.cross_attention(q, k[:, :0], v[:, :0], 2, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    assert ops.cross_attention(q[:, :0], k, v, 2).shape == (4, 0, 256)


@pytest.mark.parametrize("sq", [2, 300])
def test_cross_attention_strides(sq):
    """Slices of fused buffers, a shared context, a strided mask, rows off 16 bytes, large scores."""
    qb, kvb = _randn(3, sq + 4, 1024, seed=1, dtype=BF), _randn(150, 3, 512, seed=2, dtype=BF)
    q, k, v = qb[:, 2:sq + 2, 256:512], kvb.transpose(0, 1)[..., :256], kvb.transpose(0, 1)[..., 256:]
    ob = torch.full((3, sq + 2, 512), 7.0, device=_dev(), dtype=BF)
    mask = (torch.rand(150, 6, device=_dev()) < 0.7).t()[::2]
    o = ops.cross_attention(q, k, v, 2, key_mask=mask, out=ob[:, 1:sq + 1, 128:384])
    oracle.check_cross(o, None, q, k, v, 2, allowed=mask)
    assert (ob[:, 0] == 7).all() and (ob[:, -1] == 7).all() and (ob[..., :128] == 7).all() and (ob[..., 384:] == 7).all()
    ks, vs = k[:1].expand(3, -1, -1), v[:1].expand(3, -1, -1)
    oracle.check_cross(ops.cross_attention(q, ks, vs, 2), None, q, ks, vs, 2)
    odd = qb[:, :sq, 257:513]
    oracle.check_cross(ops.cross_attention(odd, k, v, 2), None, odd, k, v, 2)
    # a running maximum that climbs from tile to tile
    ramp = (k.float() * torch.linspace(0, 6, 150, device=_dev())[None, :, None]).to(BF)
    o, lse = ops.cross_attention(q, ramp, v, 2, return_lse=True, scale=0.5)
    oracle.check_cross(o, lse, q, ramp, v, 2, scale=0.5)


# ---- together, other streams, graphs ----------------------------------------------------------
def _block(x, res, w, wq, ws, b, pos, ctx, lens, heads, d):
    xq, xs, h = ops.rms_norm_quant(x, w, residual=res)
    qkv = ops.linear_fp8(xq, xs, wq, ws, b)
    n = heads * d
    q, k, v = qkv[:, :n], qkv[:, n:2 * n], qkv[:, 2 * n:]
    ops.rope_axes(q, pos, (44, 42, 42), k=k, head_dim=d, out=q, k_out=k)
    a = ops.attention(q, k, v, heads)
    c = ops.cross_attention(a.view(lens.numel(), -1, n), ctx[..., :n], ctx[..., n:], heads, kv_lens=lens)
    return h, qkv, c


def _block_inputs(seed=0):
    heads, d = 4, 128
    n = heads * d
    wq, ws = ops.quantize_rows_fp8(_randn(3 * n, n, seed=seed + 3, std=n ** -0.5, dtype=BF))
    return dict(x=_randn(2 * 60, n, seed=seed, dtype=BF), res=_randn(2 * 60, n, seed=seed + 1, dtype=BF),
                w=(1 + 0.1 * _randn(n, seed=seed + 2)).to(BF), wq=wq, ws=ws, b=_randn(3 * n, seed=seed + 4, dtype=BF),
                pos=ops.grid_positions((3, 4, 5), _dev()), ctx=_randn(2, 77, 2 * n, seed=seed + 5, dtype=BF),
                lens=torch.tensor([77, 20], device=_dev(), dtype=torch.int32), heads=heads, d=d)


def test_block_in_one_run():
    """Norm, 8-bit projection, rotation, self and cross attention: the last against the CPU's run of the same."""
    s = _block_inputs()
    got = _block(**s)
    ops.check_status(_dev())
    want = _block(**{k: v.cpu() if torch.is_tensor(v) else v for k, v in s.items()})
    assert torch.equal(got[0].cpu(), want[0])
    # e4m3 codes next to a border may fall to either side (2^-3 of few values), bf16 rounds each stage
    for a, b in zip(got[1:], want[1:]):
        a, b = a.cpu().float(), b.float()
        assert ((a - b).norm() / b.norm()).item() < 2 ** -6


def test_block_on_another_stream_and_in_graphs():
    s, other = _block_inputs(), _block_inputs(seed=50)
    want = _block(**s)
    want2 = _block(**other)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(**s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for inputs in (s, s):  # two captured graphs, replayed in turn on new values
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _block(**inputs)
        graphs.append((g, out))
    for name in ("x", "res", "w", "wq", "ws", "b", "ctx", "lens"):
        s[name].copy_(other[name])
    for g, out in graphs + graphs[::-1]:
        for t in out:
            t.zero_()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want2))
    ops.check_status(_dev())


def test_refusals_on_the_device():
    x = _randn(4, 64, dtype=BF)
    with pytest.raises(Exception):
        ops.rms_norm_quant(x, torch.ones(64, dtype=BF))  # weight on the CPU
    with pytest.raises(ValueError):
        ops.rms_norm_quant(x, residual=x, residual_out=x.view(-1)[4:4 + 0].view(0, 64))
    wide = _randn(5, 64, dtype=BF)
    with pytest.raises(ValueError):
        ops.rms_norm_quant(wide[:4], residual=x, residual_out=wide[1:])
    xq, xs, wq, ws = _quantised(4, 64, 64)
    with pytest.raises(Exception):
        ops.linear_fp8(xq, xs.cpu(), wq, ws)
    with pytest.raises(Exception):
        ops.rope_axes(x, ops.grid_positions((4,)), (64,), head_dim=64)
    q = x.view(1, 4, 64)
    with pytest.raises(Exception):
        ops.cross_attention(q, q, q, 1, kv_lens=torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.cross_attention(q, q, q, 1, out=q)


def _to_dev(case):
    """The CPU refusals' calls on CUDA tensors: creation functions inside them run under a default device."""
    def run(*args):
        with torch.device(_dev()):
            case(*(a.to(_dev()) for a in args))
    return run


def test_refusals_of_the_cpu_hold_on_the_device():
    import test_block_ops as cpu
    marks = {f.__name__: f.pytestmark[0].args[1] for f in (cpu.test_rms_norm_quant_refusals, cpu.test_linear_fp8_refusals,
                                                           cpu.test_rope_axes_refusals, cpu.test_cross_attention_refusals)}
    args = {"test_rms_norm_quant_refusals": (torch.ones(4, 16, dtype=BF), torch.ones(16, dtype=BF)),
            "test_linear_fp8_refusals": (*cpu._quantised(4, 6, 32), torch.zeros(6, dtype=BF)),
            "test_rope_axes_refusals": (torch.ones(8, 64, dtype=BF), ops.grid_positions((2, 2, 2))),
            "test_cross_attention_refusals": (torch.ones(2, 3, 128, dtype=BF), torch.ones(2, 5, 128, dtype=BF))}
    before = ops.launch_counts()
    for name, cases in marks.items():
        for i, case in enumerate(cases):
            with pytest.raises(ValueError):
                _to_dev(case)(*args[name])
                pytest.fail(f"{name}[{i}] was not refused")
    assert ops.launch_counts() == before  # nothing ran


# ---- more work than the device holds at once, wide strides, calls side by side ------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,sq,sk,heads,heads_kv,d", [
    (8, 300, 200, 24, 24, 64), (6, 260, 333, 16, 16, 128), (5, 1024, 333, 24, 24, 64), (7, 130, 140, 30, 10, 128),
    (4, 700, 129, 48, 16, 64)])
def test_cross_attention_several_units_a_block(dtype, B, sq, sk, heads, heads_kv, d):
    """Row tiles for several rounds of the device, odd counts of them, entries of every length with empty ones between."""
    q = _randn(B, sq, heads * d, seed=1, dtype=dtype)
    k, v = _randn(B, sk, heads_kv * d, seed=2, dtype=dtype), _randn(B, sk, heads_kv * d, seed=3, dtype=dtype)
    lens = torch.tensor([(sk, 0, 1, sk // 2 + 1, 128, sk - 1, 0, 129)[i] for i in range(B)], device=_dev(), dtype=torch.int32)
    mask = torch.rand(B, sk, device=_dev(), generator=torch.Generator(device=_dev()).manual_seed(4)) < 0.6
    mask[0, sk // 3:] = False  # padding that the mask alone gives
    valid = torch.arange(sk, device=_dev()) < lens[:, None]
    for kw, allowed in ((dict(), valid | True), (dict(kv_lens=lens), valid), (dict(key_mask=mask), mask),
                        (dict(kv_lens=lens, key_mask=mask), valid & mask)):
        ki, vi = k.masked_fill(~allowed[..., None], math.nan), v.masked_fill(~allowed[..., None], math.nan)
        o, lse = ops.cross_attention(q, ki, vi, heads, heads_kv=heads_kv, return_lse=True, **kw)
        ops.check_status(_dev())
        oracle.check_cross(o, lse, q, ki, vi, heads, heads_kv, allowed)
        again = ops.cross_attention(q, ki, vi, heads, heads_kv=heads_kv, **kw)
        assert torch.equal(o, again)


@pytest.mark.parametrize("B,sq,sk,heads,masked", [(70, 130, 200, 1, False), (70, 130, 200, 2, True), (2, 300, 33000, 8, True)])
def test_cross_attention_more_keys_than_a_block_lists(B, sq, sk, heads, masked):
    q, k, v = (_randn(B, n, heads * 64, seed=s, dtype=BF) for n, s in ((sq, 1), (sk, 2), (sk, 3)))
    lens = torch.tensor([(i * 37) % (sk + 1) for i in range(B)], device=_dev(), dtype=torch.int32)
    lens[-1] = sk
    allowed = torch.arange(sk, device=_dev()) < lens[:, None]
    mask = None
    if masked:
        mask = torch.rand(B, sk, device=_dev(), generator=torch.Generator(device=_dev()).manual_seed(5)) < 0.5
        mask[B // 2] = False
        allowed = allowed & mask
    o, lse = ops.cross_attention(q, k, v, heads, kv_lens=lens, key_mask=mask, return_lse=True)
    ops.check_status(_dev())
    oracle.check_cross(o, lse, q, k, v, heads, None, allowed)


def _wide(buf, rows, cols, pitch, at, dtype, seed):
    """[rows, cols] of ``buf`` (bytes) with rows ``pitch`` elements apart from byte ``at`` on, filled."""
    t = buf.view(dtype).as_strided((rows, cols), (pitch, 1), at // dtype.itemsize)
    t.copy_(_randn(rows, cols, seed=seed, dtype=FL).to(dtype))
    return t


def test_rows_that_lie_more_than_32_bits_apart():
    buf = torch.empty(10 << 30, device=_dev(), dtype=torch.uint8)  # rows' last elements behind 2^32 of them
    wide = 1 << 30
    for rows, pitch in ((5, wide), (1200, wide >> 8)):
        x, r, h = (_wide(buf, rows, 256, pitch, i * 1024, BF, i) for i in range(3))
        q = _wide(buf, rows, 256, 2 * pitch, 4096, torch.float8_e4m3fn, 5)
        want = ops.rms_norm_quant(x.contiguous(), residual=r.contiguous())
        got = ops.rms_norm_quant(x, residual=r, residual_out=h, out=q)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
    pos = torch.arange(5, device=_dev())
    x, y = _wide(buf, 5, 256, wide, 0, BF, 1), _wide(buf, 5, 256, wide, 1024, BF, 2)
    assert torch.equal(ops.rope_axes(x, pos, (64,), out=y), ops.rope_axes(x.contiguous(), pos, (64,)))
    for m, n, cols in ((5, 5, 64), (300, 2000, 1024)):
        pitch = wide >> (0 if m == 5 else 6)
        x = _wide(buf, m, cols, 2 * pitch, 0, torch.float8_e4m3fn, 1)
        w = _wide(buf, n, cols, 2 * pitch, 1024, torch.float8_e4m3fn, 2) if m == 5 else _quantised(n, 1, cols)[0]
        sx, sw = torch.rand(m, device=_dev()), torch.rand(n, device=_dev())
        y = _wide(buf, m, n, pitch, 4096, BF, 3)
        want = ops.linear_fp8(x.contiguous(), sx, w.contiguous(), sw)
        assert torch.equal(ops.linear_fp8(x, sx, w, sw, out=y), want)
    pitch = wide >> 5
    far = torch.empty(10 << 29, device=_dev(), dtype=BF)
    for sq, heads in ((3, 2), (140, 20)):
        n = heads * 128
        k, v = (_wide(buf, 150, n, pitch, i * 8192, BF, i)[None] for i in range(2))
        q, o = (_wide(buf, sq, n, pitch, i * 8192, BF, i)[None] for i in (2, 3))
        want = ops.cross_attention(*(t.contiguous() for t in (q, k, v)), heads)
        # columns of one buffer meet in their spans: the result has to lie elsewhere
        with pytest.raises(ValueError):
            ops.cross_attention(q, k, v, heads, out=o)
        assert torch.equal(ops.cross_attention(q, k, v, heads, out=far.as_strided((1, sq, n), (0, pitch, 1))), want)
    ops.check_status(_dev())


def test_calls_side_by_side_on_two_streams():
    """Many-tile forms on two streams at once: neither keeps anything that the other could meet."""
    work = []
    for seed in (0, 40):
        q = _randn(4, 520, 12 * 64, seed=seed, dtype=BF)
        k, v = _randn(4, 300, 12 * 64, seed=seed + 1, dtype=BF), _randn(4, 300, 12 * 64, seed=seed + 2, dtype=BF)
        xq, xs, wq, ws = _quantised(1500, 1100, 640, seed=seed + 3)
        a, b, c, d = _quantised(20, 256, 8192, seed=seed + 7)

        def run(q=q, k=k, v=v, xq=xq, xs=xs, wq=wq, ws=ws, a=a, b=b, c=c, d=d):
            return (ops.cross_attention(q, k, v, 12), ops.linear_fp8(xq, xs, wq, ws), ops.linear_fp8(a, b, c, d),
                    ops.cross_attention(q[:, :2], k, v, 12), *ops.rms_norm_quant(q)[:2])
        work.append((run, run()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(10):
        for i, (run, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i].append(run())
    torch.cuda.synchronize()
    ops.check_status(_dev())
    for (_, want), runs in zip(work, got):
        for out in runs:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))


def test_theta_is_taken_by_value():
    x, pos = _randn(6, 128, dtype=BF), torch.arange(6, device=_dev())
    theta = torch.tensor([100.0])
    first = ops.rope_axes(x, pos, (64,), theta=theta)
    assert torch.equal(first, ops.rope_axes(x, pos, (64,), theta=100.0))
    theta.fill_(5000.0)
    assert torch.equal(ops.rope_axes(x, pos, (64,), theta=theta), ops.rope_axes(x, pos, (64,), theta=5000.0))


def test_outputs_on_operands_are_refused():
    x = _randn(8, 64, dtype=BF)
    with pytest.raises(ValueError):
        ops.rms_norm_quant(x, out=x.view(torch.float8_e4m3fn)[:, :64])
    h = torch.empty_like(x)
    with pytest.raises(ValueError):
        ops.rms_norm_quant(x, residual=x.clone(), residual_out=h, out=h.view(torch.float8_e4m3fn)[:, :64])
    # other columns of one buffer are apart
    buf = torch.zeros(8, 256, device=_dev(), dtype=torch.uint8)
    xs = buf[:, :128].view(BF)
    xs.copy_(x)
    oracle.check_norm_quant(ops.rms_norm_quant(xs, out=buf[:, 128:192].view(torch.float8_e4m3fn)), x, None, None, 1e-6)
    # a scale on the input is written last, through a copy
    want = ops.rms_norm_quant(x)
    f = x.clone()
    q, s, _ = ops.rms_norm_quant(f, scale_out=f.view(-1)[:16].view(FL))
    assert torch.equal(q.float(), want[0].float()) and torch.equal(s, want[1])
    xq, sx, wq, sw = _quantised(32, 32, 64)
    with pytest.raises(ValueError):
        ops.linear_fp8(xq, sx, wq, sw, out=xq.view(BF))
    with pytest.raises(ValueError):
        ops.linear_fp8(xq, sx, wq, sw, out=wq.view(BF))


@pytest.mark.parametrize("m,n,k", [(512, 10240, 4096), (513, 9001, 300), (1300, 4000, 96), (260, 19000, 130)])
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_linear_fp8_twin_tiles(m, n, k, dtype):
    """Between one and two rounds of tiles: two neighbours at once, the second behind the last channel among them."""
    test_linear_fp8(m, n, k, dtype)


@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_linear_fp8_twin_tiles_of_one_block(dtype):
    """One row of tiles for more channels than the device has blocks: twins without CTA pairs."""
    test_linear_fp8(100, 40000, 256, dtype)


@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("n", [641, 1555])
def test_linear_fp8_rows_off_16_bytes_in_place(n, dtype):
    """Odd rows with a gated residual that is the output, inside a wider buffer."""
    m, k = 700, 1700
    xq, xs, wq, ws = _quantised(m, n, k)
    buf, gate = _randn(m + 1, n + 4, seed=6, dtype=dtype), _randn(2, n, seed=7)
    keep = buf.clone()
    out = buf[:m, 3:n + 3]
    rows = torch.arange(m, device=_dev()) // 400
    want = oracle.linear(xq, xs, wq, ws, residual=out.clone(), gate_rows=gate[rows])
    ops.linear_fp8(xq, xs, wq, ws, residual=out, gate=gate, rows_per_batch=400, out=out)
    ops.check_status(_dev())
    oracle.check_linear(out, *want)
    buf[:m, 3:n + 3] = keep[:m, 3:n + 3]
    assert torch.equal(buf, keep)


@pytest.mark.parametrize("dtype", [BF, FL])
def test_linear_fp8_broadcast_residual(dtype):
    """One row of residual for all rows (a stride of 0), and rows of it that overlap."""
    m, n, k = 400, 1024, 1500
    xq, xs, wq, ws = _quantised(m, n, k)
    flat = _randn(n + 8 * m, seed=6, dtype=dtype)
    for r in (flat[:n].expand(m, n), flat.as_strided((m, n), (8, 1))):
        y = ops.linear_fp8(xq, xs, wq, ws, residual=r, out_dtype=dtype)
        ops.check_status(_dev())
        oracle.check_linear(y, *oracle.linear(xq, xs, wq, ws, residual=r))
