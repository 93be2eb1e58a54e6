"""The block operators on the CPU: their fp32 statements against 64 bits, and what they refuse."""
import math

import pytest
import torch

import block_ops_oracle as oracle
from ditserve_b200 import ops

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 96), (4, 256)])
def test_rms_norm_quant(dtype, shape):
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(dtype)
    oracle.check_norm_quant(ops.rms_norm_quant(x, w, residual=r), x, w, r, 1e-6)
    oracle.check_norm_quant(ops.rms_norm_quant(x, None, eps=1e-3), x, None, None, 1e-3)
    out, s, h = torch.empty(shape).to(ops.fp8.E4M3), torch.empty(shape[:-1]), r.clone()
    got = ops.rms_norm_quant(x, w, residual=h, out=out, scale_out=s, residual_out=h)
    assert got[0] is out and got[1] is s and got[2] is h
    oracle.check_norm_quant(got, x, w, r, 1e-6)


def test_rms_norm_quant_zero_and_nan_rows():
    x = torch.zeros(3, 32, dtype=BF)
    x[1, 4] = math.inf
    q, s, _ = ops.rms_norm_quant(x)
    assert s[0] == s[2] == torch.tensor(1e-30) and not q[0].float().any()
    assert s[1].isnan() and q[1].float().isnan().all()


@pytest.mark.parametrize("bad", [
    lambda x, w: ops.rms_norm_quant(x.double()),
    lambda x, w: ops.rms_norm_quant(x[:, :0]),
    lambda x, w: ops.rms_norm_quant(x, w[:-1]),
    lambda x, w: ops.rms_norm_quant(x, w.float()),
    lambda x, w: ops.rms_norm_quant(x, w, residual=x[:1]),
    lambda x, w: ops.rms_norm_quant(x, w, residual=x.float()),
    lambda x, w: ops.rms_norm_quant(x, w, residual_out=x),
    lambda x, w: ops.rms_norm_quant(x, w, out=torch.empty(x.shape)),
    lambda x, w: ops.rms_norm_quant(x, w, scale_out=torch.empty(x.shape)),
])
def test_rms_norm_quant_refusals(bad):
    with pytest.raises(ValueError):
        bad(torch.ones(4, 16, dtype=BF), torch.ones(16, dtype=BF))


def _quantised(m, n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    xq, xs = ops.quantize_rows_fp8(torch.randn(m, k, generator=g))
    wq, ws = ops.quantize_rows_fp8(torch.randn(n, k, generator=g) / math.sqrt(k))
    return xq, xs, wq, ws


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 17), (16, 64, 100)])
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_linear_fp8(m, n, k, dtype):
    xq, xs, wq, ws = _quantised(m, n, k)
    b, r, gate = torch.randn(n).to(dtype), torch.randn(m, n).to(dtype), torch.randn(2, n)
    rows = torch.arange(m) // ((m + 1) // 2)
    for kw, okw in (({}, {}), (dict(act="gelu"), dict(act="gelu")), (dict(residual=r), dict(residual=r)),
                    (dict(residual=r, gate=gate, rows_per_batch=(m + 1) // 2), dict(residual=r, gate_rows=gate[rows])),
                    (dict(residual=r, gate=gate, row_batch=(1 - rows).int()), dict(residual=r, gate_rows=gate[1 - rows]))):
        y = ops.linear_fp8(xq, xs, wq, ws, b, out_dtype=dtype, **kw)
        oracle.check_linear(y, *oracle.linear(xq, xs, wq, ws, b, **okw))
    out = torch.empty(m, n, dtype=dtype)
    assert ops.linear_fp8(xq, xs, wq, ws, out=out) is out


def test_quantize_rows_fp8_rows_start_on_16_bytes():
    w = torch.randn(5, 19)
    q, s = ops.quantize_rows_fp8(w)
    assert q.shape == w.shape and q.stride() == (32, 1)
    # half a step: 2^-4 of a normal value, 2^-10 * scale below
    assert ((q.float() * s[:, None] - w).abs() <= w.abs() * 2.0 ** -4 * 1.001 + s[:, None] * 2.0 ** -10).all()


@pytest.mark.parametrize("bad", [
    lambda x, s, w, t, b: ops.linear_fp8(x.float(), s, w, t),
    lambda x, s, w, t, b: ops.linear_fp8(x[:, :-1], s, w, t),
    lambda x, s, w, t, b: ops.linear_fp8(x, s[:-1], w, t),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t.double()),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b.float()),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b, act="relu"),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b, act="gelu", residual=torch.ones(4, 6, dtype=BF)),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b, residual=torch.ones(4, 6)),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b, gate=torch.ones(6)),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b, gate=torch.ones(1, 6), rows_per_batch=2,
                                         residual=torch.ones(4, 6, dtype=BF)),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, b, gate=torch.ones(6), row_batch=torch.zeros(4),
                                         residual=torch.ones(4, 6, dtype=BF)),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, out_dtype=torch.float64),
    lambda x, s, w, t, b: ops.linear_fp8(x, s, w, t, out=torch.empty(4, 5)),
    lambda x, s, w, t, b: ops.quantize_rows_fp8(s),
])
def test_linear_fp8_refusals(bad):
    with pytest.raises(ValueError):
        bad(*_quantised(4, 6, 32), torch.zeros(6, dtype=BF))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dims,head_dim", [((44, 42, 42), 128), ((6, 4), 12), ((2,), 2), ((4, 4, 2, 2), 16)])
@pytest.mark.parametrize("dtype", [BF, FL])
def test_rope_axes(layout, dims, head_dim, dtype):
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(-50, 1000, (6, len(dims)), generator=g)
    x, k = torch.randn(12, 3 * head_dim, generator=g).to(dtype), torch.randn(12, head_dim, generator=g).to(dtype)
    theta = tuple(10000.0 / (i + 1) for i in range(len(dims)))
    y, ky = ops.rope_axes(x, pos, dims, k=k, head_dim=head_dim, theta=theta, layout=layout)
    oracle.check_rope(y, x, pos, dims, head_dim, theta, layout)
    oracle.check_rope(ky, k, pos, dims, head_dim, theta, layout)
    z = ops.rope_axes(x, pos, dims, head_dim=head_dim, theta=theta, layout=layout, inverse=True)
    oracle.check_rope(z, x, pos, dims, head_dim, theta, layout, True)


def test_rope_axes_inverse_is_the_gradient():
    """The rotation is linear, so its gradient is its transpose: against autograd through the formula."""
    g = torch.Generator().manual_seed(2)
    pos, dims = ops.grid_positions((2, 3, 4)), (4, 6, 6)
    x = torch.randn(24, 32, generator=g, requires_grad=True)
    dy = torch.randn(24, 32, generator=g)
    ops.rope_axes_reference(x, pos, dims, 16, (1e4,) * 3).backward(dy)
    got = ops.rope_axes(dy, pos, dims, head_dim=16, inverse=True)
    # two products and a sum on either side
    torch.testing.assert_close(got, x.grad, rtol=0, atol=8 * 2.0 ** -24 * float(dy.abs().max()) * 2)


def test_rope_axes_is_wans_table_rotation():
    """On a raster grid the op agrees with the table-driven rotation that the video model uses."""
    from ditserve_b200.models.wan.config import CONFIGS
    from ditserve_b200.models.wan.model import rope_tables
    cfg = CONFIGS["wan2.1-t2v-1.3b"]
    cos, sin = rope_tables(cfg, (2, 3, 5), "cpu")
    x = torch.randn(30, 256)
    got = ops.rope_axes(x, ops.grid_positions((2, 3, 5)), (44, 42, 42), head_dim=128, theta=cfg.rope_theta)
    torch.testing.assert_close(got, ops.rope_reference(x, cos, sin, 128), rtol=0, atol=8 * 2.0 ** -24 * 8)


@pytest.mark.parametrize("bad", [
    lambda x, p: ops.rope_axes(x, p, (8, 8)),
    lambda x, p: ops.rope_axes(x, p, (3, 8, 8), head_dim=32),
    lambda x, p: ops.rope_axes(x, p, (16, 16, 16), head_dim=32),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=33),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, theta=(1e4, 1e4)),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, theta=0.0),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, layout="pairs"),
    lambda x, p: ops.rope_axes(x, p.to(torch.int16), (8, 8, 8), head_dim=32),
    lambda x, p: ops.rope_axes(x, p[:5], (8, 8, 8), head_dim=32),
    lambda x, p: ops.rope_axes(x, p[:0], (8, 8, 8), head_dim=32),
    lambda x, p: ops.rope_axes(x.double(), p, (8, 8, 8), head_dim=32),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, k=x[:4]),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, k=x.float()),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, k_out=x),
    lambda x, p: ops.rope_axes(x, p, (8, 8, 8), head_dim=32, out=x.float()),
])
def test_rope_axes_refusals(bad):
    with pytest.raises(ValueError):
        bad(torch.ones(8, 64, dtype=BF), ops.grid_positions((2, 2, 2)))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,heads_kv,d", [(2, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("sq,sk", [(1, 1), (5, 9), (3, 40)])
def test_cross_attention(dtype, heads, heads_kv, d, sq, sk):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(3, sq, heads * d, generator=g).to(dtype)
    k, v = (torch.randn(3, sk, heads_kv * d, generator=g).to(dtype) for _ in range(2))
    lens = torch.tensor([sk, 0, (sk + 1) // 2])
    mask = torch.rand(3, sk, generator=g) < 0.7
    valid = torch.arange(sk) < lens[:, None]
    k[~valid] = math.nan  # what padding holds does not matter
    v[~valid] = math.inf
    for kw, allowed in ((dict(kv_lens=lens), valid), (dict(kv_lens=lens.int(), key_mask=mask), valid & mask)):
        o, lse = ops.cross_attention(q, k, v, heads, heads_kv=heads_kv, return_lse=True, **kw)
        oracle.check_cross(o, lse, q, k, v, heads, heads_kv, allowed)


def test_cross_attention_without_keys():
    q = torch.randn(2, 3, 64).to(BF)
    o, lse = ops.cross_attention(q, q[:, :0], q[:, :0], 1, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    assert ops.cross_attention(q[:, :0], q, q, 1).shape == (2, 0, 64)
    assert ops.cross_attention(q[0], q[1], q[1], 1).shape == (3, 64)


@pytest.mark.parametrize("bad", [
    lambda q, k: ops.cross_attention(q, k[0], k[0], 2),
    lambda q, k: ops.cross_attention(q.float(), k.float(), k.float(), 2),
    lambda q, k: ops.cross_attention(q, k.half(), k.half(), 2),
    lambda q, k: ops.cross_attention(q, k, k, 3),
    lambda q, k: ops.cross_attention(q, k, k, 4),
    lambda q, k: ops.cross_attention(q, k, k, 2, heads_kv=1),
    lambda q, k: ops.cross_attention(q, k, k[:, :-1], 2),
    lambda q, k: ops.cross_attention(q, k[:1], k[:1], 2),
    lambda q, k: ops.cross_attention(q, k, k, 2, kv_lens=torch.ones(3, dtype=torch.int32)),
    lambda q, k: ops.cross_attention(q, k, k, 2, kv_lens=torch.ones(2)),
    lambda q, k: ops.cross_attention(q, k, k, 2, key_mask=torch.ones(2, 4, dtype=torch.bool)),
    lambda q, k: ops.cross_attention(q, k, k, 2, key_mask=torch.ones(2, 5)),
    lambda q, k: ops.cross_attention(q, k, k, 2, scale=0.0),
    lambda q, k: ops.cross_attention(q, k, k, 2, scale=-1.0),
    lambda q, k: ops.cross_attention(q, k, k, 2, out=q.float()),
    lambda q, k: ops.cross_attention(q, k, k, 2, out=q),
])
def test_cross_attention_refusals(bad):
    with pytest.raises(ValueError):
        bad(torch.ones(2, 3, 128, dtype=BF), torch.ones(2, 5, 128, dtype=BF))


def test_overlap_of_outputs():
    from ditserve_b200.ops.fp8 import _partial_overlap as over
    buf = torch.zeros(8, 96)
    a, b = buf[:, :32], buf[:, 32:64]
    assert not over(a, a) and not over(a, b) and not over(b, a) and not over(a, torch.zeros(8, 32))
    assert over(buf[:, 16:48], a) and over(a, buf[:, 16:48]) and over(buf[1:, :32], buf[:-1, :32])
    assert over(buf[:, :32], buf[:, :32].reshape(-1)[:0].new_empty(0, 32)) is False


@pytest.mark.parametrize("bad", [
    lambda q, k: ops.cross_attention(q, k, k, 2, heads_kv=0),
    lambda q, k: ops.cross_attention(q[:1].expand(65536, -1, -1), k[:1].expand(65536, -1, -1), k[:1].expand(65536, -1, -1), 2),
])
def test_cross_attention_refuses_counts(bad):
    with pytest.raises(ValueError):
        bad(torch.ones(2, 1, 128, dtype=BF), torch.ones(2, 1, 128, dtype=BF))
