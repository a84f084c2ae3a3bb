"""ops.dropout, ops.layer_norm and ops.linear_cross_entropy (csrc/pg_norm.hip, csrc/pg_xent_linear.hip) against plain 64-bit
computations of the same inputs. Tolerances: one rounding of the result (half a step of its type), plus the fp32 roundings on the
way, counted: at most as many additions stand behind one another in a sum as its bound names, each off by 2^-24 of a partial sum
that is no larger than the sum of absolute values."""
import ctypes
import os

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24
gpu = pytest.mark.gpu


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """half of the smallest step a result may fall on: what a value near zero is off by"""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def close(got, ref, extra, what=""):
    """|got - ref| <= half a step of got's type + extra (both 64-bit), NaN where ref is NaN"""
    t, got = got.dtype, got.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    same_nan = torch.isnan(got) == torch.isnan(ref)
    assert same_nan.all(), f"{what}: NaN in other places"
    ref_ = torch.nan_to_num(ref, nan=0.0, posinf=0.0, neginf=0.0)
    got_ = torch.where(torch.isfinite(ref), got, torch.zeros_like(got))
    assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)]), what
    bound = half_step(t) * (ref_.abs() + extra) + extra + tiny(t)
    over = (got_ - ref_).abs() - bound
    assert not (over > 0).any(), f"{what}: off by {(got_ - ref_).abs().max():.3e}, {over.max():.3e} over the bound"


def gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def spec_of(dev, p, step=5, seed=0x1234567890ABCDEF, tag=7):
    from pagraph_amd import ops
    return ops.DropoutSpec(p, seed, tag, torch.tensor([step], dtype=torch.int64, device=dev))


def mask_of(oracle, n, d, spec, step):
    keep, scale = oracle.dropout_mask(n, d, spec.threshold, spec.seed, spec.tag, step)
    return torch.from_numpy(keep), float(scale)


# ---- without a GPU ---------------------------------------------------------------------------------------------------------
def test_refuses_host_tensors(hiplib):
    from pagraph_amd import _lib, ops
    lin, norm = torch.nn.Linear(8, 5), torch.nn.LayerNorm(8)
    spec = ops.DropoutSpec(0.5, 1, 2, None)
    with pytest.raises(_lib.PgError):
        ops.dropout(torch.zeros(3, 8), spec)
    with pytest.raises(_lib.PgError):
        ops.layer_norm(torch.zeros(3, 8), norm)
    with pytest.raises(_lib.PgError):
        ops.linear_cross_entropy(torch.zeros(3, 8), lin, torch.zeros(3, dtype=torch.int64))
    x = torch.zeros(3, 8)
    assert ops.dropout(x, None) is x and ops.dropout(x, ops.DropoutSpec(0.0, 1, 2, None)) is x


def test_library_refuses_bad_arguments(hiplib):
    from pagraph_amd import _lib as L
    ref = lambda o: ctypes.addressof(o) if o is not None else None
    drop = L.PgDropout(100, 0, 1, None, 0)
    call = lambda n=1, d=4, xs=4, ys=4, dt=0, dr=drop: hiplib.pg_dropout_apply(None, xs, None, ys, n, d, dt, ref(dr), None, None)
    assert call(n=-1) == call(d=0) == call(xs=3) == call(ys=3) == call(dt=3) == call(dr=None) == call() == -1
    assert call(dr=L.PgDropout(0, 0, 1, None, 0)) == -1
    assert call(n=1 << 32) == -4 and call(n=0) == 0
    a = L.PgNormDesc()
    assert hiplib.pg_layer_norm_fwd(None, None) == -1 and hiplib.pg_layer_norm_fwd(ref(a), None) == -1          # no columns
    a.n, a.d, a.x_stride, a.y_stride = 2, 8, 8, 8
    assert hiplib.pg_layer_norm_fwd(ref(a), None) == -1                                                         # no rows given
    a.d = L.PG_NORM_MAX_COLUMNS + 1
    assert hiplib.pg_layer_norm_fwd(ref(a), None) == -4 and hiplib.pg_layer_norm_bwd(ref(a), None) == -4
    a.d, a.has_drop, a.drop = 8, 1, drop
    assert hiplib.pg_layer_norm_fwd(ref(a), None) == -1                                                         # dropout without a residual
    assert hiplib.pg_layer_norm_scratch(10, 0, 0) == 0 and hiplib.pg_layer_norm_scratch(10, 8, 0) >= 16
    x = L.PgLinearXentDesc()
    assert hiplib.pg_linear_xent_fwd(None, None) == hiplib.pg_linear_xent_bwd(ref(x), None) == hiplib.pg_linear_xent_fwd(ref(x), None) == -1
    assert hiplib.pg_linear_xent_scratch(-1, 8, 8, 0, 0) == -1 and hiplib.pg_linear_xent_scratch(4, 8, 8, 5, 0) == -1
    assert hiplib.pg_linear_xent_scratch(1 << 31, 8, 1 << 20, 0, 1) == -1                                  # more tiles than a grid has
    assert hiplib.pg_linear_xent_scratch(0, 8, 8, 0, 1) == 0


def test_descriptors_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pagraph_amd import _lib
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    pairs = {"pg_norm_desc_t": _lib.PgNormDesc, "pg_linear_xent_desc_t": _lib.PgLinearXentDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{os.path.join(ROOT, "include", "pagraph_hip.h")}"', "int main(void) {"]
    for cname, cls in pairs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    (tmp_path / "a.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "a"), str(tmp_path / "a.c")], check=True)
    got = dict((tuple(l.split()[:2]), int(l.split()[2])) for l in
               subprocess.run([str(tmp_path / "a")], capture_output=True, text=True).stdout.splitlines())
    for cname, cls in pairs.items():
        assert got[(cname, "size")] == ctypes.sizeof(cls)
        for f in cls._fields_:
            assert got[(cname, f[0])] == getattr(cls, f[0]).offset, (cname, f[0])
    # the packed forms ops.py hands over are the same bytes
    from pagraph_amd import ops
    drop = (1, 2, 3, 4, 5)
    ptrs, sizes = tuple(range(10, 26)), tuple(range(-5, 5))
    assert ops._DROP_DESC(*drop) == bytes(_lib.PgDropout(*drop))
    assert ops._NORM_DESC(*ptrs, *sizes, 1, 2, 0.5, True, *drop) == bytes(_lib.PgNormDesc(*ptrs, *sizes, 1, 2, 0.5, 1, _lib.PgDropout(*drop)))
    assert ops._XENT_DESC(*ptrs[:14], *sizes[:7], 1, 2) == bytes(_lib.PgLinearXentDesc(*ptrs[:14], *sizes[:7], 1, 2))


def test_a_capture_meets_no_living_eager_graph(monkeypatch):
    """the rule of ops._watch_graph, with the streams made up"""
    from pagraph_amd import _lib, ops
    state = {"capturing": False, "stream": 1}
    monkeypatch.setattr(ops, "_capture_state", lambda device: (state["capturing"], state["stream"]))
    monkeypatch.setattr(ops, "_EAGER_GRAPHS", type(ops._EAGER_GRAPHS)())

    class F(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ops._watch_graph("f", ctx, x.device, x, w)
            return x * w

        @staticmethod
        def backward(ctx, g):
            return g, g
    x, w, v = (torch.ones(3, requires_grad=True) for _ in range(3))
    kept = F.apply(x, w)
    assert len(ops._EAGER_GRAPHS) == 1
    state.update(capturing=True)
    F.apply(x, w)                                   # the stream the graph was recorded on: autograd has nothing to wait for
    state.update(stream=2)
    F.apply(v, v)                                   # other leaves
    with pytest.raises(_lib.PgError, match="still alive"):
        F.apply(v, w)
    del kept
    assert len(ops._EAGER_GRAPHS) == 0
    F.apply(x, w)


# ---- dropout ---------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("n,d", [(1, 1), (1, 64), (3, 5), (257, 60), (100, 255), (100, 257), (33, 511), (33, 513), (700, 602), (40, 1030),
                                 (2, 9000)])
def test_dropout_vs_oracle(dev, hiplib, oracle, n, d, t):
    from pagraph_amd import ops
    g = gen(n * 1000 + d, dev)
    x = torch.randn(n, d, generator=g, device=dev).to(t).requires_grad_()
    gy = torch.randn(n, d, generator=g, device=dev).to(t)
    spec = spec_of(dev, 0.3)
    keep, scale = mask_of(oracle, n, d, spec, 5)
    keep = keep.to(dev)
    y = ops.dropout(x, spec)
    spec.step.add_(1)                                     # the gradient's mask is the forward's all the same
    gx, = torch.autograd.grad(y, x, gy)
    zero = torch.zeros((), dtype=t, device=dev)
    for got, src in ((y, x), (gx, gy)):
        want = torch.where(keep, (src.detach().float() * torch.tensor(scale, dtype=F32, device=dev)).to(t), zero)
        assert torch.equal(got.detach(), want)


@gpu
def test_dropout_layouts_and_edges(dev, hiplib, oracle):
    from pagraph_amd import _lib, ops
    spec = spec_of(dev, 0.5)
    base = torch.randn(41, 131, device=dev)
    want = ops.dropout(base[3:40, 5:90].contiguous(), spec)
    assert torch.equal(ops.dropout(base[3:40, 5:90], spec), want)                       # rows apart, off any alignment
    b16 = torch.randn(12, 77, device=dev).to(BF16)
    assert torch.equal(ops.dropout(b16[:, 3:70], spec), ops.dropout(b16[:, 3:70].contiguous(), spec))
    assert torch.equal(ops.dropout(base.t(), spec), ops.dropout(base.t().contiguous(), spec))
    row = torch.randn(1, 50, device=dev)
    assert torch.equal(ops.dropout(row.expand(9, 50), spec), ops.dropout(row.expand(9, 50).contiguous(), spec))
    x3 = torch.randn(4, 6, 20, device=dev)
    assert torch.equal(ops.dropout(x3, spec), ops.dropout(x3.view(24, 20), spec).view(4, 6, 20))
    v = torch.randn(30, device=dev)
    assert torch.equal(ops.dropout(v, spec), ops.dropout(v.view(1, 30), spec).view(30))
    e = torch.zeros(0, 8, device=dev, requires_grad=True)
    assert ops.dropout(e, spec).shape == (0, 8)
    assert torch.autograd.grad(ops.dropout(e, spec).sum(), e)[0].shape == (0, 8)
    host = ops.DropoutSpec(0.5, spec.seed, spec.tag, None, step_value=5)                # the step kept by the caller
    assert torch.equal(ops.dropout(base, host), ops.dropout(base, spec))
    bad = base.clone()
    bad[::2] = float("inf")
    keep, _ = mask_of(oracle, 41, 131, spec, 5)
    out = ops.dropout(bad, spec).cpu()
    assert (out[~keep] == 0).all() and torch.isinf(out[::2][keep[::2]]).all()
    with pytest.raises(_lib.PgError):
        ops.dropout(base.double(), spec)
    with pytest.raises(_lib.PgError):
        ops.dropout(base, ops.DropoutSpec(0.5, 1, 2, torch.tensor([1])))                # a step on the host
    with pytest.raises(_lib.PgError):
        ops.dropout(torch.zeros(3, 0, device=dev), spec)


@gpu
@pytest.mark.parametrize("d", [64, 600])
def test_dropout_is_the_aggregations_dropout(dev, hiplib, d):
    """aggregating dropped rows == dropping inside the aggregation, to the bit"""
    from pagraph_amd import ops
    n = 500
    g = gen(d, dev)
    h = torch.randn(n, d, generator=g, device=dev)
    indptr = torch.arange(0, 2 * 300 + 1, 2, dtype=torch.int32, device=dev)
    src = torch.randint(0, n, (600,), generator=g, device=dev).to(torch.int32)
    spec = spec_of(dev, 0.25)
    assert torch.equal(ops.block_aggregate(indptr, src, ops.dropout(h, spec), 300), ops.block_aggregate(indptr, src, h, 300, dropout=spec))


# ---- layer norm ------------------------------------------------------------------------------------------------------------
def norm_reference(x, w, b, eps, gy, gs=None):
    """(y, ds, dw, db) and what their bounds need, in 64 bits; x are the rows that are normalised"""
    x, gy = x.double(), gy.double()
    w = torch.ones(x.size(1), dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    gh = gy * w
    ds = rstd * (gh - gh.mean(1, keepdim=True) - xh * (gh * xh).mean(1, keepdim=True))
    # a row's sums: at most 32 additions in a lane, then 10 across lanes, for mean and variance: (x - mean) * rstd is off by
    # 2^-24 times 42 of the row's largest |x| * rstd for the mean, and by the variance's 2 * 42 and a few more relative to itself
    amp = x.abs().amax(1, keepdim=True) * rstd if x.size(0) else rstd
    exh = 128 * E * (1 + amp) * (1 + xh.abs())
    ey = exh * w.abs() + 4 * E * b.abs()
    top = gh.abs().amax(1, keepdim=True) if x.size(0) else rstd
    xtop = xh.abs().amax(1, keepdim=True) if x.size(0) else rstd
    eds = 256 * E * (1 + amp) * rstd * top * (1 + xtop) * (1 + xtop)
    if gs is not None:
        ds = ds + gs.double()
        eds = eds + 4 * E * ds.abs()
    return xh * w + b, ds, (gy * xh).sum(0), gy.sum(0), ey, eds, (gy.abs() * exh).sum(0), (gy * xh).abs().sum(0), gy.abs().sum(0)


def check_norm(dev, n, d, t, wt, residual=False, p=0.0, oracle=None, seed=0, shift=0.25):
    from pagraph_amd import ops
    g = gen(seed + n * 31 + d, dev)
    norm = torch.nn.LayerNorm(d, device=dev, dtype=wt)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.25 * torch.randn(d, generator=g, device=dev))
        norm.bias.copy_(0.25 * torch.randn(d, generator=g, device=dev))
    x = (torch.randn(n, d, generator=g, device=dev) * 1.5 + shift).to(t).requires_grad_()
    gy = torch.randn(n, d, generator=g, device=dev).to(t)
    leaves = [x, norm.weight, norm.bias]
    if residual:
        res = torch.randn(n, d, generator=g, device=dev).to(t).requires_grad_()
        gs = torch.randn(n, d, generator=g, device=dev).to(t)
        spec = spec_of(dev, p) if p else None
        y, s = ops.layer_norm(x, norm, residual=res, dropout=spec)
        if spec is not None:
            spec.step.add_(3)
        dx, dw, db, dres = torch.autograd.grad((y, s), leaves + [res], (gy, gs))
        m = torch.ones(n, d, dtype=torch.float64, device=dev)
        if p:
            keep, scale = mask_of(oracle, n, d, spec, 5)
            m = keep.to(dev).double() * scale
        close(s, x.detach().double() * m + res.detach().double(), 2 * E * (x.detach().double() * m).abs(), "sum")
        rows = s.detach()
    else:
        gs, m, rows = None, None, x.detach()
        y = ops.layer_norm(x, norm)
        dx, dw, db = torch.autograd.grad(y, leaves, gy)
    ry, rds, rdw, rdb, ey, eds, exw, sw, sb = norm_reference(rows, norm.weight.detach(), norm.bias.detach(), norm.eps, gy, gs)
    # rows a lane group walks (<= 512 workgroups, or one row a group where fewer), the waves, then 32 + 16 partial rows
    adds = n / 512 + 80
    close(y, ry, ey, "y")
    if residual:
        close(dres, rds, eds, "dres")
        close(dx, rds * m, eds * m + 2 * E * (rds * m).abs(), "dx")
    else:
        close(dx, rds, eds, "dx")
    close(dw, rdw, exw + adds * E * sw, "dw")
    close(db, rdb, adds * E * sb, "db")
    assert dw.dtype == wt and db.dtype == wt and dx.dtype == t and y.dtype == t


@gpu
@pytest.mark.parametrize("n,d", [(1, 2), (3, 1), (5, 7), (1, 64), (300, 64), (2, 65), (77, 128), (1001, 60), (9, 129), (13, 255), (13, 257),
                                 (7, 512), (7, 513), (1200, 602), (3, 1024), (3, 1025), (40, 2048), (5, 2049), (2, 4096), (3, 4100),
                                 (2, 8192), (3, 8193), (600, 2500), (1, 32768), (2, 20001)])
def test_layer_norm_vs_64_bits(dev, hiplib, n, d):
    check_norm(dev, n, d, F32, F32)


@gpu
@pytest.mark.parametrize("t,wt", [(BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("n,d", [(1, 33), (64, 64), (700, 602), (5, 1111), (4, 4096), (2, 9001)])
def test_layer_norm_types(dev, hiplib, n, d, t, wt):
    check_norm(dev, n, d, t, wt)


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("n,d", [(1, 5), (200, 64), (90, 259), (500, 602), (17, 2048), (6, 5000), (2, 16500)])
def test_layer_norm_with_residual(dev, hiplib, oracle, n, d, p, t):
    check_norm(dev, n, d, t, t, residual=True, p=p, oracle=oracle)


@gpu
def test_layer_norm_of_far_rows(dev, hiplib):
    """a mean a thousand times the spread: the variance is taken of centred values"""
    check_norm(dev, 40, 600, F32, F32, shift=1500.0)


@gpu
def test_layer_norm_many_rows_twice_the_same(dev, hiplib):
    from pagraph_amd import ops
    x = torch.randn(40000, 48, device=dev, requires_grad=True)
    norm = torch.nn.LayerNorm(48, device=dev)
    gy = torch.randn(40000, 48, device=dev)
    check_norm(dev, 40000, 48, F32, F32)
    a = torch.autograd.grad(ops.layer_norm(x, norm), [x, norm.weight, norm.bias], gy)
    b = torch.autograd.grad(ops.layer_norm(x, norm), [x, norm.weight, norm.bias], gy)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@gpu
def test_layer_norm_layouts_and_edges(dev, hiplib):
    from pagraph_amd import ops
    norm = torch.nn.LayerNorm(85, device=dev)
    base = torch.randn(41, 131, device=dev)
    view, flat = base[3:40, 5:90], base[3:40, 5:90].contiguous()
    assert torch.equal(ops.layer_norm(view, norm), ops.layer_norm(flat, norm))
    assert torch.equal(ops.layer_norm(flat.view(37, 1, 85), norm), ops.layer_norm(flat, norm).view(37, 1, 85))
    tr = torch.randn(85, 20, device=dev)
    assert torch.equal(ops.layer_norm(tr.t(), norm), ops.layer_norm(tr.t().contiguous(), norm))
    res = torch.randn(41, 90, device=dev)[2:39, 1:86]
    got, want = ops.layer_norm(view, norm, residual=res), ops.layer_norm(flat, norm, residual=res.contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # gradients that come in as one row, or transposed
    x = flat.clone().requires_grad_()
    row = torch.randn(1, 85, device=dev)
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x, norm), x, row.expand(37, 85))[0],
                       torch.autograd.grad(ops.layer_norm(x, norm), x, row.expand(37, 85).contiguous())[0])
    gt = torch.randn(85, 37, device=dev).t()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x, norm), x, gt)[0],
                       torch.autograd.grad(ops.layer_norm(x, norm), x, gt.contiguous())[0])
    # weight, bias or both absent
    for kw in ({"elementwise_affine": False}, {"bias": False}):
        m = torch.nn.LayerNorm(85, device=dev, **kw)
        y = ops.layer_norm(x, m)
        ry, rds = norm_reference(flat, m.weight.detach() if m.weight is not None else None, None, m.eps, torch.ones_like(flat))[:2]
        assert (y.double() - ry).abs().max() < 1e-5
        y.sum().backward()
        assert (x.grad.double() - rds).abs().max() < 1e-5
        x.grad = None
    # one output used, or none of the parameters wanted
    rs = res.contiguous().requires_grad_()
    y, s = ops.layer_norm(x, norm, residual=rs)
    gx, = torch.autograd.grad(s.sum(), x)
    assert (gx == 1).all()
    y, s = ops.layer_norm(x, norm, residual=rs)
    g1, g2 = torch.autograd.grad((y * y).sum(), [x, rs])
    assert torch.equal(g1, g2) and torch.isfinite(g1).all()
    # no rows; a constant row; a row that holds a NaN changes no other
    e = torch.zeros(0, 85, device=dev, requires_grad=True)
    ge = torch.autograd.grad(ops.layer_norm(e, norm).sum(), [e, norm.weight, norm.bias])
    assert ge[0].shape == (0, 85) and (ge[1] == 0).all() and (ge[2] == 0).all()
    c = torch.full((2, 85), 3.0, device=dev)
    assert torch.equal(ops.layer_norm(c, norm), norm.bias.detach().expand(2, 85))
    bad = flat.clone()
    bad[5, 7], bad[9, 0] = float("nan"), float("inf")
    y, good = ops.layer_norm(bad, norm), ops.layer_norm(flat, norm)
    keep = torch.ones(37, dtype=torch.bool, device=dev)
    keep[[5, 9]] = False
    assert torch.equal(y[keep], good[keep]) and torch.isnan(y[5]).all() and torch.isnan(y[9]).all()


@gpu
def test_layer_norm_refusals(dev, hiplib):
    from pagraph_amd import _lib, ops
    x = torch.randn(4, 16, device=dev)
    spec = spec_of(dev, 0.5)
    bad = [lambda: ops.layer_norm(x, torch.nn.LayerNorm(8, device=dev)), lambda: ops.layer_norm(x, torch.nn.LayerNorm((4, 16), device=dev)),
           lambda: ops.layer_norm(x, torch.nn.LayerNorm(16)), lambda: ops.layer_norm(x.double(), torch.nn.LayerNorm(16, device=dev).double()),
           lambda: ops.layer_norm(x, torch.nn.LayerNorm(16, device=dev, dtype=BF16)),
           lambda: ops.layer_norm(x, torch.nn.LayerNorm(16, device=dev), dropout=spec),
           lambda: ops.layer_norm(x, torch.nn.LayerNorm(16, device=dev), residual=x[:1]),
           lambda: ops.layer_norm(x, torch.nn.LayerNorm(16, device=dev), residual=x.half()),
           lambda: ops.layer_norm(torch.zeros(1, 32769, device=dev), torch.nn.LayerNorm(32769, device=dev))]
    for f in bad:
        with pytest.raises(_lib.PgError):
            f()


# ---- the wide class head's loss --------------------------------------------------------------------------------------------
def head(dev, K, C, t, g, bias=True, scale=2.0):
    lin = torch.nn.Linear(K, C, bias=bias, device=dev, dtype=t)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(C, K, generator=g, device=dev) * (scale / K ** 0.5))
        if bias:
            lin.bias.copy_(torch.randn(C, generator=g, device=dev) * 0.5)
    return lin


def xent_reference(h, lin, lab, up):
    """row losses, and for row factors `up` (d objective / d row loss): dh, dw, db, with bounds for the roundings on the way"""
    t = h.dtype
    n, K = h.shape
    C = lin.weight.size(0)
    H, W = h.detach().double(), lin.weight.detach().double()
    b = lin.bias.detach().double() if lin.bias is not None else torch.zeros(C, dtype=torch.float64, device=h.device)
    ok = (lab >= 0) & (lab < C)
    H = torch.where(ok.view(-1, 1), H, torch.zeros_like(H))
    at = torch.where(ok, lab, torch.zeros_like(lab)).view(-1, 1)
    z = H @ W.t() + b
    top = z.amax(1, keepdim=True) if n else z[:, :1]
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    zero = torch.zeros(n, dtype=torch.float64, device=h.device)
    loss = torch.where(ok, (lse - z.gather(1, at)).view(-1), zero)
    # a logit: K products, each exact to 2^-22 at worst (fp32 in three bf16 parts drops x1 y2 + x2 y1 + x2 y2 < 2^-22.9 |x y|, 16-bit
    # products are exact), K + 8 additions
    mag = H.abs() @ W.abs().t() + torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b))
    ez = (K + 16) * E * (mag.amax(1) if n else zero) if n else zero
    # the sum of exponentials: exp2 and the scaled argument (|z - max| <= 128 counts), 128 in a tile's order, then tiles / 64 + 8
    eexp = 256 * E + (C / 8192 + 80) * E
    eloss = torch.where(ok, 2 * ez + eexp + 8 * E * (lse.view(-1).abs() + loss.abs()), zero)
    P = torch.exp(z - lse)
    G = P.clone()
    G.scatter_add_(1, at, torch.full((n, 1), -1.0, dtype=torch.float64, device=h.device))
    f = torch.where(ok, up.double(), zero).view(-1, 1)
    G = torch.where(f != 0, G * f, torch.zeros_like(G))
    # an element of G: the exponential's argument is off by the logit and the lse; then one rounding to its type (fp32 G: one to
    # 32 bits and the parts' 2^-24); fp16 keeps steps of 2^-24 below its normal range, of values times 2^14: 2^-38 per unit
    eG = (P * f.abs()) * (2 * ez + eexp + 160 * E + 8 * E * lse.view(-1).abs()).view(-1, 1) + G.abs() * (half_step(t) if t != F32 else 4 * E)
    if t == F16:
        eG = eG + f.abs().max() * 2.0 ** -38 if n else eG
    # an exponential below the smallest normal number, 2^-126, comes out as 0, and so may the second and third bf16 parts of an
    # fp32 value (each at most 2^-8 of the one before: below 2^-126 wherever they are lost): off by less than 3 * 2^-126
    eG = eG + 3 * 2.0 ** -126 * (1 + f.abs())
    eG = torch.where(f != 0, eG, torch.zeros_like(eG))
    return {"loss": loss, "eloss": eloss, "ok": ok,
            "dh": G @ W, "edh": eG @ W.abs() + (G.abs() @ W.abs()) * (C + 32) * E,
            "dw": G.t() @ H, "edw": eG.t() @ H.abs() + (G.abs().t() @ H.abs()) * (n + 32) * E,
            "db": G.sum(0), "edb": eG.sum(0) + G.abs().sum(0) * (n + 32) * E}


def check_xent(dev, n, K, C, t, ignored=0.0, reduction="mean", bias=True, seed=0, h=None, lab=None, lin=None, ignore_index=-100):
    from pagraph_amd import ops
    g = gen(seed + n * 7 + K * 3 + C, dev)
    if lin is None:
        lin = head(dev, K, C, t, g, bias)
    if h is None:
        h = torch.randn(n, K, generator=g, device=dev).to(t)
    if lab is None:
        lab = torch.randint(0, C, (n,), generator=g, device=dev)
        skip = torch.rand(n, generator=g, device=dev) < ignored
        lab = torch.where(skip, torch.full_like(lab, ignore_index), lab)
    h = h.detach().requires_grad_()
    loss = ops.linear_cross_entropy(h, lin, lab, ignore_index=ignore_index, reduction=reduction)
    assert loss.dtype == F32
    seen = torch.where(lab == ignore_index, torch.full_like(lab, -1), lab)
    count = int(((seen >= 0) & (seen < C)).sum())
    if reduction == "none":
        up = torch.randn(n, generator=g, device=dev)
        up[::5] = 0.0
        grads = torch.autograd.grad(loss, [h] + list(lin.parameters()), up)
    else:
        k = 0.75
        up = torch.full((n,), k / max(count, 1) if reduction == "mean" else k, dtype=torch.float64, device=dev)
        grads = torch.autograd.grad(loss * k, [h] + list(lin.parameters()))
    ref = xent_reference(h, lin, seen, up)
    if reduction == "none":
        close(loss, ref["loss"], ref["eloss"], "loss")
    else:
        adds = n / 1024 + 16                                                       # the row losses' sum in one workgroup
        total = ref["loss"].sum()
        e = ref["eloss"].sum() + adds * E * ref["loss"].abs().sum()
        if reduction == "mean":
            total, e = (total / count, e / count + 2 * E * total.abs() / count) if count else (torch.full_like(total, float("nan")), e)
        close(loss, total, e, "loss")
    factor = 4 * E                                                                 # g * 1 / #rows, and the product with it
    for name, got in zip(("dh", "dw", "db"), grads):
        close(got, ref[name], ref["e" + name] + factor * ref[name].abs(), name)
    assert (grads[0][~ref["ok"]] == 0).all()
    return loss, grads


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("n,K,C", [(1, 1, 1), (1, 64, 1000), (2, 3, 5), (63, 16, 61), (64, 64, 128), (65, 65, 129), (300, 64, 172),
                                   (130, 602, 257), (777, 100, 1153), (1500, 33, 300), (128, 1024, 1024), (5, 7, 5000), (2000, 130, 70)])
def test_linear_cross_entropy_vs_64_bits(dev, hiplib, n, K, C, t):
    check_xent(dev, n, K, C, t, ignored=0.1 if n > 4 else 0.0)


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("bias", [True, False])
def test_linear_cross_entropy_reductions(dev, hiplib, t, reduction, bias):
    check_xent(dev, 333, 48, 500, t, ignored=0.2, reduction=reduction, bias=bias)


@gpu
@pytest.mark.parametrize("n,K,C,t", [(4099, 40, 20011, F32), (4099, 40, 20011, BF16), (4099, 131, 11003, F32), (4099, 260, 33001, BF16),
                                     (300, 300, 9000, F16), (2500, 520, 4097, BF16), (1300, 1030, 2050, F32),
                                     (8201, 131, 11003, F32), (8201, 260, 33001, BF16), (4099, 1030, 8200, BF16), (3000, 1030, 6001, F16),
                                     (8201, 300, 11003, F32)])
def test_linear_cross_entropy_large(dev, hiplib, n, K, C, t):
    """several splits of the classes and rows, several pieces of the vocabulary with a ragged last one, large and small tiles"""
    check_xent(dev, n, K, C, t, ignored=0.05)


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("K", [64, 128, 192, 256, 320])
def test_linear_cross_entropy_every_row_width(dev, hiplib, K, t):
    """rows that fill their padding exactly, read in place where the type allows, and one column less"""
    check_xent(dev, 150, K, 700, t)
    check_xent(dev, 150, K - 1, 700, t, ignored=0.3)
    check_xent(dev, 90, K, 321, t, reduction="none")


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_linear_cross_entropy_ignored_rows(dev, hiplib, t):
    from pagraph_amd import ops
    g = gen(11, dev)
    n, K, C = 200, 72, 300
    lin = head(dev, K, C, t, g)
    h = torch.randn(n, K, generator=g, device=dev).to(t)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    lab[::3], lab[1::7], lab[50] = -100, C, -5                      # the ignored index, labels out of range
    clean = check_xent(dev, n, K, C, t, h=h, lab=lab, lin=lin)
    # what ignored rows hold does not matter, not even NaN
    dirty = h.clone()
    dirty[::3], dirty[1::7], dirty[50] = float("nan"), float("inf"), float("-inf")
    dirty.requires_grad_()
    loss = ops.linear_cross_entropy(dirty, lin, lab)
    grads = torch.autograd.grad(loss, [dirty, lin.weight, lin.bias])
    ref = ops.linear_cross_entropy(h.requires_grad_(), lin, lab)
    want = torch.autograd.grad(ref, [h, lin.weight, lin.bias])
    assert torch.equal(loss, ref) and all(torch.equal(a, b) for a, b in zip(grads, want))
    # no row counts: a mean over nothing, gradients of zero
    none = torch.full_like(lab, 9)
    x = dirty.detach().requires_grad_()
    loss = ops.linear_cross_entropy(x, lin, none, ignore_index=9)
    grads = torch.autograd.grad(loss, [x, lin.weight, lin.bias])
    assert torch.isnan(loss) and all((q == 0).all() for q in grads)
    assert ops.linear_cross_entropy(x, lin, none, ignore_index=9, reduction="sum") == 0
    # no row at all
    e = torch.zeros(0, K, dtype=t, device=dev, requires_grad=True)
    le = torch.zeros(0, dtype=torch.int64, device=dev)
    loss = ops.linear_cross_entropy(e, lin, le)
    assert torch.isnan(loss) and ops.linear_cross_entropy(e, lin, le, reduction="none").shape == (0,)
    grads = torch.autograd.grad(loss, [e, lin.weight, lin.bias])
    assert grads[0].shape == (0, K) and all((q == 0).all() for q in grads)


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_linear_cross_entropy_masked_classes_and_extremes(dev, hiplib, t):
    """classes that a bias of -inf or of the type's lowest value takes out, a whole tile of them too; logits far apart"""
    g = gen(5, dev)
    n, K, C = 70, 24, 520
    lin = head(dev, K, C, t, g)
    with torch.no_grad():
        lin.bias[128:256] = float("-inf")
        lin.bias[3], lin.bias[519] = float("-inf"), torch.finfo(t).min
    lab = torch.randint(256, 500, (n,), generator=g, device=dev)
    loss, grads = check_xent(dev, n, K, C, t, lab=lab, lin=lin)
    assert (grads[1][128:256] == 0).all() and (grads[2][3] == 0) and (grads[2][519] == 0)
    big = head(dev, K, C, t, g, scale=60.0)
    check_xent(dev, n, K, C, t, lab=lab, lin=big)
    # the label's own class masked: that row's loss is infinite, as in ops.cross_entropy
    from pagraph_amd import ops
    lab2 = lab.clone()
    lab2[4] = 200
    each = ops.linear_cross_entropy(torch.randn(n, K, generator=g, device=dev).to(t), lin, lab2, reduction="none")
    assert each[4] == float("inf") and torch.isfinite(each[:4]).all() and torch.isfinite(each[5:]).all()


@gpu
def test_linear_cross_entropy_matches_the_given_logits_loss(dev, hiplib):
    """ops.cross_entropy over the head's logits is the same loss"""
    from pagraph_amd import ops
    g = gen(3, dev)
    lin = head(dev, 64, 172, F32, g)
    h = torch.randn(600, 64, generator=g, device=dev, requires_grad=True)
    lab = torch.randint(0, 172, (600,), generator=g, device=dev)
    lab[::9] = -100
    a, b = ops.linear_cross_entropy(h, lin, lab), ops.cross_entropy(lin(h), lab)
    assert abs(a.item() - b.item()) < 2e-6 * abs(b.item())
    for u, v in zip(torch.autograd.grad(a, [h, lin.weight, lin.bias]), torch.autograd.grad(b, [h, lin.weight, lin.bias])):
        assert (u - v).abs().max() <= 2e-6 * v.abs().max()


@gpu
def test_linear_cross_entropy_layouts_and_parts(dev, hiplib):
    from pagraph_amd import ops
    g = gen(8, dev)
    for t in (F32, BF16, F16):
        lin = head(dev, 50, 333, t, g)
        wide = torch.randn(100, 131, generator=g, device=dev).to(t)
        lab = torch.randint(0, 333, (100,), generator=g, device=dev)
        flat = wide[:, 7:57].contiguous()
        want = torch.autograd.grad(ops.linear_cross_entropy(flat.requires_grad_(), lin, lab), [flat, lin.weight, lin.bias])
        v = wide[:, 7:57].detach().requires_grad_()
        got = torch.autograd.grad(ops.linear_cross_entropy(v, lin, lab), [v, lin.weight, lin.bias])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        x3 = flat.detach().view(4, 25, 50).requires_grad_()
        got = torch.autograd.grad(ops.linear_cross_entropy(x3, lin, lab.view(4, 25)), [x3, lin.weight, lin.bias])
        assert torch.equal(got[0].view(100, 50), want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert ops.linear_cross_entropy(x3, lin, lab.view(4, 25), reduction="none").shape == (4, 25)
        # a weight that is a view of a larger table
        table = torch.randn(333, 80, generator=g, device=dev).to(t)
        holder = torch.nn.Linear(50, 333, device=dev, dtype=t)
        holder.weight = torch.nn.Parameter(table[:, 11:61])
        holder.bias = torch.nn.Parameter(lin.bias.detach().clone())
        packed = torch.nn.Linear(50, 333, device=dev, dtype=t)
        packed.weight, packed.bias = torch.nn.Parameter(table[:, 11:61].contiguous()), holder.bias
        a = torch.autograd.grad(ops.linear_cross_entropy(flat, holder, lab), [flat, holder.weight, holder.bias])
        b = torch.autograd.grad(ops.linear_cross_entropy(flat, packed, lab), [flat, packed.weight, packed.bias])
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        # a single gradient wanted
        for which in range(3):
            leaf = [flat, lin.weight, lin.bias]
            for i, q in enumerate(leaf):
                q.requires_grad_(i == which)
            one, = torch.autograd.grad(ops.linear_cross_entropy(flat, lin, lab), leaf[which])
            assert torch.equal(one, want[which])
            for q in leaf:
                q.requires_grad_(True)


@gpu
def test_outputs_are_the_callers(dev, hiplib):
    """outputs may be changed in place; inputs that a gradient needs may not (autograd says so); a second pass over a kept graph is
    the first; a gradient's own graph is refused"""
    from pagraph_amd import _lib, ops
    g = gen(14, dev)
    lin, norm, spec = head(dev, 24, 90, F32, g), torch.nn.LayerNorm(24, device=dev), spec_of(dev, 0.5)
    lab = torch.randint(0, 90, (40,), generator=g, device=dev)
    for f in (lambda x: ops.linear_cross_entropy(x, lin, lab), lambda x: ops.linear_cross_entropy(x, lin, lab, reduction="none"),
              lambda x: ops.layer_norm(x, norm), lambda x: ops.dropout(x, spec), lambda x: ops.layer_norm(x, norm, residual=x, dropout=spec)[0]):
        x = torch.randn(40, 24, generator=g, device=dev, requires_grad=True)
        y = f(x)
        a = torch.autograd.grad(y.sum(), x, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(y.sum(), x, retain_graph=True)[0], a)
        with pytest.raises(_lib.PgError):
            torch.autograd.grad(y.sum(), x, create_graph=True)
        z = f(x)
        z.mul_(2.0)
        assert torch.equal(torch.autograd.grad(z.sum(), x)[0], torch.autograd.grad((2.0 * f(x)).sum(), x)[0])
    loss = ops.linear_cross_entropy(x, lin, lab)
    lab.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    y, s = ops.layer_norm(x, norm, residual=x)
    s.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("K", [40, 300])
def test_linear_cross_entropy_gradients_that_are_not_finite(dev, hiplib, K, t):
    """an infinite or NaN gradient of one row's loss stays with that row, and is not lost where it is the only one"""
    from pagraph_amd import ops
    g = gen(17, dev)
    lin = head(dev, K, 700, t, g)
    h = torch.randn(60, K, generator=g, device=dev).to(t).requires_grad_()
    lab = torch.randint(0, 700, (60,), generator=g, device=dev)
    up = torch.randn(60, generator=g, device=dev)
    rest = torch.ones(60, dtype=torch.bool, device=dev)
    rest[7], rest[33] = False, False
    clean = torch.where(rest, up, torch.zeros_like(up))
    want, = torch.autograd.grad(ops.linear_cross_entropy(h, lin, lab, reduction="none"), h, clean)
    for a, b in ((float("nan"), float("inf")), (float("-inf"), float("inf"))):
        dirty = up.clone()
        dirty[7], dirty[33] = a, b
        dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, lin, lab, reduction="none"), [h, lin.weight], dirty)
        assert torch.equal(dh[rest], want[rest])
        assert not torch.isfinite(dh[~rest]).any() and not torch.isfinite(dw).any()
    dh, = torch.autograd.grad(ops.linear_cross_entropy(h, lin, lab, reduction="none"), h, torch.full_like(up, float("nan")))
    assert torch.isnan(dh).all()


@gpu
def test_linear_cross_entropy_refusals(dev, hiplib):
    from pagraph_amd import _lib, ops
    h, lin = torch.randn(6, 16, device=dev), torch.nn.Linear(16, 100, device=dev)
    lab = torch.zeros(6, dtype=torch.int64, device=dev)
    bad = [lambda: ops.linear_cross_entropy(h[:, :8], lin, lab), lambda: ops.linear_cross_entropy(h.half(), lin, lab),
           lambda: ops.linear_cross_entropy(h, lin, lab.int()), lambda: ops.linear_cross_entropy(h, lin, lab[:5]),
           lambda: ops.linear_cross_entropy(h, lin, lab.cpu()), lambda: ops.linear_cross_entropy(h, torch.nn.Linear(16, 100), lab),
           lambda: ops.linear_cross_entropy(h, lin, lab, reduction="max"), lambda: ops.linear_cross_entropy(h.double(), lin.double(), lab)]
    for f in bad:
        with pytest.raises(_lib.PgError):
            f()


# ---- together --------------------------------------------------------------------------------------------------------------
class Tail(torch.nn.Module):
    """dropout -> residual + norm -> wide class head's loss, as a model would end"""

    def __init__(self, d, C, dev):
        super().__init__()
        self.inner, self.norm, self.head = torch.nn.Linear(d, d, device=dev), torch.nn.LayerNorm(d, device=dev), torch.nn.Linear(d, C, device=dev)

    def forward(self, x, lab, s1, s2):
        from pagraph_amd import ops
        y = torch.relu(self.inner(ops.dropout(x, s1)))
        y, total = ops.layer_norm(y, self.norm, residual=x, dropout=s2)
        return ops.linear_cross_entropy(y + 0.1 * total, self.head, lab)


def tail_reference(m, x, lab, k1, k2):
    """the same in 64 bits, masks given; returns loss and gradients of x and every parameter"""
    ps = {k: v.detach().double().requires_grad_() for k, v in m.named_parameters()}
    x = x.detach().double().requires_grad_()
    y = torch.relu((x * k1) @ ps["inner.weight"].t() + ps["inner.bias"])
    s = y * k2 + x
    yn = torch.nn.functional.layer_norm(s, (s.size(1),), ps["norm.weight"], ps["norm.bias"], m.norm.eps)
    z = (yn + 0.1 * s) @ ps["head.weight"].t() + ps["head.bias"]
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    ok = lab >= 0
    loss = -(logp.gather(1, lab.clamp(min=0).view(-1, 1)).view(-1) * ok).sum() / ok.sum()
    return loss, torch.autograd.grad(loss, [x] + list(ps.values()))


@gpu
def test_tail_against_64_bits_and_differences(dev, hiplib, oracle):
    g = gen(21, dev)
    n, d, C = 90, 60, 230
    m = Tail(d, C, dev)
    x = torch.randn(n, d, generator=g, device=dev, requires_grad=True)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    lab[::11] = -100
    s1, s2 = spec_of(dev, 0.2, tag=1), spec_of(dev, 0.4, tag=2)
    k1, k2 = [(lambda km: km[0].to(dev).double() * km[1])(mask_of(oracle, n, d, s, 5)) for s in (s1, s2)]
    loss = m(x, lab, s1, s2)
    grads = torch.autograd.grad(loss, [x] + list(m.parameters()))
    rl, rg = tail_reference(m, x, lab, k1, k2)
    # four fp32 products of depth <= 230 one behind the other: 230 * 2^-24 each relative to sums of absolute values that are at
    # most some ten times the largest gradient
    tol = 4 * 230 * E * 10
    assert abs(loss.item() - rl.item()) <= tol * abs(rl.item())
    for a, b in zip(grads, rg):
        assert (a.double() - b).abs().max() <= tol * b.abs().max()
    # differences along a random direction, of the kernels' own losses: (f(+e) - f(-e)) / 2e is off by e^2 f''' / 6 and by the
    # losses' own roundings (their tolerance above) / e
    with torch.no_grad():
        for p, gp in zip([x] + list(m.parameters()), grads):
            v = torch.randn(p.shape, generator=g, device=dev)
            v /= v.norm()
            e, old = 2e-2, p.detach().clone()
            p.copy_(old + e * v)
            up = m(x, lab, s1, s2).item()
            p.copy_(old - e * v)
            down = m(x, lab, s1, s2).item()
            p.copy_(old)
            along = (gp * v).sum().item()
            assert abs((up - down) / (2 * e) - along) <= tol * abs(rl.item()) / e + e * e * (1 + gp.norm().item())


@gpu
def test_tail_captured_and_replayed(dev, hiplib):
    """a training step of the three captured into a graph on its own stream, replayed on new data with eager work in between, against
    the eager step; the step counter is advanced inside"""
    g = gen(33, dev)
    n, d, C = 300, 64, 900
    m = Tail(d, C, dev)
    x = torch.randn(n, d, generator=g, device=dev)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    s1, s2 = spec_of(dev, 0.2, tag=1), spec_of(dev, 0.4, tag=2)
    s2.step = s1.step
    params = list(m.parameters())

    def step():
        s1.step.add_(1)
        loss = m(x, lab, s1, s2)
        return [loss.detach()] + list(torch.autograd.grad(loss, params))
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.copy_(torch.randn(n, d, generator=g, device=dev))
        lab.copy_(torch.randint(0, C, (n,), generator=g, device=dev))
        lab[:k] = -100
        s1.step.fill_(100 + k)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        s1.step.fill_(100 + k)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@gpu
def test_capture_is_refused_while_an_eager_graph_lives(dev, hiplib):
    from pagraph_amd import _lib, ops
    g = gen(55, dev)
    lin, x = head(dev, 32, 200, F32, g), torch.randn(50, 32, generator=g, device=dev)
    lab = torch.randint(0, 200, (50,), generator=g, device=dev)

    def step():
        loss = ops.linear_cross_entropy(x, lin, lab)
        return [loss.detach()] + list(torch.autograd.grad(loss, [lin.weight, lin.bias]))
    want = step()
    kept = ops.linear_cross_entropy(x, lin, lab)
    with pytest.raises(_lib.PgError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    torch.cuda.synchronize()
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step()


@gpu
@pytest.mark.parametrize("shape", [(24,), (5, 24), (2, 3, 24)])
def test_outputs_of_any_rank_may_be_changed_in_place(dev, hiplib, shape):
    from pagraph_amd import ops
    norm, spec = torch.nn.LayerNorm(24, device=dev), spec_of(dev, 0.5)
    for f in (lambda x: ops.dropout(x, spec), lambda x: ops.layer_norm(x, norm), lambda x: ops.layer_norm(x, norm, residual=x)[0]):
        x = torch.randn(shape, device=dev, requires_grad=True)
        y = f(x)
        assert y.shape == x.shape
        want, = torch.autograd.grad((3.0 * f(x)).sum(), x)
        y.mul_(3.0)
        got, = torch.autograd.grad(y.sum(), x)
        assert got.shape == x.shape and torch.equal(got, want)


@gpu
def test_both_summands_keep_gradients_of_their_own(dev, hiplib):
    """x and the residual get the same values in different memory, also where rows have leading dimensions"""
    from pagraph_amd import ops
    norm = torch.nn.LayerNorm(24, device=dev)
    for shape in ((6, 24), (2, 3, 24), (2, 1, 3, 24)):
        x = torch.randn(shape, device=dev, requires_grad=True)
        r = torch.randn(shape, device=dev, requires_grad=True)
        once = None
        for k in range(3):
            y, total = ops.layer_norm(x, norm, residual=r)
            (y * y * y + total).sum().backward()
            if once is None:
                once = x.grad.clone()
                assert x.grad.data_ptr() != r.grad.data_ptr()
            want = once if k == 0 else want + once
            assert torch.equal(x.grad, want) and torch.equal(r.grad, want)


@gpu
def test_capture_without_gradients_beside_an_eager_graph(dev, hiplib):
    """an evaluation that records no graph may be captured whatever graphs of the same parameters live"""
    from pagraph_amd import ops
    g = gen(56, dev)
    lin, norm = head(dev, 32, 200, F32, g), torch.nn.LayerNorm(32, device=dev)
    x = torch.randn(50, 32, generator=g, device=dev, requires_grad=True)
    lab = torch.randint(0, 200, (50,), generator=g, device=dev)
    spec = spec_of(dev, 0.3)

    def run():
        return ops.linear_cross_entropy(ops.layer_norm(ops.dropout(x, spec), norm), lin, lab)
    kept = run()
    with torch.no_grad():
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kept)
    assert len(torch.autograd.grad(kept, [x, lin.weight, lin.bias, norm.weight, norm.bias])) == 5


@gpu
def test_two_streams_at_once(dev, hiplib):
    """two steps on two streams at the same time share nothing"""
    g = gen(44, dev)
    ms = [Tail(64, 700, dev) for _ in range(2)]
    xs = [torch.randn(2000, 64, generator=g, device=dev) for _ in range(2)]
    lab = torch.randint(0, 700, (2000,), generator=g, device=dev)
    spec = spec_of(dev, 0.3)

    def step(i):
        loss = ms[i](xs[i], lab, spec, spec)
        return [loss.detach()] + list(torch.autograd.grad(loss, list(ms[i].parameters())))
    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
