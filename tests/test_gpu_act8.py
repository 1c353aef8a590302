"""8-bit activation checkpoints and residual norms against plain 64-bit statements (tests/act8_reference.py).

Bounds, with u = 2^-24 (half a step of fp32) and half steps of 2^-8 for bf16, 2^-4 for e4m3 (and 2^-10 scales below its normal
range; a scale is under amax / 224):
  * packing is exact: same codes, same scale bytes
  * a sum over d columns is at most 24 additions in a lane, 6 over the wave and 3 over the waves: 40 u of the sum of magnitudes
  * GELU: the kernels' erf is off by 1.5e-7, half of it in the cdf, and a few roundings: 5e-7 |z| (6e-7 |dg| for the derivative)
  * sums over rows: one lane adds rows / (4 blocks) <= 64 of them, the second kernel 64 partial rows in a thread and 16 of those: 160 u
"""
import pytest
import torch

import act8_reference as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from vita_amd import ops as _ops
    return _ops


def rows_of(rows, d, dtype, scale, seed, step=8, junk=True):
    """[rows, d] on padded rows; the pads hold NaN, which nothing may read."""
    g = torch.Generator().manual_seed(seed)
    base = torch.full((rows, -(-d // step) * step), float("nan") if junk else 0.0, dtype=dtype)
    base[:, :d] = (torch.randn(rows, d, generator=g) * scale).to(dtype)
    return base.cuda()[:, :d]


def close(got, ref, tol, what=""):
    got = got.detach().cpu().double()
    bad = (got - ref).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), (got - ref).abs()[bad].max().item(), tol[bad].min().item() if torch.is_tensor(tol) else tol)
    assert torch.isfinite(got).all(), what


def zero_pads(t, d):
    assert torch.count_nonzero(t[:, d:]) == 0


SHAPES = [(1, 1), (1, 7), (3, 31), (2, 32), (5, 33), (7, 64), (37, 129), (1, 1025), (130, 1025), (65, 1088), (9, 2050), (3, 4100), (2, 8191)]


# ------------------------------------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_pack_is_exact(ops, rows, d, dtype):
    x = rows_of(rows, d, dtype, 1.5, rows + d)
    x[0, : d // 2] *= 1e-3                           # groups of different sizes, and one with a lone large value
    x[-1, d - 1] = 300.0
    a = ops.act8_pack(x)
    ref, scale = R.quantise(x.cpu())
    assert torch.equal(a.scale.view(torch.uint8).cpu(), scale)
    assert torch.equal(R.values(a), ref)
    assert torch.count_nonzero(a.q.view(torch.uint8)[:, d:]) == 0
    for out_dtype in (BF16, F32):
        y = ops.act8_unpack(a, dtype=out_dtype, ldo=(d + 63) // 64 * 64)
        assert torch.equal(y[:, :d].cpu().double(), ref)
        zero_pads(y, d)


def test_pack_borders(ops):
    """Ties, group maxima next to 1.75 * 2^k, signed zeros, denormals, the largest and smallest floats, NaN and infinities."""
    inf, nan = float("inf"), float("nan")
    big, tiny = torch.finfo(F32).max, 2.0 ** -149
    up = lambda v: torch.nextafter(torch.tensor(v), torch.tensor(inf)).item()
    rows = [
        [448.0, 17.0, 19.0, 18.0, 1.0625, 1.1875, -17.0, -0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, up(2.0 ** -10), 2.0 ** -11],
        [1.75, 1.0, 0.1], [up(1.75), 1.0, 0.1], [448.0], [up(448.0)], [-3.5], [up(3.5), 2.0 ** -8],
        [big, 1.0, -big], [1.75 * 2.0 ** 127, 2.0 ** 118], [tiny], [2.0 ** -126, -tiny], [2.0 ** -109, 2.0 ** -126], [0.0, -0.0],
        [nan, 1.0, inf, -inf, 3.0], [nan], [inf, -inf], [2.0 ** -117 * 448, 2.0 ** -126],
    ]
    x = torch.zeros(len(rows), 40)
    for i, r in enumerate(rows):
        x[i, : len(r)] = torch.tensor(r)
        x[i, 32:] = x[i, :8].flip(0) * 0.5 if i % 2 else 0.0
    ref, scale = R.quantise(x)
    a = ops.act8_pack(x.cuda())
    assert torch.equal(a.scale.view(torch.uint8).cpu(), scale)
    got = R.values(a)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.nan_to_num(1.0), ref.nan_to_num(1.0))
    y = ops.act8_unpack(a)
    assert torch.equal(y.cpu().double().nan_to_num(1.0), ref.nan_to_num(1.0))      # normal numbers: exact in bf16, no infinities
    assert not torch.isinf(y).any()


def test_every_code_decodes(ops):
    codes = torch.arange(256, dtype=torch.uint8).repeat(3, 1).view(torch.float8_e4m3fn)
    scale = torch.tensor([[10] * 8, [127] * 8, [246] * 8], dtype=torch.uint8).view(torch.float8_e8m0fnu)
    a = ops.Act8(codes.cuda(), scale.cuda(), 256)
    ref = R.values(a)
    y = ops.act8_unpack(a, dtype=F32).cpu().double()
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(y.nan_to_num(7.0), ref.nan_to_num(7.0))


@pytest.mark.parametrize("rows,d", [(1, 1), (5, 33), (64, 1025), (3, 4100)])
def test_unpack_affine(ops, rows, d):
    x = rows_of(rows, d, F32, 1.0, 3)
    gamma, beta = rows_of(1, d, F32, 0.5, 4)[0] + 1, rows_of(1, d, F32, 0.5, 5)[0]
    gamma, beta = gamma.contiguous(), beta.contiguous()
    a = ops.act8_pack(x)
    v = R.values(a)
    for b in (None, beta):
        ref = v * gamma.cpu().double() + (0 if b is None else b.cpu().double())
        for dtype in (BF16, F32):
            y = ops.act8_unpack(a, gamma, b, dtype=dtype)
            close(y[:, :d], ref, HALF[dtype] * ref.abs() + U * ref.abs() + 1e-37)
            zero_pads(y, d)


def test_strided_codes_and_rows(ops):
    """Every matrix as a window of a wider one: other strides, and nothing outside the window is written."""
    rows, d = 19, 100
    x = rows_of(rows, d, BF16, 1.0, 1, step=160)
    ref, scale = R.quantise(x.cpu())
    q = torch.full((rows, 256), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((rows, 11), 0x55, dtype=torch.uint8, device="cuda")
    a = ops.Act8(q[:, 16:144].view(torch.float8_e4m3fn), s[:, 3:7].view(torch.float8_e8m0fnu), d)
    from vita_amd import _lib
    L = _lib.lib()
    assert L.vita_act8_pack(x.data_ptr(), 0, 160, rows, d, a.q.data_ptr(), 256, a.scale.data_ptr(), 11, ops._s()) == 0
    assert torch.equal(R.values(a), ref) and torch.equal(s[:, 3:7].cpu(), scale)
    assert (q[:, :16] == 0x55).all() and (q[:, 144:] == 0x55).all() and (s[:, :3] == 0x55).all() and (s[:, 7:] == 0x55).all()
    assert torch.equal(ops.act8_unpack(a)[:, :d].cpu().double(), ref)
    dg = rows_of(rows, d, BF16, 1.0, 2, step=160)
    whole = ops.Act8(a.q.contiguous(), a.scale.contiguous(), d)
    for t, u in zip(ops.gelu_act8_bwd(dg, a), ops.gelu_act8_bwd(dg.contiguous() if d % 8 == 0 else rows_of(rows, d, BF16, 1.0, 2), whole)):
        assert torch.equal(t, u)


# ------------------------------------------------------------------------------------------------ GELU
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_gelu(ops, rows, d, dtype):
    z = rows_of(rows, d, dtype, 2.0, rows * 3 + d)
    ldg = (d + 63) // 64 * 64
    g, a = ops.gelu_act8_fwd(z, ldg=ldg)
    zc = z.cpu().double()
    ref, scale = R.quantise(z.cpu())
    assert torch.equal(a.scale.view(torch.uint8).cpu(), scale) and torch.equal(R.values(a), ref)
    want, _ = R.gelu(zc)
    close(g[:, :d], want, 2.0 ** -8 * want.abs() + 5e-7 * zc.abs(), "g")
    zero_pads(g, d)
    dg = rows_of(rows, d, BF16, 1.0, 17)
    dz, g2 = ops.gelu_act8_bwd(dg, a, ldo=ldg)
    gv, dv = R.gelu(ref)
    dgc = dg.cpu().double()
    close(dz[:, :d], dgc * dv, 2.0 ** -8 * (dgc * dv).abs() + 6e-7 * dgc.abs() * 1.01, "dz")
    close(g2[:, :d], gv, 2.0 ** -8 * gv.abs() + 5e-7 * ref.abs(), "g2")
    zero_pads(dz, d); zero_pads(g2, d)
    only, none = ops.gelu_act8_bwd(dg, a, want_g=False, ldo=ldg)
    assert none is None and torch.equal(only, dz)


def test_gelu_gradient_against_differences(ops):
    """dz is the derivative of the forward kernel's function at the stored value: central differences of its fp32 formula."""
    z = torch.linspace(-6, 6, 1024).view(8, 128).cuda()
    _, a = ops.gelu_act8_fwd(z)
    v = R.values(a)
    dz, _ = ops.gelu_act8_bwd(torch.ones(8, 128, dtype=BF16, device="cuda"), a)
    h = 1e-5
    num = (R.gelu(v + h)[0] - R.gelu(v - h)[0]) / (2 * h)
    close(dz, num, 2.0 ** -8 * num.abs() + 1e-6)


# ------------------------------------------------------------------------------------------------ weight gradient
@pytest.mark.parametrize("k,m,n", [(1, 1, 1), (1, 8, 33), (3, 17, 100), (64, 40, 64), (130, 129, 257), (777, 300, 129), (2048, 520, 1025),
                                   (4100, 1025, 320), (5000, 96, 4100), (100, 4100, 4100), (2000, 3075, 1025), (9000, 40, 40), (20000, 8, 8),
                                   (65, 4352, 4160), (300, 4400, 4000)])
def test_wgrad(ops, k, m, n):
    x, dy = rows_of(k, n, F32, 1.0, k), rows_of(k, m, BF16, 1.0, m, junk=False)
    a = ops.act8_pack(x)
    dw = ops.act8_wgrad(dy, a)
    assert dw.shape == (m, n) and dw.dtype == F32
    v, d = R.values(a), dy.cpu().double()
    # products are exact in fp32; k additions at most, in chains of partial sums: k u of the magnitudes is never exceeded, and
    # sqrt(k) u (with a factor 8) is what rounding errors of either sign come to
    close(dw, d.t() @ v, (8 * k ** 0.5 + 8) * U * (d.abs().t() @ v.abs()) + 1e-30)
    assert torch.equal(dw, ops.act8_wgrad(dy, a))          # no order of summation that changes from call to call


# ------------------------------------------------------------------------------------------------ norms, forward
def _norm_case(rows, d, xt, rt, kind, seed, offset=0.0):
    x = rows_of(rows, d, xt, 1.0, seed)
    x += offset
    res = rows_of(rows, d, rt, 2.0, seed + 1) if rt is not None else None
    gamma = (1 + 0.2 * rows_of(1, d, F32, 1.0, seed + 2)[0]).contiguous()
    beta = (0.3 * rows_of(1, d, F32, 1.0, seed + 3)[0]).contiguous() if kind == "layer" else None
    return x, res, gamma, beta


def _check_norm(ops, x, res, gamma, beta, kind, eps, y_dtype, sum_dtype, pack, ldy=None):
    d = x.shape[1]
    a = ops.addnorm_fwd(x, gamma, beta, residual=res, kind=kind, eps=eps, y_dtype=y_dtype, sum_dtype=sum_dtype, pack=pack, ldy=ldy)
    c = lambda t: None if t is None else t.cpu()
    ref = R.norm_fwd(c(x), c(res), c(gamma), c(beta), kind, eps)
    if sum_dtype is not None:
        want = (x.float() + res.float()).to(sum_dtype)
        assert torch.equal(a.sum[:, :d], want)
        zero_pads(a.sum, d)
    # the mean is off by 40 u of the mean magnitude; that moves n by rstd times as much, and rstd to second order
    mag = ref["s"].abs().mean(1) + 1e-38
    dmu = 40 * U * mag if kind == "layer" else 0 * mag
    drel = 44 * U + (dmu * ref["rstd"]) ** 2 + 2 * U * (ref["s"].abs().amax(1) * ref["rstd"])
    close(a.rstd, ref["rstd"], drel * ref["rstd"], "rstd")
    if kind == "layer":
        close(a.mean, ref["mu"], dmu + U * ref["mu"].abs(), "mean")
    dn = ref["n"].abs() * drel[:, None] + (dmu * ref["rstd"])[:, None] + 4 * U * (ref["s"].abs() * ref["rstd"][:, None])
    gam = 1.0 if gamma is None else gamma.cpu().double().abs()
    dyv = gam * dn + 2 * U * ref["y"].abs()
    if y_dtype is not None:
        close(a.y[:, :d], ref["y"], dyv + HALF[y_dtype] * (ref["y"].abs() + dyv), "y")
        zero_pads(a.y, d)
    if pack is not None:
        want, err = (ref["n"], dn) if pack == "normed" else (ref["y"], dyv)
        g = torch.nn.functional.pad(want.abs(), (0, -d % 32)).reshape(want.shape[0], -1, 32).amax(-1)
        small = (2.0 ** -10 / 224) * g.repeat_interleave(32, 1)[:, :d]
        close(R.values(a.act), want, 1.001 * (err + 2.0 ** -4 * want.abs() + small) + 2.0 ** -127, "act")
    return a, ref


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,d", SHAPES + [(1500, 1025), (1100, 600), (1030, 1000), (1030, 1060), (1030, 1100), (1030, 1500), (1030, 2000),
                                             (20000, 40)])
def test_addnorm_fwd_shapes(ops, rows, d, kind):
    x, res, gamma, beta = _norm_case(rows, d, BF16, F32, kind, rows + d)
    _check_norm(ops, x, res, gamma, beta, kind, 1e-5, BF16, F32, "normed", ldy=(d + 63) // 64 * 64 if d < 8100 else None)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("rt", [None, BF16, F32])
@pytest.mark.parametrize("pack", [None, "normed", "output"])
def test_addnorm_fwd_types(ops, kind, xt, rt, pack):
    x, res, gamma, beta = _norm_case(21, 205, xt, rt, kind, 9)
    for y_dtype in (BF16, F32) + ((None,) if pack else ()):
        for st in ((None,) if rt is None else (None, BF16, F32)):
            _check_norm(ops, x, res, gamma, beta, kind, 1e-6, y_dtype, st, pack)
    _check_norm(ops, x, res, None, None, kind, 1e-6, F32, None, pack)


def test_addnorm_fwd_hard_rows(ops):
    """Rows of zeros, of one value, tiny and huge rows, a large offset, NaN and infinity confined to their own rows."""
    d = 129
    x = torch.randn(9, 136, generator=torch.Generator().manual_seed(0)).cuda()[:, :d]
    x[0] = 0; x[1] = 5.0; x[2] *= 1e-20; x[3] *= 1e15; x[4] += 1000.0
    for kind in ("rms", "layer"):
        _check_norm(ops, x[:5], None, None, None, kind, 1e-5, F32, None, "normed")
    x[6, 3] = float("nan"); x[7, 5] = float("inf")
    for kind in ("rms", "layer"):
        a = ops.addnorm_fwd(x, kind=kind, eps=1e-5, y_dtype=F32, pack="normed")
        clean = ops.addnorm_fwd(x[:6], kind=kind, eps=1e-5, y_dtype=F32, pack="normed")
        assert torch.equal(a.y[:6], clean.y) and torch.equal(a.act.q[:6].view(torch.uint8), clean.act.q.view(torch.uint8))
        assert torch.isnan(a.y[6, :d]).all() and torch.isnan(R.values(a.act)[6]).all()
        assert torch.isnan(a.y[7, 5]) and torch.isfinite(a.y[8, :d]).all()
        zero_pads(a.y, d)                                # also in the rows that are NaN
        assert torch.count_nonzero(a.act.q.view(torch.uint8)[:, d:]) == 0
    wide = torch.randn(3, 1032, device="cuda")[:, :1025]
    wide[1, 1024] = float("nan")
    many = torch.zeros(2100, 1032, device="cuda")[:, :1025]      # more rows: another kernel
    many.copy_(wide.repeat(700, 1))
    for rows in (wide, many):
        a = ops.addnorm_fwd(rows, kind="layer", eps=1e-5, y_dtype=BF16, pack="normed", ldy=1088)
        zero_pads(a.y, 1025)
        assert torch.count_nonzero(a.act.q.view(torch.uint8)[:, 1025:]) == 0
        assert torch.isnan(a.y[1, :1025]).all() and torch.isfinite(a.y[0, :1025]).all() and torch.isfinite(a.y[2, :1025]).all()


# ------------------------------------------------------------------------------------------------ norms, backward
def _check_bwd(ops, rows, d, kind, src_kind, dyt, dxt, with_in, seed, gamma=True):
    x, _, gam, beta = _norm_case(rows, d, BF16 if src_kind == "bf16" else F32, None, kind, seed)
    gam = gam if gamma else None
    ref = R.norm_fwd(x.cpu(), None, None, None, kind, 1e-5)
    rstd, mean = ref["rstd"].float().cuda(), ref["mu"].float().cuda()
    if src_kind == "act8":
        src = ops.addnorm_fwd(x, kind=kind, eps=1e-5, y_dtype=None, pack="normed").act
        n, dn = R.values(src), 0.0
    else:
        src = x
        n = (x.cpu().double() - (mean.cpu().double()[:, None] if kind == "layer" else 0.0)) * rstd.cpu().double()[:, None]
        dn = 4 * U * (x.cpu().double().abs() * rstd.cpu().double()[:, None] + n.abs())
    dy = rows_of(rows, d, dyt, 1.0, seed + 5)
    dx_in = rows_of(rows, d, dxt, 1.0, seed + 6) if with_in else None
    ldx = (d + 63) // 64 * 64 if d < 8100 else None
    dx, dg, db = ops.addnorm_bwd(dy, src, rstd, gam, kind=kind, mean=mean if kind == "layer" else None, dx_in=dx_in, dx_dtype=dxt, lddx=ldx)
    c = lambda t: None if t is None else t.cpu()
    want = R.norm_bwd(c(dy), n, c(rstd), c(gam), kind, c(dx_in))
    tol = 48 * U * want["size"]
    if src_kind != "act8":
        tol = tol + 2 * dn.amax(1, keepdim=True) * want["size"]        # n enters twice, relative to |n| >= its own size
    close(dx[:, :d], want["dx"], tol + HALF[dxt] * (want["dx"].abs() + tol) + 1e-37, "dx")
    zero_pads(dx, d)
    dyc = dy.cpu().double().abs()
    close(dg, want["dgamma"], 160 * U * want["dgamma_size"] + (dyc * dn).sum(0) + 1e-37, "dgamma")
    if kind == "layer":
        close(db, want["dbeta"], 160 * U * want["dbeta_size"] + 1e-37, "dbeta")
    else:
        assert db is None
    # the bf16 copy, sums added to a buffer, and no sums at all
    (dx2, dxb), n1, n2 = ops.addnorm_bwd(dy, src, rstd, gam, kind=kind, mean=mean if kind == "layer" else None, dx_in=dx_in,
                                         dx_dtype=dxt, lddx=ldx, want_bf16=True, acc=(dg.clone(), db.clone() if db is not None else None))
    assert n1 is None and n2 is None and torch.equal(dx2, dx) and torch.equal(dxb, dx.to(BF16))
    buf = torch.full_like(dg, 3.0), (torch.full_like(db, -2.0) if db is not None else None)
    ops.addnorm_bwd(dy, src, rstd, gam, kind=kind, mean=mean if kind == "layer" else None, dx_in=dx_in, dx_dtype=dxt, lddx=ldx, acc=buf)
    assert torch.equal(buf[0], dg + 3.0) and (db is None or torch.equal(buf[1], db - 2.0))
    dx3, g3, b3 = ops.addnorm_bwd(dy, src, rstd, gam, kind=kind, mean=mean if kind == "layer" else None, dx_in=dx_in, dx_dtype=dxt,
                                  lddx=ldx, want_dgamma=False, want_dbeta=False)
    assert g3 is None and b3 is None and torch.equal(dx3, dx)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("src", ["act8", "f32"])
@pytest.mark.parametrize("rows,d", SHAPES + [(4000, 129), (3000, 1025), (500, 600), (300, 1000), (300, 1060), (300, 1100), (300, 1500), (300, 2000)])
def test_addnorm_bwd_shapes(ops, rows, d, src, kind):
    _check_bwd(ops, rows, d, kind, src, BF16, F32, True, rows + d)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("src", ["act8", "bf16", "f32"])
@pytest.mark.parametrize("dyt", [BF16, F32])
@pytest.mark.parametrize("dxt", [BF16, F32])
@pytest.mark.parametrize("with_in", [False, True])
def test_addnorm_bwd_types(ops, kind, src, dyt, dxt, with_in):
    _check_bwd(ops, 23, 205, kind, src, dyt, dxt, with_in, 5, gamma=with_in)


@pytest.mark.parametrize("rows,d", [(1, 5), (2, 5), (3, 5), (40, 5), (41, 69), (33, 130), (33, 250), (70, 300), (40, 777), (40, 1601), (40, 2636),
                                    (40, 3500), (40, 5001), (40, 7003)])
def test_rows_that_end_inside_a_chunk(ops, rows, d):
    """Every way a row is held, with a last chunk of 8 columns that is not whole: against the formulas, and the same bits on rows
    without room between them (fp32 rows 4 columns apart reach into the next row) as on rows far apart."""
    _check_bwd(ops, rows, d, "layer", "act8", F32, BF16, True, rows + d)
    _check_bwd(ops, rows, d, "rms", "f32", BF16, F32, True, rows + d)
    x, res, gamma, beta = _norm_case(rows, d, F32, BF16, "layer", rows + d)
    a, _ = _check_norm(ops, x, res, gamma, beta, "layer", 1e-5, F32, BF16, "output")
    tight = lambda t, step: rows_of(rows, d, t.dtype, 1.0, 0, step=step).copy_(t)
    same = lambda u, v: all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(u, v))
    b = ops.addnorm_fwd(tight(x, 4), gamma, beta, residual=tight(res, 64), kind="layer", eps=1e-5, y_dtype=F32, sum_dtype=BF16, pack="output")
    assert same((a.y, a.sum, a.act.q, a.act.scale, a.rstd, a.mean), (b.y, b.sum, b.act.q, b.act.scale, b.rstd, b.mean))
    dy = rows_of(rows, d, F32, 1.0, d)
    f = lambda k: ops.addnorm_bwd(tight(dy, k), tight(x, k), a.rstd, gamma, kind="layer", mean=a.mean, dx_in=tight(dy, k))
    assert same(f(4), f(64))
    z = rows_of(rows, d, BF16, 1.0, d + 1)
    for u, v in ((x, 4), (z, 8)):
        p, q = ops.act8_pack(tight(u, v)), ops.act8_pack(tight(u, 64))
        assert same(p[:2], q[:2])
        (g, p), (h, q) = ops.gelu_act8_fwd(tight(u, v)), ops.gelu_act8_fwd(tight(u, 64))
        assert same((g,) + p[:2], (h,) + q[:2])
    assert same(ops.gelu_act8_bwd(tight(z, 8), p), ops.gelu_act8_bwd(tight(z, 64), p))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_addnorm_gradient_against_differences(ops, kind):
    """dx and dgamma from the kept sum against central differences of the 64-bit forward formula."""
    rows, d, eps = 3, 24, 1e-5
    x, _, gamma, beta = _norm_case(rows, d, F32, None, kind, 2)
    w = rows_of(rows, d, F32, 1.0, 8)
    a = ops.addnorm_fwd(x, gamma, beta, kind=kind, eps=eps, y_dtype=F32)
    dx, dg, _ = ops.addnorm_bwd(w, x, a.rstd, gamma, kind=kind, mean=a.mean)
    xc, gc, bc, wc = x.cpu().double(), gamma.cpu().double(), None if beta is None else beta.cpu().double(), w.cpu().double()
    f = lambda xx, gg: (R.norm_fwd(xx, None, gg, bc, kind, eps)["y"] * wc).sum().item()
    h = 1e-5
    for i, j in ((0, 0), (1, 7), (2, 23)):
        e = torch.zeros(rows, d, dtype=torch.float64); e[i, j] = h
        assert abs((f(xc + e, gc) - f(xc - e, gc)) / (2 * h) - dx[i, j].item()) < 1e-5 * (1 + abs(dx[i, j].item()))
        e = torch.zeros(d, dtype=torch.float64); e[j] = h
        assert abs((f(xc, gc + e) - f(xc, gc - e)) / (2 * h) - dg[j].item()) < 1e-5 * (1 + abs(dg[j].item()))


# ------------------------------------------------------------------------------------------------ use
def test_streams_and_graphs(ops):
    """The chain norm -> 8 bits -> gradients, eager, on another stream, and captured: every replay equals eager on its inputs."""
    rows, d, m = 200, 205, 96
    x, res, gamma, beta = _norm_case(rows, d, BF16, F32, "layer", 1)
    dy, dw_in = rows_of(rows, d, BF16, 1.0, 2), rows_of(rows, m, BF16, 1.0, 3, junk=False)

    def chain():
        a = ops.addnorm_fwd(x, gamma, beta, residual=res, kind="layer", sum_dtype=F32, pack="normed")
        g, z8 = ops.gelu_act8_fwd(a.y[:, :d])
        dz, g2 = ops.gelu_act8_bwd(dy, z8)
        dx, dg, db = ops.addnorm_bwd(dz[:, :d], a.act, a.rstd, gamma, kind="layer", dx_in=a.sum[:, :d])
        return a.y, a.sum, a.rstd, g, g2, dx, dg, db, ops.act8_unpack(a.act, gamma, beta), ops.act8_wgrad(dw_in, a.act)

    want = [t.clone() for t in chain()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    x0 = x.clone()
    for k in range(4):
        x.copy_(x0 * (1 + k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = chain()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
    x.copy_(x0)


def test_two_graphs_do_not_share_scratch(ops):
    """Two captured backward passes replayed on two streams at once: each has its own partial sums and workspace."""
    outs, graphs, wants, alive = [], [], [], []
    for seed in (1, 2):
        x, _, gamma, _ = _norm_case(3000, 205, F32, None, "rms", seed)
        dy = rows_of(3000, 205, BF16, 1.0, seed + 9, junk=False)
        a = ops.addnorm_fwd(x, gamma, pack="normed")
        f = lambda a=a, dy=dy, gamma=gamma: (*ops.addnorm_bwd(dy, a.act, a.rstd, gamma)[:2], ops.act8_wgrad(dy, a.act))
        alive.append(f)                                   # a graph reads its inputs where they were: they have to live on
        wants.append([t.clone() for t in f()])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_offsets_beyond_32_bits(ops):
    rows, d = (1 << 22) + 3, 520                          # 2.2e9 values
    x = torch.zeros(rows, d, dtype=BF16, device="cuda")
    tail = rows_of(5, d, BF16, 1.0, 4)
    x[-5:] = tail
    a = ops.act8_pack(x)
    ref, scale = R.quantise(tail.cpu())
    last = ops.Act8(a.q[-5:], a.scale[-5:], d)
    assert torch.equal(R.values(last), ref)
    y = ops.act8_unpack(a)
    assert torch.equal(y[-5:].cpu().double(), ref) and torch.count_nonzero(y[:-5]) == 0
    del y
    g, a2 = ops.gelu_act8_fwd(x)
    assert torch.equal(a2.q[-5:].view(torch.uint8), a.q[-5:].view(torch.uint8))
    assert torch.equal(g[-5:], ops.gelu_act8_fwd(tail)[0])
    dz, _ = ops.gelu_act8_bwd(x, a, want_g=False)
    assert torch.equal(dz[-5:], ops.gelu_act8_bwd(tail, last, want_g=False)[0])
    del g, a2, dz
    nrm = ops.addnorm_fwd(x, pack="normed")
    few = ops.addnorm_fwd(tail, pack="normed")
    assert torch.equal(nrm.y[-5:], few.y) and torch.equal(nrm.act.q[-5:].view(torch.uint8), few.act.q.view(torch.uint8))
    dx, _, _ = ops.addnorm_bwd(x, nrm.act, nrm.rstd, dx_dtype=BF16, want_dgamma=False)
    assert torch.equal(dx[-5:], ops.addnorm_bwd(tail, few.act, few.rstd, dx_dtype=BF16, want_dgamma=False)[0])


@pytest.mark.parametrize("k,m,n", [(46082, 20, 20), (46082, 300, 200), (46082, 300, 300), (69262, 8, 6625)])
def test_wgrad_of_many_parts(ops, k, m, n):
    """Long sums in 32 and more parts to an element, joined by one lane or by eight; the last case deals out a line of short pieces.
    The 64-bit product is taken on the device."""
    g = torch.Generator(device="cuda").manual_seed(k + m)
    x = torch.randn(k, -(-n // 8) * 8, device="cuda", generator=g).to(BF16)[:, :n]
    dy = torch.randn(k, -(-m // 8) * 8, device="cuda", generator=g).to(BF16)[:, :m]
    a = ops.act8_pack(x)
    dw = ops.act8_wgrad(dy, a)
    v, d = ops.act8_unpack(a)[:, :n].double(), dy.double().t().contiguous()
    close(dw, (d @ v).cpu(), ((8 * k ** 0.5 + 8) * U * (d.abs() @ v.abs())).cpu() + 1e-30)
    assert torch.equal(dw, ops.act8_wgrad(dy, a))


@pytest.mark.parametrize("which", ["dy", "codes"])
def test_wgrad_over_more_than_2_gib(ops, which):
    """Rows 2 MiB (dy) or 1 MiB (codes) apart: the sum needs more than one call of the kernel; pads of dy hold NaN."""
    k, m, n, pitch = 2600, 40, 100, 1 << 20
    x, dy = rows_of(k, n, F32, 1.0, 3), rows_of(k, m, BF16, 1.0, 5)
    a = ops.act8_pack(x)
    want, start = ops.act8_wgrad(dy, a), torch.randn(m, n, generator=torch.Generator().manual_seed(6)).cuda()
    if which == "dy":
        far = torch.empty(k, pitch, dtype=BF16, device="cuda")
        far[:, m:m + 8] = float("nan")
        far[:, :m] = dy
        got, acc = ops.act8_wgrad(far[:, :m], a), ops.act8_wgrad(far[:, :m], a, out=start.clone())
    else:
        q = torch.empty(k, pitch, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        q.view(torch.uint8)[:, :128] = a.q.view(torch.uint8)
        far = ops.Act8(q[:, :128], a.scale, n)
        got, acc = ops.act8_wgrad(dy, far), ops.act8_wgrad(dy, far, out=start.clone())
    v, d = R.values(a), dy.cpu().double()
    tol = (8 * k ** 0.5 + 8) * U * (d.abs().t() @ v.abs()) + 1e-30
    close(got, d.t() @ v, tol)
    close(want, d.t() @ v, tol)
    close(acc, start.cpu().double() + d.t() @ v, tol + 8 * U * start.cpu().double().abs())


def test_refusals_on_the_device(ops):
    x = torch.zeros(4, 64, device="cuda")
    with pytest.raises(ValueError, match="16-byte"):
        ops.act8_pack(torch.zeros(4, 33, device="cuda"))                    # rows of 132 bytes
    with pytest.raises(ValueError, match="16-byte"):
        ops.act8_pack(torch.zeros(4, 64, dtype=BF16, device="cuda")[:, 1:50])
    with pytest.raises(ValueError, match="contiguous"):
        ops.act8_pack(torch.zeros(64, 4, device="cuda").t())
    with pytest.raises(ValueError, match="overlap"):
        ops.act8_pack(torch.zeros(1, 64, device="cuda").expand(4, 64))
    with pytest.raises(ValueError):
        ops.addnorm_fwd(x, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError):
        ops.addnorm_fwd(x, torch.ones(64, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError):
        ops.addnorm_fwd(x, residual=torch.zeros(1, 64, device="cuda"))      # no broadcasting
    with pytest.raises(RuntimeError, match="8192"):
        ops.addnorm_fwd(torch.zeros(2, 8200, device="cuda"))
    a = ops.act8_pack(x)
    with pytest.raises(ValueError):
        ops.act8_wgrad(torch.zeros(5, 8, dtype=BF16, device="cuda"), a)
    with pytest.raises(ValueError):
        ops.addnorm_bwd(x, x, torch.ones(4, device="cuda"), kind="layer")   # needs the mean
    with pytest.raises(RuntimeError):
        ops.act8_pack(torch.zeros(4, 64))
