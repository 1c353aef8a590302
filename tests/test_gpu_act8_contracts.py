"""What the entry points of the 8-bit checkpoints and residual norms promise beside their formulas: Blocks whose two norms differ,
second derivatives, capture, buffers that serve as input and output, sums added to what a buffer holds, matrices that end with
their last element."""
import pytest
import torch
from torch import nn

import act8_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
BF16_TOL, STORED = 2e-2, 2.0 ** -4          # roundings of bf16 products; half an e4m3 step


@pytest.fixture(scope="module")
def V():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import vita_amd.nn as v
    return v


def rel(a, b):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


# ------------------------------------------------------------------------------------------------ norms of two kinds
def mixed_block(V, D, H, first, second, bits):
    torch.manual_seed(D)
    b = V.Block(D, H, 4.0, qkv_bias=True, norm_layer=first, saved_bits=bits)
    b.norm2 = second(D, eps=1e-3)                      # another eps too
    with torch.no_grad():
        for n, p in b.named_parameters():
            if "norm" in n:
                p.copy_((1.0 if "weight" in n else 0.0) + 0.5 * torch.randn_like(p))
            elif p.dim() == 1:
                p.copy_(0.1 * torch.randn_like(p))
    return b.cuda()


def plain_block(P, x, norms, H):
    """The Block in float64: norms = (module class, eps) of norm1 and norm2."""
    B, N, D = x.shape

    def norm(t, k):
        cls, eps = norms[k - 1]
        if cls is nn.LayerNorm:
            t = t - t.mean(-1, keepdim=True)
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * P[f"norm{k}.weight"]
        return t + P[f"norm{k}.bias"] if cls is nn.LayerNorm else t

    qkv = (norm(x, 1) @ P["attn.qkv.weight"].t() + P["attn.qkv.bias"]).view(B, N, 3, H, D // H).permute(2, 0, 3, 1, 4)
    o = ((qkv[0] @ qkv[1].transpose(-1, -2)) * (D // H) ** -0.5).softmax(-1) @ qkv[2]
    x = x + o.transpose(1, 2).reshape(B, N, D) @ P["attn.proj.weight"].t() + P["attn.proj.bias"]
    z = norm(x, 2) @ P["mlp.fc1.weight"].t() + P["mlp.fc1.bias"]
    return x + R.gelu(z)[0] @ P["mlp.fc2.weight"].t() + P["mlp.fc2.bias"]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("first,second", [(nn.RMSNorm, nn.LayerNorm), (nn.LayerNorm, nn.RMSNorm)])
def test_block_whose_norms_differ(V, first, second, bits):
    """Each norm is its own kind, forward and backward.  8 bits: the stored factors add half an e4m3 step to the gradients."""
    D, H, B, N = 129, 3, 2, 50
    blk = mixed_block(V, D, H, first, second, bits)
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(B, N, D, generator=g) + 1.0).cuda().requires_grad_()      # a mean that only LayerNorm takes away
    dy = torch.randn(B, N, D, generator=g).cuda()
    y = blk(x)
    y.backward(dy)
    P = {n: p.detach().cpu().double().requires_grad_() for n, p in blk.named_parameters()}
    xr = x.detach().cpu().double().requires_grad_()
    eps1 = torch.finfo(F32).eps if first is nn.RMSNorm else 1e-5
    yr = plain_block(P, xr, ((first, eps1), (second, 1e-3)), H)
    yr.backward(dy.cpu().double())
    tol = BF16_TOL if bits == 16 else 2 * BF16_TOL + STORED
    assert rel(y, yr) < BF16_TOL
    assert rel(x.grad, xr.grad) < tol
    for n, p in blk.named_parameters():
        assert rel(p.grad, P[n].grad) < tol, n


# ------------------------------------------------------------------------------------------------ matrices that end with their last element
@pytest.mark.parametrize("k,m,n", [(1, 1, 1), (1, 13, 40), (2, 15, 33), (64, 41, 64), (65, 6, 100), (130, 129, 257), (777, 300, 129), (129, 263, 4100),
                                   (2000, 3075, 1025), (65, 4355, 4160), (300, 4403, 4000), (9001, 43, 40), (46082, 20, 20), (69262, 13, 6625)])
def test_wgrad_of_a_dy_that_ends_with_its_last_element(V, k, m, n):
    """dy's memory stops behind column m of the last token, inside a 16-byte piece; what would follow holds NaN in one of two runs and
    does not exist for the caller in the other.  The last token counts in full, wherever its sum ends up (a tile, a part, a piece), and
    a buffer's old values are added once."""
    from vita_amd import ops
    ld = -(-m // 8) * 8
    g = torch.Generator(device="cuda").manual_seed(k + m + n)
    x = torch.randn(k, -(-n // 8) * 8, device="cuda", generator=g).to(BF16)[:, :n]
    x[-1] *= 8.0                                          # the last token weighs what the others do together
    flat = torch.full(((k - 1) * ld + m,), float("nan"), dtype=BF16, device="cuda")
    dy = flat.as_strided((k, m), (ld, 1))
    dy.copy_(torch.randn(k, m, device="cuda", generator=g))
    more = torch.cat([flat, torch.full((64,), float("nan"), dtype=BF16, device="cuda")])
    a = ops.act8_pack(x)
    dw = ops.act8_wgrad(dy, a)
    v, d = ops.act8_unpack(a)[:, :n].double(), dy.double().t().contiguous()
    tol = (8 * k ** 0.5 + 8) * U * (d.abs() @ v.abs()) + 1e-30       # k additions of exact products, as for every other weight gradient
    assert ((dw.double() - d @ v).abs() <= tol).all()
    assert torch.equal(dw, ops.act8_wgrad(more.as_strided((k, m), (ld, 1)), a))
    start = torch.randn(m, n, device="cuda", generator=g)
    assert torch.equal(ops.act8_wgrad(dy, a, out=start.clone()), start + dw)


# ------------------------------------------------------------------------------------------------ second derivatives
def test_second_derivatives_of_an_8_bit_linear_layer_are_refused(V):
    lin = nn.Linear(64, 32).cuda()
    x = torch.randn(1, 5, 64, device="cuda", requires_grad=True)
    f = lambda: V.linear_padded(x, lin, V._Shadows(), 64, 8)[..., :32].square().sum()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(f(), x, create_graph=True)
    want = 2 * torch.nn.functional.linear(x, lin.weight, lin.bias) @ lin.weight
    assert rel(torch.autograd.grad(f(), x)[0], want) < BF16_TOL


# ------------------------------------------------------------------------------------------------ capture
@pytest.mark.parametrize("bits", [8, 16])
def test_the_first_block_of_a_device_inside_a_capture(V, monkeypatch, bits):
    """No eager pass has chosen the second stream yet: the capture neither probes for it nor uses it, its replays equal eager passes
    (weight gradients add at most 64 partial sums with atomics in any order: 64 half steps, and a factor 4), and the first eager pass
    behind it probes."""
    torch.manual_seed(2)
    blk = V.Block(129, 3, 4.0, qkv_bias=True, saved_bits=bits).cuda()
    x = torch.randn(2, 70, 129, device="cuda", requires_grad=True)
    dy = torch.randn(2, 70, 129, device="cuda")
    leaves = [x] + list(blk.parameters())
    f = lambda: torch.autograd.grad(blk(x), leaves, dy)
    f()                                                  # every library and copy that a capture may not create exists
    torch.cuda.synchronize()
    monkeypatch.setattr(V, "_SIDE_STREAMS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    assert V._SIDE_STREAMS == {}
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(2, 70, 129, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, f()):
            assert rel(a, b) < 2.0 ** -16, k
    assert len(V._SIDE_STREAMS) == 1


# ------------------------------------------------------------------------------------------------ the C entries' buffers
def fwd_desc(ops, x, y, rstd, **kw):
    from vita_amd import _lib
    d = dict(x=x.data_ptr(), y=y.data_ptr(), rstd=rstd.data_ptr(), rows=x.shape[0], d=x.shape[1], ldx=x.stride(0), ldy=y.stride(0),
             x_dtype=ops._dt(x), y_dtype=ops._dt(y), eps=1e-5)
    return _lib.AddNormFwdDesc(**{**d, **kw})


def bwd_desc(ops, dy, src, rstd, dx, **kw):
    from vita_amd import _lib
    d = dict(dy=dy.data_ptr(), src=src.data_ptr(), rstd=rstd.data_ptr(), dx=dx.data_ptr(), rows=dy.shape[0], d=dy.shape[1], lddy=dy.stride(0),
             ldx=src.stride(0), lddx=dx.stride(0), dy_dtype=ops._dt(dy), src_dtype=ops._dt(src), dx_dtype=ops._dt(dx))
    return _lib.AddNormBwdDesc(**{**d, **kw})


def test_an_rms_norm_has_no_mean(V):
    """A caller with one set of buffers for both kinds passes its mean along: the RMS norm neither writes nor reads it."""
    import ctypes as C
    from vita_amd import _lib, ops
    rows, d = 40, 200
    x, dy = torch.randn(rows, d, device="cuda"), torch.randn(rows, d, device="cuda")
    y, dx, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda")
    mean = torch.full((rows,), 7.0, device="cuda")
    want = ops.addnorm_fwd(x, kind="rms", eps=1e-5, y_dtype=F32)
    dwant, _, _ = ops.addnorm_bwd(dy, x, want.rstd, kind="rms", want_dgamma=False)
    L = _lib.lib()
    assert L.vita_addnorm_fwd(C.byref(fwd_desc(ops, x, y, rstd, mean=mean.data_ptr())), ops._s()) == 0
    assert torch.equal(y, want.y) and torch.equal(rstd, want.rstd) and (mean == 7.0).all()
    assert L.vita_addnorm_bwd(C.byref(bwd_desc(ops, dy, x, rstd, dx, mean=mean.data_ptr())), ops._s()) == 0
    assert torch.equal(dx, dwant)


def wide(rows, d, dtype, seed, ld):
    """[rows, d] on rows of ld elements, NaN behind each; ends with its last element."""
    t = torch.full((rows, ld), float("nan"), dtype=dtype, device="cuda")
    t[:, :d] = torch.randn(rows, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)
    return t[:, :d]


@pytest.mark.parametrize("rows,d", [(1, 5), (41, 69), (70, 130), (70, 300), (2100, 777), (40, 777), (2100, 1025), (70, 1025), (1500, 1500), (40, 1601),
                                    (40, 2636), (40, 5001), (40, 7003)])
def test_outputs_in_place_of_inputs(V, rows, d):
    """The sum in place of x or of the residual, dx in place of dx_in, dz in place of dg: the same bits as in memory of their own, with
    rows that leave no room between them (4 fp32 columns behind a row are the next row's)."""
    import ctypes as C
    from vita_amd import _lib, ops
    L = _lib.lib()
    gamma = (1 + 0.2 * torch.randn(d, device="cuda")).contiguous()
    for dtype, step in ((F32, 4), (BF16, 8)):
        ld = -(-d // step) * step
        x, res = wide(rows, d, dtype, 1, ld), wide(rows, d, dtype, 2, ld)
        want = ops.addnorm_fwd(x, gamma, residual=res, eps=1e-5, y_dtype=BF16, sum_dtype=dtype, pack="normed")
        for place in ("x", "res"):
            t = {k: wide(rows, d, dtype, 0, ld).copy_(v) for k, v in (("x", x), ("res", res))}
            y, rstd = torch.empty_like(want.y), torch.empty_like(want.rstd)
            q, s = torch.empty_like(want.act.q), torch.empty_like(want.act.scale)
            desc = fwd_desc(ops, t["x"], y, rstd, gamma=gamma.data_ptr(), res=t["res"].data_ptr(), ldr=ld, res_dtype=ops._dt(res),
                            sum=t[place].data_ptr(), ldsum=ld, sum_dtype=ops._dt(x), q=q.data_ptr(), scale=s.data_ptr(), ldq=q.stride(0),
                            lds=s.shape[1])
            desc.d, desc.ldx, desc.ldy = d, ld, y.stride(0)
            assert L.vita_addnorm_fwd(C.byref(desc), ops._s()) == 0
            assert torch.equal(t[place], want.sum[:, :d]) and torch.equal(y, want.y) and torch.equal(rstd, want.rstd)
            assert torch.equal(q.view(torch.uint8), want.act.q.view(torch.uint8)) and torch.equal(s.view(torch.uint8), want.act.scale.view(torch.uint8))
        src, dy, dx_in = wide(rows, d, dtype, 3, ld), wide(rows, d, dtype, 4, ld), wide(rows, d, dtype, 5, ld)
        dwant, _, _ = ops.addnorm_bwd(dy, src, want.rstd, gamma, dx_in=dx_in, dx_dtype=dtype, want_dgamma=False)
        desc = bwd_desc(ops, dy, src, want.rstd, dx_in, gamma=gamma.data_ptr(), dx_in=dx_in.data_ptr(), lddx_in=ld)
        desc.lddy = desc.ldx = desc.lddx = ld
        assert L.vita_addnorm_bwd(C.byref(desc), ops._s()) == 0
        assert torch.equal(dx_in, dwant[:, :d])
    ld = -(-d // 8) * 8
    dg = wide(rows, d, BF16, 6, ld)
    _, act = ops.gelu_act8_fwd(wide(rows, d, BF16, 7, ld))
    want, g = ops.gelu_act8_bwd(dg, act)
    g2 = torch.empty_like(g)
    assert L.vita_gelu_act8_bwd(dg.data_ptr(), ld, act.q.data_ptr(), act.q.stride(0), act.scale.data_ptr(), act.scale.shape[1], rows, d,
                                dg.data_ptr(), ld, g2.data_ptr(), ld, ops._s()) == 0
    assert torch.equal(dg, want[:, :d]) and torch.equal(g2, g)


# ------------------------------------------------------------------------------------------------ which of two codes
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("pack", ["normed", "output"])
@pytest.mark.parametrize("rows,d", [(60000, 29), (30000, 100), (15000, 200), (9000, 300), (5000, 600), (4000, 1025), (700, 1025), (4000, 1060),
                                    (3000, 1500), (2000, 2000), (1000, 4000), (600, 7000)])
def test_codes_are_those_of_the_64_bit_norm(V, rows, d, kind, pack):
    """x and the residual are multiples of 2^-8 below 8, so that their sum is exact in 32 bits; no beta, whose addition may cancel.  What
    is left of the norm's own arithmetic then is a few 2^-52: the codes and the scales are those of the 64-bit formula, value by value,
    where 32 bits would put about one in two million on the other side of a border (a step of 2^-3)."""
    from vita_amd import ops
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    mk = lambda: ((torch.randn(rows, -(-d // 8) * 8, device="cuda", generator=g) * 128).round().clamp(-1024, 1024) / 256).to(BF16)[:, :d]
    x, res = mk(), mk()
    gamma = 1 + 0.2 * torch.randn(d, device="cuda", generator=g)
    wrong = total = 0
    for r in (None, res):
        a = ops.addnorm_fwd(x, gamma, residual=r, kind=kind, eps=1e-5, y_dtype=None, pack=pack)
        s = x.double() if r is None else x.double() + r.double()
        assert torch.equal(s.float().double(), s)
        n = s - s.mean(1, keepdim=True) if kind == "layer" else s
        n = n / torch.sqrt(n.square().mean(1, keepdim=True) + 1e-5)
        # on the CPU: powers of two from the device's pow are not all exact
        want, scale = R.quantise((n * gamma.double() if pack == "output" else n).cpu())
        wrong += (R.values(a.act) != want).sum().item() + (a.act.scale.view(torch.uint8).cpu() != scale).sum().item()
        total += want.numel()
    assert wrong == 0, (wrong, total)
