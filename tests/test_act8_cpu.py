"""Refusals of the 8-bit checkpoint and residual norm entry points, checked without a GPU: the Python wrappers before any call,
the C entry points before any launch."""
import ctypes as C

import pytest
import torch

import act8_reference as R

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from vita_amd import ops as _ops
    return _ops


def test_reference_format_against_torch_casts():
    """The tests' own statement of the format: e4m3 rounding as torch casts it, the scale the smallest that holds the group."""
    x = torch.randn(50, 70, generator=torch.Generator().manual_seed(0)) * torch.logspace(-30, 30, 50)[:, None]
    v, s = R.quantise(x)
    g = torch.nn.functional.pad(x, (0, 26)).reshape(50, 3, 32)
    scale = torch.exp2(s.float() - 127).unsqueeze(-1)
    assert torch.equal(((g / scale).to(torch.float8_e4m3fn).float() * scale).reshape(50, -1)[:, :70].double(), v)
    top = g.abs().amax(-1) / scale[..., 0]
    assert (top <= 448).all() and ((top > 224) | (s == 10)).all()
    assert torch.equal(v.to(BF16).double(), v)


def test_wrappers_refuse(ops):
    x = torch.zeros(4, 64)
    act = ops.Act8(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu), 64)
    for f in (ops.act8_pack, ops.gelu_act8_fwd, ops.addnorm_fwd):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f(x)
        with pytest.raises(TypeError):
            f(x.half())
        with pytest.raises(TypeError):
            f(x.double())
        with pytest.raises(ValueError, match="2-D"):
            f(x[None])
        with pytest.raises(ValueError, match="empty"):
            f(x[:0])
        with pytest.raises(ValueError, match="empty"):
            f(x[:, :0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.act8_unpack(act)
    with pytest.raises(TypeError):
        ops.act8_unpack(x)
    with pytest.raises(TypeError):
        ops.act8_unpack(act, dtype=torch.float16)
    with pytest.raises(ValueError, match="beta needs gamma"):
        ops.act8_unpack(act, beta=torch.zeros(64))
    for bad in (act._replace(q=act.q.view(torch.uint8)), act._replace(d=65), act._replace(scale=act.scale[:3]), act._replace(q=act.q[:0]),
                act._replace(d=0), act._replace(scale=act.scale.view(torch.uint8))):
        with pytest.raises(ValueError):
            ops.act8_unpack(bad)
    for kw in (dict(kind="batch"), dict(pack="codes"), dict(beta=torch.zeros(64)), dict(sum_dtype=F32), dict(y_dtype=None),
               ):
        with pytest.raises(ValueError):
            ops.addnorm_fwd(x, **kw)
    with pytest.raises(TypeError):
        ops.addnorm_fwd(x, y_dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.addnorm_bwd(x, act, torch.ones(4), kind="batch")
    with pytest.raises(TypeError):
        ops.addnorm_bwd(x, act, torch.ones(4), dx_dtype=torch.float16)


def test_c_entries_refuse_before_any_launch():
    from vita_amd import _lib
    L = _lib.lib()
    p = 1 << 20                                             # an aligned address that is never dereferenced
    pack = lambda x=p, dt=1, ldx=64, rows=4, d=64, q=p, ldq=64, s=p, lds=2: L.vita_act8_pack(x, dt, ldx, rows, d, q, ldq, s, lds, None)
    for kw in (dict(x=0), dict(x=p + 4), dict(dt=2), dict(ldx=63), dict(ldx=62), dict(rows=0), dict(d=0), dict(d=65), dict(q=0),
               dict(q=p + 8), dict(ldq=56), dict(ldq=32), dict(s=0), dict(lds=1), dict(d=(1 << 20) + 1, ldx=1 << 21, ldq=1 << 21, lds=1 << 16),
               dict(dt=0, ldx=68), dict(rows=1 << 60)):
        assert pack(**kw) == -1, kw
        assert b"invalid argument" in L.vita_last_error()
    un = lambda q=p, ldq=64, s=p, lds=2, rows=4, d=64, g=None, b=None, y=p, dt=0, ldy=64: L.vita_act8_unpack(q, ldq, s, lds, rows, d, g, b, y, dt, ldy, None)
    for kw in (dict(q=0), dict(y=0), dict(y=p + 2), dict(ldy=60), dict(ldy=56), dict(b=p), dict(rows=-1), dict(dt=7), dict(lds=1)):
        assert un(**kw) == -1, kw
    gf = lambda z=p, dt=0, ldz=64, rows=4, d=64, g=p, ldg=64, q=p, ldq=64, s=p, lds=2: L.vita_gelu_act8_fwd(z, dt, ldz, rows, d, g, ldg, q, ldq, s, lds, None)
    for kw in (dict(z=0), dict(g=0), dict(ldg=63), dict(ldz=60), dict(s=0), dict(rows=0)):
        assert gf(**kw) == -1, kw
    gb = lambda dg=p, ldd=64, q=p, ldq=64, s=p, lds=2, rows=4, d=64, dz=p, ldz=64, g=None, ldg=0: L.vita_gelu_act8_bwd(dg, ldd, q, ldq, s, lds, rows, d, dz, ldz, g, ldg, None)
    for kw in (dict(dg=0), dict(dz=0), dict(ldd=60), dict(g=p, ldg=32), dict(d=0)):
        assert gb(**kw) == -1, kw
    wg = lambda dy=p, ldy=64, q=p, ldq=64, s=p, lds=2, dw=p, ldw=64, m=64, n=64, k=10, ws=p, wb=1 << 30: L.vita_act8_wgrad(dy, ldy, q, ldq, s, lds, dw, ldw, m, n, k, 0, ws, wb, None)
    for kw in (dict(dy=0), dict(ldy=60), dict(dw=0), dict(ldw=63), dict(m=0), dict(n=0), dict(k=0), dict(q=0), dict(ldq=32)):
        assert wg(**kw) == -1, kw
    need = L.vita_act8_wgrad_ws_bytes(64, 64, 10)
    if need > 0:
        assert wg(wb=need - 1) == -1 and wg(ws=0) == -1 and wg(ws=p + 8) == -1
    good = dict(x=p, y=p, rows=4, d=64, ldx=64, ldy=64, x_dtype=1, y_dtype=0, eps=1e-5)
    for kw in (dict(x=0), dict(y=0), dict(ldx=62), dict(kind=2), dict(kind=-1), dict(rows=0), dict(d=0), dict(sum=p, ldsum=64), dict(beta=p),
               dict(res=p, ldr=63), dict(res=p + 4, ldr=64, res_dtype=1), dict(q=p, scale=p, ldq=64, lds=1), dict(q=p, scale=p, ldq=64, lds=2, pack=3),
               dict(res=p, ldr=64, res_dtype=1, sum=p, ldsum=60, sum_dtype=1), dict(y_dtype=5), dict(x_dtype=3)):
        assert L.vita_addnorm_fwd(C.byref(_lib.AddNormFwdDesc(**{**good, **kw})), None) == -1, kw
    assert L.vita_addnorm_fwd(C.byref(_lib.AddNormFwdDesc(**{**good, "d": 8200, "ldx": 8200, "ldy": 8200})), None) == -2
    assert L.vita_addnorm_fwd(None, None) == -1
    good = dict(dy=p, src=p, rstd=p, dx=p, rows=4, d=64, lddy=64, ldx=64, lddx=64, dy_dtype=0, src_dtype=1, dx_dtype=1)
    for kw in (dict(dy=0), dict(src=0), dict(rstd=0), dict(dx=0), dict(q=p, scale=p, ldq=64, lds=2), dict(kind=1), dict(kind=3), dict(dgamma=p),
               dict(partial=p), dict(dbeta=p, partial=p), dict(lddx=60), dict(dx_in=p, lddx_in=2), dict(dx_bf16=p, lddxb=60), dict(rows=0),
               dict(src=0, q=p, scale=0, ldq=64, lds=2), dict(src_dtype=9)):
        assert L.vita_addnorm_bwd(C.byref(_lib.AddNormBwdDesc(**{**good, **kw})), None) == -1, kw
    assert L.vita_addnorm_bwd(C.byref(_lib.AddNormBwdDesc(**{**good, "d": 8200, "ldx": 8200, "lddx": 8200, "lddy": 8200})), None) == -2
    assert L.vita_addnorm_bwd(None, None) == -1


def test_modules_take_and_refuse_the_new_options():
    from torch import nn
    from vita_amd.networks import ImagingMaskedEncoder, ViTDecoder
    from vita_amd.nn import Block, add_rms_norm
    b = Block(16, 2, 4.0, qkv_bias=True, norm_layer=nn.RMSNorm, saved_bits=8)
    assert set(b.state_dict()) == {k for k in Block(16, 2, 4.0, qkv_bias=True).state_dict() if not k.startswith("norm") or k.endswith("weight")}
    for bad in (4, "8", None):
        with pytest.raises(ValueError):
            Block(16, 2, 4.0, saved_bits=bad)
    with pytest.raises(NotImplementedError):
        Block(16, 2, 4.0, norm_layer=nn.BatchNorm1d)
    enc = ImagingMaskedEncoder(enc_embed_dim=17, patch_size=(5, 8, 8), img_shape=[9, 10, 16, 16], enc_num_heads=1, enc_depth=2, mlp_ratio=4.0,
                               mask_ratio=0.5, mask_type="random", use_both_axes=True, use_enc_pe=True, saved_bits=8)
    assert all(blk.saved_bits == 8 for blk in enc.encoder)
    assert all(blk.saved_bits == 16 for blk in ViTDecoder(16, 2, 1, 4.0).network)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        b(torch.zeros(1, 4, 16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        add_rms_norm(torch.zeros(2, 16), None, torch.ones(16))
