"""Blocks and models that keep their activations in 8 bits (saved_bits=8) and / or use RMS norms, and add_rms_norm.

The reference below is a Block in float64 whose backward pass uses what the kernels store: the normalised rows and the MLP's
pre-activation rounded to the 8-bit format.  What remains between it and the kernels are the roundings of the bf16 matrix products,
held to 2e-2 of each tensor's norm like every other bf16 path of these tests.  Against the 16-bit gradients the stored factors add
at most half an e4m3 step, 2^-4 of themselves.

The stored values themselves follow the kernels' forward pass, whose pre-activations differ from the float64 ones by the roundings
of bf16 products, at least by the last one (up to 2^-8 of the value).  A value that far from the border between two codes falls on
the other side with probability delta / step and is then a whole step away, so rounding turns a difference delta into one of
mean square delta * step <= 2^-8 * 2^-3 of the value's square: sqrt(2^-11) = 2.2e-2 more on tensors made from stored values."""
from types import SimpleNamespace

import pytest
import torch
from torch import nn

import act8_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
BF16_TOL, STORED = 2e-2, 2.0 ** -4
FLIPS = 2.0 ** -5.5


@pytest.fixture(scope="module")
def V():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import vita_amd.nn as v
    return v


def rel(a, b):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def make_block(V, D, H, kind, bits, seed=0, ratio=4.0, cls=None):
    torch.manual_seed(seed)
    b = V.Block(D, H, ratio, qkv_bias=True, norm_layer=nn.RMSNorm if kind == "rms" else nn.LayerNorm, saved_bits=bits)
    for n, p in b.named_parameters():
        with torch.no_grad():
            if "norm" in n:
                p.copy_((1.0 if "weight" in n else 0.0) + 0.2 * torch.randn_like(p))
            elif p.dim() == 1:
                p.copy_(0.1 * torch.randn_like(p))
    return b.cuda()


def reference_block(blk, x, dy, stored):
    """float64 forward and hand-written backward -> (y, dx, {name: gradient})."""
    P = {n: p.detach().cpu().double() for n, p in blk.named_parameters()}
    kind = "rms" if isinstance(blk.norm1, nn.RMSNorm) else "layer"
    eps1, eps2 = [torch.finfo(F32).eps if n.eps is None else n.eps for n in (blk.norm1, blk.norm2)]
    x, dy = x.detach().cpu().double(), dy.detach().cpu().double()
    B, N, D = x.shape
    H = blk.attn.num_heads
    keep = (lambda t: R.quantise(t.reshape(-1, t.shape[-1]))[0].reshape(t.shape)) if stored else (lambda t: t)
    norm = lambda s, k, e: R.norm_fwd(s.reshape(-1, D), None, P[f"norm{k}.weight"], P.get(f"norm{k}.bias"), kind, e)
    f1 = norm(x, 1, eps1)
    qkv = (f1["y"] @ P["attn.qkv.weight"].t() + P["attn.qkv.bias"]).view(B, N, 3 * D).requires_grad_()
    q, k, v = qkv.view(B, N, 3, H, D // H).permute(2, 0, 3, 1, 4)
    o = ((q @ k.transpose(-1, -2)) * (D // H) ** -0.5).softmax(-1) @ v
    o = o.transpose(1, 2).reshape(B, N, D)
    x1 = x + o.detach() @ P["attn.proj.weight"].t() + P["attn.proj.bias"]
    f2 = norm(x1, 2, eps2)
    z = f2["y"] @ P["mlp.fc1.weight"].t() + P["mlp.fc1.bias"]
    g, _ = R.gelu(z)
    y = x1 + (g @ P["mlp.fc2.weight"].t() + P["mlp.fc2.bias"]).view(B, N, D)
    # backward
    G = {}
    d = dy.reshape(-1, D)
    gv, dv = R.gelu(keep(z))
    G["mlp.fc2.weight"], G["mlp.fc2.bias"] = d.t() @ gv, d.sum(0)
    dz = (d @ P["mlp.fc2.weight"]) * dv

    def norm_bwd(dout, f, k, dx_in):
        n = keep(f["n"])
        r = R.norm_bwd(dout, n, f["rstd"], P[f"norm{k}.weight"], kind, dx_in)
        G[f"norm{k}.weight"] = r["dgamma"]
        if kind == "layer":
            G[f"norm{k}.bias"] = r["dbeta"]
        return r["dx"], n * P[f"norm{k}.weight"] + P.get(f"norm{k}.bias", 0.0)

    dx1, y2 = norm_bwd(dz @ P["mlp.fc1.weight"], f2, 2, d)
    G["mlp.fc1.weight"], G["mlp.fc1.bias"] = dz.t() @ y2, dz.sum(0)
    G["attn.proj.weight"], G["attn.proj.bias"] = dx1.t() @ o.detach().reshape(-1, D), dx1.sum(0)
    (dqkv,) = torch.autograd.grad(o, qkv, (dx1 @ P["attn.proj.weight"]).view(B, N, D))
    dqkv = dqkv.reshape(-1, 3 * D)
    dx, y1 = norm_bwd(dqkv @ P["attn.qkv.weight"], f1, 1, dx1)
    G["attn.qkv.weight"], G["attn.qkv.bias"] = dqkv.t() @ y1, dqkv.sum(0)
    return y, dx.view(B, N, D), G


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D,H,B,N", [(129, 3, 2, 50), (64, 2, 1, 1), (205, 1, 1, 77), (1025, 5, 2, 130), (48, 4, 3, 33)])
def test_block(V, D, H, B, N, kind, bits):
    if kind == "layer" and bits == 16:
        pytest.skip("the reference configuration, covered by the other Block tests")
    blk = make_block(V, D, H, kind, bits)
    g = torch.Generator().manual_seed(D + N)
    x = torch.randn(B, N, D, generator=g).cuda().requires_grad_()
    dy = torch.randn(B, N, D, generator=g).cuda()
    y = blk(x)
    y.backward(dy)
    ry, rdx, RG = reference_block(blk, x, dy, bits == 8)
    tol = BF16_TOL + (FLIPS if bits == 8 else 0.0)
    assert rel(y, ry) < BF16_TOL
    assert rel(x.grad, rdx) < tol
    top = max(v.norm().item() for v in RG.values())
    for n, p in blk.named_parameters():
        if RG[n].norm() < 1e-6 * top:          # one token: the softmax has no gradient
            assert p.grad.norm().item() < 1e-3 * top, n
            continue
        assert rel(p.grad, RG[n]) < tol, (n, rel(p.grad, RG[n]))


def test_block_gradients_near_the_16_bit_ones(V):
    a, b = make_block(V, 129, 3, "layer", 16), make_block(V, 129, 3, "layer", 8)
    x = torch.randn(2, 200, 129, generator=torch.Generator().manual_seed(1)).cuda()
    outs = []
    for blk in (a, b):
        xx = x.clone().requires_grad_()
        y = blk(xx)
        (y * torch.linspace(-1, 1, 129, device="cuda")).sum().backward()
        outs.append((y, xx.grad))
    assert rel(outs[1][0], outs[0][0]) < BF16_TOL and rel(outs[1][1], outs[0][1]) < BF16_TOL + STORED
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert rel(q.grad, p.grad) < 2 * BF16_TOL + STORED, n


def test_block_keeps_less(V):
    """Bytes a forward pass leaves behind for the backward pass, its input (the caller's) and output not counted.  A token of D = 1025
    (stream rows of 1088, heads padded to 5 x 224, hidden rows of 4160): 16 bits keep the sum behind the attention (4352 bytes), two
    norm outputs (2 x 2176), q k v (6720), the attention output (2240), GELU and its derivative (2 x 8320), 3 + 2 x 4 statistics of 4
    bytes a head or row = 34.3 KB; 8 bits keep two rows of 1056 + 33, q k v, the output, 4128 + 129 and the statistics = 15.4 KB and
    what the allocator rounds up (512 bytes a tensor): 0.45 to 0.46."""
    held = {}
    for bits in (16, 8):
        blk = make_block(V, 1025, 5, "layer", bits)
        x = torch.randn(2, 1500, 1088, device="cuda")
        x[..., 1025:] = 0
        x.requires_grad_()
        blk.forward_padded(x).sum().backward()           # shadows and workspaces exist from here on
        x.grad = None
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = blk.forward_padded(x)
        held[bits] = torch.cuda.memory_allocated() - before - y.numel() * 4
        del y
    assert held[8] < 0.47 * held[16], held


def test_checkpointed_and_in_place_gradients(V):
    """grad_checkpointing around 8-bit Blocks gives the same bits; gradients added into existing buffers equal fresh ones."""
    from vita_amd.networks import ViTDecoder
    grads = []
    for ckpt in (False, True):
        torch.manual_seed(3)
        m = ViTDecoder(129, 3, 2, 4.0, grad_checkpointing=ckpt, saved_bits=8).cuda()
        x = torch.randn(1, 65, 129, generator=torch.Generator().manual_seed(5)).cuda()
        for rep in range(2):                             # the second pass adds into the .grad of the first
            m(x).square().sum().backward()
        grads.append({n: p.grad.clone() for n, p in m.named_parameters()})
    for n in grads[0]:
        assert rel(grads[1][n], grads[0][n]) < 1e-5, n
    m.zero_grad(set_to_none=True)
    m(x).square().sum().backward()
    for n, p in m.named_parameters():
        assert rel(p.grad * 2, grads[0][n]) < 1e-5, n


@pytest.mark.parametrize("norm_layer", [nn.LayerNorm, nn.RMSNorm])
def test_stage1_step_with_saved_bits_8(V, norm_layer):
    from vita_amd.train import FlatAdam, ReconMAE, stage1_train_step
    cfg = dict(patch_size=(5, 8, 8), enc_embed_dim=129, enc_depth=2, enc_num_heads=3, dec_embed_dim=129, dec_depth=1, dec_num_heads=3,
               mlp_ratio=4.0, mask_ratio=0.7, mask_type="random", use_enc_pe=True, norm_layer=norm_layer)
    imgs = torch.rand(2, 9, 10, 32, 32, generator=torch.Generator().manual_seed(2)).cuda()
    res = {}
    for bits in (16, 8):
        torch.manual_seed(0)
        m = ReconMAE(img_shape=[9, 10, 32, 32], use_both_axes=True, saved_bits=bits, **cfg).cuda()
        opt = FlatAdam(m.parameters(), lr=1e-3)
        torch.manual_seed(7)
        loss = stage1_train_step(m, opt, imgs)
        res[bits] = (loss.item(), opt.g.clone())
        assert torch.isfinite(opt.p).all()
    assert abs(res[8][0] - res[16][0]) < BF16_TOL * abs(res[16][0])
    assert rel(res[8][1], res[16][1]) < BF16_TOL + STORED


def test_stage2_step_with_saved_bits_8(V):
    from vita_amd.train import FlatAdam, MultimodalSimCLR, stage2_train_step
    feats = {"numerical": ["a", "b"], "single_categorical": ["c"], "multi_categorical": {"m0": [3], "m1": [5]}}
    res = {}
    for bits in (16, 8):
        imaging = dict(patch_size=(5, 8, 8), enc_embed_dim=129, enc_depth=1, enc_num_heads=3, mlp_ratio=4.0, mask_ratio=0.5,
                       mask_type="random", use_enc_pe=True, grad_checkpointing=False, projection_dim=16, saved_bits=bits)
        tab = SimpleNamespace(grad_checkpointing=False, embedding_dim=129, encoder_num_heads=3, encoder_mlp_ratio=4.0,
                              encoder_num_layers=1, projection_dim=16, saved_bits=bits)
        torch.manual_seed(0)
        m = MultimodalSimCLR([9, 10, 16, 16], imaging, tab, feats).cuda()
        assert all(b.saved_bits == bits for b in list(m.encoder_imaging.encoder) + list(m.encoder_tabular.network))
        opt = FlatAdam(m.parameters(), lr=1e-4)
        g = torch.Generator().manual_seed(4)
        imgs = torch.rand(16, 9, 10, 16, 16, generator=g).cuda()
        tabs = torch.cat([torch.randn(16, 2, generator=g), torch.randint(0, 2, (16, 3), generator=g).float()], 1).cuda()
        torch.manual_seed(9)
        loss, _, _ = stage2_train_step(m, opt, imgs, tabs)
        res[bits] = (loss.item(), opt.g.clone())
    assert abs(res[8][0] - res[16][0]) < BF16_TOL * abs(res[16][0])
    # BatchNorm makes the batch's cotangents cancel, which amplifies relative errors of their sums (4e-2 in the 16-bit tests)
    assert rel(res[8][1], res[16][1]) < 2 * BF16_TOL + 2 * STORED


# ------------------------------------------------------------------------------------------------ add_rms_norm
def rms_reference(x, r, w, eps):
    x = x.detach().cpu().double().requires_grad_()
    w = w.detach().cpu().double().requires_grad_()
    r = None if r is None else r.detach().cpu().double().requires_grad_()
    s = x if r is None else x + r
    return x, r, w, s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * w, s


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("xt,rt", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16), (BF16, None), (F32, None)])
@pytest.mark.parametrize("shape", [(1, 1025), (2, 7, 64), (3, 129), (2, 3, 4, 200)])
def test_add_rms_norm(V, shape, xt, rt, bits):
    g = torch.Generator().manual_seed(len(shape))
    mk = lambda t: None if t is None else torch.randn(*shape, generator=g).to(t).cuda().requires_grad_()
    x, r = mk(xt), mk(rt)
    w = (1 + 0.2 * torch.randn(shape[-1], generator=g)).cuda().requires_grad_()
    out = V.add_rms_norm(x, r, w, 1e-5, saved_bits=bits)
    y, s = (out, None) if r is None else out
    rx, rr, rw, ry, rs = rms_reference(x, r, w, 1e-5)
    assert y.dtype == xt and y.shape == x.shape and (s is None or (s.shape == x.shape and s.dtype == torch.promote_types(xt, rt)))
    half = {BF16: 2.0 ** -8, F32: 2.0 ** -20}
    assert rel(y, ry) < half[xt] and (s is None or rel(s, rs) < half[s.dtype])
    dy = torch.randn(*shape, generator=g).to(xt).cuda()
    ds = None if s is None else torch.randn(*shape, generator=g).to(s.dtype).cuda()
    torch.autograd.backward([y] + ([] if s is None else [s]), [dy] + ([] if s is None else [ds]))
    torch.autograd.backward([ry] + ([] if s is None else [rs]), [dy.cpu().double()] + ([] if s is None else [ds.cpu().double()]))
    # 8 bits: n is off by half a step, it enters dx by n mean(h n) (off by at most 2 half steps of it) and dgamma linearly; the sum
    # kept in bf16 by half a bf16 step, twice in the same way
    tol = half[xt] + (2 * STORED if bits == 8 else (2 * half[BF16] if BF16 in (xt, rt) else 0)) + 1e-6
    for got, want in ((x, rx), (r, rr), (w, rw)):
        if got is not None:
            assert got.grad.dtype == got.dtype and rel(got.grad, want.grad) < tol


def test_add_rms_norm_gradients_of_one_output(V):
    x = torch.randn(5, 64, device="cuda", requires_grad=True)
    r = torch.randn(5, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, s = V.add_rms_norm(x, r, w)
    gx, gr = torch.autograd.grad(s.sum(), (x, r), retain_graph=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, torch.ones_like(r))
    gy = torch.autograd.grad(y.square().sum(), (x, r, w), retain_graph=True)
    both = torch.autograd.grad(y.square().sum() + s.sum(), (x, r, w))
    assert rel(gy[0] + 1, both[0]) < 1e-6 and torch.equal(gy[0], gy[1]) and torch.equal(gy[2], both[2])
    # the same tensor as branch and residual: both gradients reach it
    x2 = x.detach().clone().requires_grad_()
    y, s = V.add_rms_norm(x2, x2, w)
    s.sum().backward()
    assert torch.equal(x2.grad, torch.full_like(x2, 2.0))


def test_add_rms_norm_layouts_and_refusals(V):
    base = torch.randn(6, 40, 33, device="cuda")
    w = torch.ones(33, device="cuda")
    r = torch.randn(6, 40, 33, device="cuda")
    want, ws = V.add_rms_norm(base, r, w)
    for x in (base.transpose(0, 1).contiguous().transpose(0, 1), base.as_strided(base.shape, base.stride())):
        y, s = V.add_rms_norm(x, r, w)
        assert torch.equal(y, want) and torch.equal(s, ws)
    with pytest.raises(ValueError, match="broadcast"):
        V.add_rms_norm(base, r[:1], w)
    with pytest.raises(TypeError):
        V.add_rms_norm(base.half(), None, w)
    with pytest.raises(ValueError):
        V.add_rms_norm(base, r, w, saved_bits=4)
    with pytest.raises(ValueError):
        V.add_rms_norm(base, r, torch.ones(32, device="cuda"))
    with pytest.raises(ValueError):
        V.add_rms_norm(base[:0], r[:0], w)
    with pytest.raises(RuntimeError):
        V.add_rms_norm(base.cpu(), None, w)
    y, s = V.add_rms_norm(base.clone().requires_grad_(), r, w)
    s.add_(1.0)                                          # what the backward pass keeps was overwritten
    with pytest.raises(RuntimeError, match="inplace|in-place"):
        y.sum().backward()
    x8 = base.clone().requires_grad_()
    want = torch.autograd.grad(V.add_rms_norm(x8, r, w, saved_bits=8)[0].square().sum(), x8)[0]
    y, s = V.add_rms_norm(x8, r, w, saved_bits=8)
    s += 1.0                                             # the 8-bit rows are kept apart: writing the sum in place is fine
    assert torch.equal(torch.autograd.grad(y.square().sum(), x8)[0], want)


def test_second_derivatives_are_refused(V):
    """The backward passes are kernels too and have no gradient of their own: an error, not a sum with that part missing."""
    x = torch.randn(2, 5, 64, device="cuda", requires_grad=True)
    norm = nn.RMSNorm(64).cuda()
    blk = make_block(V, 64, 2, "layer", 8)
    for f in (lambda: V.add_rms_norm(x, x, norm.weight)[0], lambda: V.layer_norm_padded(x, norm), lambda: blk.forward_padded(x)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(f().square().sum(), x, create_graph=True)
        torch.autograd.grad(f().square().sum(), x)


def test_training_pass_in_a_graph(V):
    """Forward and backward of a chain of norms captured once, replayed on new inputs: each replay equals eager."""
    x = torch.randn(40, 205, device="cuda").to(BF16).requires_grad_()
    r = torch.randn(40, 205, device="cuda", requires_grad=True)
    w = torch.ones(205, device="cuda", requires_grad=True)

    def f():
        y, s = V.add_rms_norm(x, r, w, saved_bits=8)
        y2, s2 = V.add_rms_norm(y * 2, s, w, saved_bits=8)
        return torch.autograd.grad((y2.float() * s2).sum(), (x, r, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(40, 205, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = f()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_column_sums_in_a_graph(V):
    """The sums' memory is cleared in its place: it held something else earlier in the same graph.  At most 256 partial sums meet in an
    atomic, 8 rows of a thread before: 264 half steps of the sum of magnitudes."""
    from vita_amd import ops
    x = torch.randn(300, 64, device="cuda").to(BF16)
    f = lambda: [ops.colsum((x * k).contiguous(), 64, 300, 64) for k in range(1, 5)]
    f()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for _ in range(4):
        x.copy_(torch.randn(300, 64, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        f()
        for k, o in enumerate(out, 1):
            d = (x * k).cpu().double()
            assert ((o.cpu().double() - d.sum(0)).abs() <= 264 * 2.0 ** -24 * d.abs().sum(0)).all(), k


@pytest.mark.parametrize("bits,kind", [(8, "layer"), (8, "rms"), (16, "layer")])
def test_block_in_a_graph(V, bits, kind):
    """A Block's training pass captured once and replayed on new inputs.  Weight and bias gradients add at most 64 partial sums with
    atomics, in any order: 64 half steps of 2^-24, and a factor 4 for sums larger than their result."""
    blk = make_block(V, 129, 3, kind, bits, seed=5)
    x = torch.randn(2, 70, 129, device="cuda", requires_grad=True)
    dy = torch.randn(2, 70, 129, device="cuda")
    leaves = [x] + list(blk.parameters())
    f = lambda: torch.autograd.grad(blk(x), leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(2, 70, 129, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, f()):
            assert rel(a, b) < 2.0 ** -16, k
