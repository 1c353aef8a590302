"""Thin torch-tensor wrappers over the C ABI (include/vita_hip.h).  PyTorch only provides device
memory and the stream; every computation happens in libvita_hip.so."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import AddNormBwdDesc, AddNormFwdDesc, GemmDesc, check

BF16, F32 = 0, 1
EPI_NONE, EPI_GELU, EPI_RESIDUAL, EPI_GELU_BWD = 0, 1, 2, 3


def rup(x: int, m: int) -> int:
    return (int(x) + m - 1) // m * m


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _s():
    """The current stream of the current device (torch.cuda.current_stream().cuda_stream without building its Python object: 0.2
    instead of 2.7 us on the way to every launch)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return BF16
    if t.dtype == torch.float32:
        return F32
    raise TypeError(f"unsupported dtype {t.dtype}")


# Optional per-launch timing for bench.py: PROF = [] enables (name, start_event, end_event, algorithmic_work).
PROF = None


class _Timed:
    def __init__(self, name, work):
        self.name, self.work = name, work

    def __enter__(self):
        if PROF is not None:
            self.e0 = torch.cuda.Event(enable_timing=True); self.e0.record()

    def __exit__(self, *exc):
        if PROF is not None:
            e1 = torch.cuda.Event(enable_timing=True); e1.record()
            PROF.append((self.name, self.e0, e1, self.work))


def gemm(a, b, c, m, n, k, lda, ldb, ldc, *, a_layout=0, b_layout=0, bias=None, epilogue=EPI_NONE,
         aux_in=None, aux_out=None, ld_aux=0, alpha=1.0, split_k=1, batch=(1, 1),
         a_strides=(0, 0), b_strides=(0, 0), c_strides=(0, 0), row_seg=(0, 0), col_seg=(0, 0),
         a_off=0, b_off=0, c_off=0, flops=None, variant=0):
    """C[m,n] = epi(alpha * A(m,k) B(k,n)); a/b bf16 tensors, c bf16|fp32.  *_off are element offsets.
    flops: algorithmic (un-padded) FLOPs of this launch for the roofline accounting."""
    assert a.dtype == torch.bfloat16 and b.dtype == torch.bfloat16
    d = GemmDesc()
    d.a = a.data_ptr() + 2 * a_off
    d.b = b.data_ptr() + 2 * b_off
    d.c = c.data_ptr() + c.element_size() * c_off
    d.bias = _p(bias); d.aux_in = _p(aux_in); d.aux_out = _p(aux_out)
    d.m, d.n, d.k = m, n, k
    d.lda, d.ldb, d.ldc, d.ld_aux = lda, ldb, ldc, ld_aux
    d.batch_outer, d.batch_inner = batch
    d.a_stride_outer, d.a_stride_inner = a_strides
    d.b_stride_outer, d.b_stride_inner = b_strides
    d.c_stride_outer, d.c_stride_inner = c_strides
    d.a_layout, d.b_layout = a_layout, b_layout
    d.c_dtype = _dt(c); d.epilogue = epilogue; d.split_k = split_k
    d.row_seg_phys, d.row_seg_log = row_seg
    d.col_seg_phys, d.col_seg_log = col_seg
    d.alpha = alpha
    with _Timed(f"gemm_kernel<{a_layout},{b_layout}>", flops if flops is not None else 2.0 * m * n * k * batch[0] * batch[1]):
        check(_lib.lib().vita_gemm_bf16_ex(C.byref(d), variant, _s()), "vita_gemm_bf16")
    return c


def pack_weight(w: torch.Tensor, rows_phys: int, ld_phys: int, row_seg=(0, 0), col_seg=(0, 0), out=None):
    w = w.detach()
    assert w.dtype == torch.float32 and w.is_contiguous()
    rows_log, cols_log = w.shape[0], w[0].numel()
    if out is None:
        out = torch.empty(rows_phys, ld_phys, dtype=torch.bfloat16, device=w.device)
    check(_lib.lib().vita_pack_weight_bf16(w.data_ptr(), rows_log, cols_log, out.data_ptr(), rows_phys, ld_phys,
                                           row_seg[0], row_seg[1], col_seg[0], col_seg[1], _s()), "pack_weight")
    return out


def pack_vec(v: torch.Tensor, n_phys: int, seg=(0, 0), out=None):
    v = v.detach()
    if out is None:
        out = torch.empty(n_phys, dtype=torch.float32, device=v.device)
    check(_lib.lib().vita_pack_vec_f32(v.data_ptr(), v.numel(), out.data_ptr(), n_phys, seg[0], seg[1], _s()), "pack_vec")
    return out


def unpack_vec(v: torch.Tensor, n_log: int, seg=(0, 0)):
    out = torch.zeros(n_log, dtype=torch.float32, device=v.device)
    check(_lib.lib().vita_unpack_vec_f32(v.data_ptr(), v.numel(), out.data_ptr(), n_log, seg[0], seg[1], _s()), "unpack_vec")
    return out


def layernorm_fwd(x, ldx, gamma, beta, rows, d, ldy, out_dtype=torch.bfloat16, eps=1e-5):
    y = torch.empty(rows, ldy, dtype=out_dtype, device=x.device)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(_lib.lib().vita_layernorm_fwd(x.data_ptr(), ldx, gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), ldy, _dt(y),
                                        mean.data_ptr(), rstd.data_ptr(), rows, d, eps, _s()), "layernorm_fwd")
    return y, mean, rstd


def layernorm_bwd(dy, lddy, x, ldx, gamma, mean, rstd, rows, d, lddx, dx_in=None, want_bf16=False, ld_dxb=0, acc=None):
    """acc = (dgamma_buf, dbeta_buf): fp32 [d] buffers the weight / bias gradients are ADDED to (None is then returned
    for both) instead of being materialised."""
    dev = x.device
    dx = torch.empty(rows, lddx, dtype=torch.float32, device=dev)
    dxb = torch.empty(rows, ld_dxb, dtype=torch.bfloat16, device=dev) if want_bf16 else None
    nblk = _lib.lib().vita_layernorm_bwd_nblk(rows)
    partial = torch.empty(2 * nblk * d, dtype=torch.float32, device=dev)
    if acc is not None:
        dgamma, dbeta = acc
        assert dgamma.dtype == torch.float32 and dbeta.dtype == torch.float32 and dgamma.numel() == d and dbeta.numel() == d
        assert dgamma.is_contiguous() and dbeta.is_contiguous()
        fn = _lib.lib().vita_layernorm_bwd_acc
    else:
        dgamma = torch.empty(d, dtype=torch.float32, device=dev)
        dbeta = torch.empty(d, dtype=torch.float32, device=dev)
        fn = _lib.lib().vita_layernorm_bwd
    check(fn(dy.data_ptr(), lddy, _dt(dy), x.data_ptr(), ldx, gamma.data_ptr(), mean.data_ptr(),
             rstd.data_ptr(), _p(dx_in), dx.data_ptr(), lddx, _p(dxb), ld_dxb,
             dgamma.data_ptr(), dbeta.data_ptr(), partial.data_ptr(), rows, d, _s()), "layernorm_bwd")
    return (dx, dxb, None, None) if acc is not None else (dx, dxb, dgamma, dbeta)


def argsort_mask(noise: torch.Tensor, len_keep: int):
    n, l = noise.shape
    assert noise.dtype == torch.float32 and noise.is_contiguous()
    ids_shuffle = torch.empty(n, l, dtype=torch.int64, device=noise.device)
    ids_restore = torch.empty(n, l, dtype=torch.int64, device=noise.device)
    mask = torch.empty(n, l, dtype=torch.float32, device=noise.device)
    check(_lib.lib().vita_argsort_mask(noise.data_ptr(), n, l, len_keep, ids_shuffle.data_ptr(), ids_restore.data_ptr(),
                                       mask.data_ptr(), _s()), "argsort_mask")
    return ids_shuffle, ids_restore, mask


def row_gather(x, ldx, l_in, ids, ld_ids, l_out, nb, d, ldo, fill=None, pos=None):
    out = torch.empty(nb, l_out, ldo, dtype=torch.float32, device=x.device)
    check(_lib.lib().vita_row_gather_f32(x.data_ptr(), ldx, l_in, ids.data_ptr(), ld_ids, _p(fill), _p(pos), out.data_ptr(), ldo,
                                         l_out, nb, d, _s()), "row_gather")
    return out


def row_scatter(dout, ldo, l_out, ids, ld_ids, l_in, nb, d, ldx, want_dfill=False):
    dx = torch.zeros(nb, l_in, ldx, dtype=torch.float32, device=dout.device)
    dfill = torch.zeros(d, dtype=torch.float32, device=dout.device) if want_dfill else None
    check(_lib.lib().vita_row_scatter_f32(dout.data_ptr(), ldo, l_out, ids.data_ptr(), ld_ids, dx.data_ptr(), ldx, l_in,
                                          _p(dfill), nb, d, _s()), "row_scatter")
    return dx, dfill


def im2col(img, patch, ids, n_tok, ldo, with_cls_row=False):
    """bf16 patch matrix; with_cls_row: layout [nb][1+n_tok][ldo] with a zero row 0 per batch."""
    nb, S, T, H, W = img.shape
    assert img.dtype == torch.float32 and img.is_contiguous()
    if with_cls_row:
        out = torch.zeros(nb * (n_tok + 1), ldo, dtype=torch.bfloat16, device=img.device)
        bro, r0 = n_tok + 1, 1
    else:
        out = torch.empty(nb * n_tok, ldo, dtype=torch.bfloat16, device=img.device)
        bro, r0 = n_tok, 0
    check(_lib.lib().vita_im2col_bf16(img.data_ptr(), nb, S, T, H, W, patch[0], patch[1], patch[2], _p(ids), n_tok,
                                      out.data_ptr(), ldo, bro, r0, _s()), "im2col")
    return out


def tokens_assemble(y, ldy, cls, pos, ids, nb, n_tok, d, ldo, inplace_with_cls_row=False):
    """inplace_with_cls_row: y is [nb][1+n_tok][ldy] (row 0 = scratch) and is finished in place."""
    if inplace_with_cls_row:
        assert ldy == ldo
        out = y.view(nb, n_tok + 1, ldo)
        check(_lib.lib().vita_tokens_assemble(y.data_ptr() + 4 * ldy, ldy, cls.data_ptr(), _p(pos), _p(ids), nb, n_tok, d,
                                              out.data_ptr(), ldo, n_tok + 1, _s()), "tokens_assemble")
        return out
    out = torch.empty(nb, n_tok + 1, ldo, dtype=torch.float32, device=y.device)
    check(_lib.lib().vita_tokens_assemble(y.data_ptr(), ldy, cls.data_ptr(), _p(pos), _p(ids), nb, n_tok, d,
                                          out.data_ptr(), ldo, n_tok, _s()), "tokens_assemble")
    return out


def cast_bf16(x, ldx, rows, d, ldy):
    y = torch.empty(rows, ldy, dtype=torch.bfloat16, device=x.device)
    check(_lib.lib().vita_cast_f32_bf16(x.data_ptr(), ldx, y.data_ptr(), ldy, rows, d, _s()), "cast")
    return y


def colsum(x, ld, rows, cols, out=None, accumulate=False):
    """Column sums; accumulate=True adds them to `out` (fp32 [cols]) instead of overwriting it."""
    if out is None:
        out = torch.empty(cols, dtype=torch.float32, device=x.device)
    fn = _lib.lib().vita_colsum_acc if accumulate else _lib.lib().vita_colsum
    check(fn(x.data_ptr(), _dt(x), ld, rows, cols, out.data_ptr(), _s()), "colsum")
    return out


def softmax_rows(s, lds, p, ldp, rows, n, scale):
    check(_lib.lib().vita_softmax_rows(s.data_ptr(), lds, p.data_ptr(), ldp, rows, n, scale, _s()), "softmax_rows")


def softmax_bwd_rows(p, ldp, dp, lddp, ds, ldds, rows, n, scale):
    check(_lib.lib().vita_softmax_bwd_rows(p.data_ptr(), ldp, dp.data_ptr(), lddp, ds.data_ptr(), ldds, rows, n, scale, _s()),
          "softmax_bwd_rows")


def l2_normalize_fwd(x, eps=1e-12):
    rows, d = x.shape
    y = torch.empty_like(x); inv = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(_lib.lib().vita_l2_normalize_fwd(x.data_ptr(), rows, d, eps, y.data_ptr(), inv.data_ptr(), _s()), "l2norm_fwd")
    return y, inv


def l2_normalize_bwd(dy, y, inv):
    rows, d = y.shape
    dx = torch.empty_like(y)
    check(_lib.lib().vita_l2_normalize_bwd(dy.data_ptr(), y.data_ptr(), inv.data_ptr(), rows, d, dx.data_ptr(), _s()), "l2norm_bwd")
    return dx


def sgemm(a, b, c, m, n, k, lda, ldb, ldc, a_layout=0, b_layout=0, alpha=1.0, beta=0.0):
    check(_lib.lib().vita_sgemm_f32(a.data_ptr(), b.data_ptr(), c.data_ptr(), m, n, k, lda, ldb, ldc, a_layout, b_layout,
                                    alpha, beta, _s()), "sgemm")
    return c


def ce_rows(logits, ld, rows, cols, label_offset, weight, loss, dlogits=None, row_lse=None):
    check(_lib.lib().vita_ce_rows(logits.data_ptr(), ld, rows, cols, label_offset, weight, loss.data_ptr(), _p(row_lse),
                                  _p(dlogits), ld if dlogits is None else dlogits.stride(0), _s()), "ce_rows")


def sigmoid_mse_patch(z, ldz, img, patch, mask, inv_count, loss, pred=None, dz=None, ld_dz=0):
    nb, S, T, H, W = img.shape
    check(_lib.lib().vita_sigmoid_mse_patch(z.data_ptr(), ldz, img.data_ptr(), nb, S, T, H, W, patch[0], patch[1], patch[2],
                                            _p(mask), inv_count, _p(pred), loss.data_ptr(), _p(dz), ld_dz, _s()), "sigmoid_mse_patch")


def tabular_embed_fwd(x, wptr, bptr, n_class, cls, pos, D, ldo):
    """x fp32 [B, F] -> fp32 [B, 1+F, ldo] (cls row, per-feature tokens, + pos-embed; pads zero)."""
    B, F = x.shape
    out = torch.empty(B, F + 1, ldo, dtype=torch.float32, device=x.device)
    check(_lib.lib().vita_tabular_embed_fwd(x.data_ptr(), B, F, wptr.data_ptr(), bptr.data_ptr(), n_class.data_ptr(),
                                            cls.data_ptr(), _p(pos), out.data_ptr(), ldo, D, _s()), "tabular_embed_fwd")
    return out


def tabular_embed_bwd(dout, ldo, x, n_class, gw, gb, dcls, D):
    B, F = x.shape
    check(_lib.lib().vita_tabular_embed_bwd(dout.data_ptr(), ldo, x.data_ptr(), B, F, n_class.data_ptr(), gw.data_ptr(),
                                            gb.data_ptr(), _p(dcls), D, _s()), "tabular_embed_bwd")


def token_mean_fwd(xp, D):
    B, N, ld = xp.shape
    out = torch.empty(B, D, dtype=torch.float32, device=xp.device)
    check(_lib.lib().vita_token_mean_fwd(xp.data_ptr(), ld, B, N, D, out.data_ptr(), _s()), "token_mean_fwd")
    return out


def token_mean_bwd(dy, B, N, D, ld):
    dx = torch.empty(B, N, ld, dtype=torch.float32, device=dy.device)
    check(_lib.lib().vita_token_mean_bwd(dy.data_ptr(), B, N, D, dx.data_ptr(), ld, _s()), "token_mean_bwd")
    return dx


def batchnorm_fwd(x, gamma, beta, eps, relu, running_mean=None, running_var=None, momentum=0.1):
    B, D = x.shape
    y = torch.empty_like(x)
    mean = torch.empty(D, dtype=torch.float32, device=x.device); rstd = torch.empty_like(mean)
    check(_lib.lib().vita_batchnorm_fwd(x.data_ptr(), B, D, _p(gamma), _p(beta), eps, int(relu), y.data_ptr(), mean.data_ptr(),
                                        rstd.data_ptr(), _p(running_mean), _p(running_var), momentum, _s()), "batchnorm_fwd")
    return y, mean, rstd


def batchnorm_eval(x, gamma, beta, eps, relu, running_mean, running_var):
    B, D = x.shape
    y = torch.empty_like(x)
    check(_lib.lib().vita_batchnorm_eval(x.data_ptr(), B, D, _p(gamma), _p(beta), eps, int(relu), running_mean.data_ptr(),
                                         running_var.data_ptr(), y.data_ptr(), _s()), "batchnorm_eval")
    return y


def batchnorm_bwd(dy, x, y, gamma, mean, rstd, relu):
    B, D = x.shape
    dx = torch.empty_like(x)
    dgamma = torch.empty(D, dtype=torch.float32, device=x.device); dbeta = torch.empty_like(dgamma)
    check(_lib.lib().vita_batchnorm_bwd(dy.data_ptr(), x.data_ptr(), y.data_ptr(), B, D, _p(gamma), mean.data_ptr(),
                                        rstd.data_ptr(), int(relu), dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), _s()),
          "batchnorm_bwd")
    return dx, dgamma, dbeta


def add_bias_rows(out, bias):
    rows, D = out.shape
    check(_lib.lib().vita_add_bias_rows(out.data_ptr(), rows, D, bias.data_ptr(), _s()), "add_bias_rows")
    return out


def colsum_small(x):
    rows, D = x.shape
    out = torch.empty(D, dtype=torch.float32, device=x.device)
    check(_lib.lib().vita_colsum_small_f32(x.data_ptr(), rows, D, out.data_ptr(), _s()), "colsum_small")
    return out


def adam_step(p, g, m, v, lr, beta1, beta2, eps, weight_decay, grad_scale, step):
    check(_lib.lib().vita_adam_step(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(), lr, beta1, beta2, eps,
                                    weight_decay, grad_scale, step, _s()), "adam_step")


def attn_supported(hd, hdp):
    return bool(_lib.lib().vita_attn_supported(hd, hdp))


def attn_fwd(qkv, o, lse, B, N, H, hd, hdp, scale, tail_split=True):
    ws, ws_bytes = None, 0
    if tail_split:          # scratch for the split tail launch (fixed size, reused by the caching allocator)
        ws_bytes = _lib.lib().vita_attn_fwd_ws_bytes(hdp)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
    with _Timed("attn_fwd_kernel", 4.0 * B * H * N * N * hd):
        check(_lib.lib().vita_attn_fwd(qkv.data_ptr(), o.data_ptr(), lse.data_ptr(), _p(ws), ws_bytes, B, N, H, hd, hdp, scale,
                                       _s()), "attn_fwd")


ATTN_DS_HANDOFF = True      # dS tiles through HBM scratch (B*H*N^2*2 B): dQ without the S / dP recompute


def attn_bwd(qkv, o, do, lse, dqkv, B, N, H, hd, hdp, scale, handoff=None):
    delta = torch.empty(B, H, 2, N, dtype=torch.float32, device=qkv.device)   # [lse | rowsum(dO*O)] scratch
    ws, ws_bytes = None, 0
    if ATTN_DS_HANDOFF if handoff is None else handoff:
        ws_bytes = _lib.lib().vita_attn_bwd_ws_bytes(B, N, H, hdp)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
    # algorithmic work = the four products the reference's backward performs (dV, dP, dQ, dK: 2x the forward,
    # SURVEY 8(d) "step = 3x fwd"); the S recompute of the fused kernels is overhead, not counted
    with _Timed("attn_bwd_kernels", 8.0 * B * H * N * N * hd):
        check(_lib.lib().vita_attn_bwd(qkv.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(), delta.data_ptr(),
                                       dqkv.data_ptr(), _p(ws), ws_bytes, B, N, H, hd, hdp, scale, _s()), "attn_bwd")


# ----------------------------------------------------------------------------- 8-bit activation checkpoints, residual norms
# Unlike the wrappers above these take ordinary 2-D tensors (rows of any stride the kernels can read) and check them: type,
# device (the current one, whose current stream the kernels run on), last dimension contiguous, 16-byte aligned rows.
class Act8(NamedTuple):
    """[rows, d] values in 8 bits: e4m3 codes in groups of 32 columns with one power-of-two scale (e8m0) each.
    value = code * scale, exact in bf16.  q float8_e4m3fn [rows, round_up(d, 32)], scale float8_e8m0fnu [rows, ceil(d / 32)]."""
    q: torch.Tensor
    scale: torch.Tensor
    d: int

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.scale.numel()


class AddNorm(NamedTuple):
    """What addnorm_fwd made: y / sum are [rows, ld] with zero columns behind d, None where not asked for."""
    y: Optional[torch.Tensor]
    sum: Optional[torch.Tensor]
    act: Optional[Act8]
    mean: Optional[torch.Tensor]
    rstd: torch.Tensor


_KINDS = {"rms": 0, "layer": 1}
_PACKS = {None: 0, "normed": 0, "output": 1}


_STEP = {torch.bfloat16: 8, torch.float32: 4}         # elements of 16 bytes
_FLOATS = (torch.bfloat16, torch.float32)
_BF16 = (torch.bfloat16,)


def _on_current_device(t, what):
    if not t.is_cuda:
        raise RuntimeError(f"vita_amd: {what} is on {t.device}; these operators run on an MI355X only (no CPU fallback)")
    if t.get_device() != torch.cuda.current_device():
        raise RuntimeError(f"vita_amd: {what} is on cuda:{t.get_device()} but the current device is cuda:{torch.cuda.current_device()}")


def _mat(t, what, rows=None, d=None, dtypes=_FLOATS):
    """Checks a [rows, d] matrix and returns its row stride in elements."""
    if isinstance(t, torch.Tensor) and t.dim() == 2 and t.dtype in dtypes and t.is_cuda:
        n, c = t.shape
        ld, one = t.stride()
        step = _STEP[t.dtype]
        if n == 1:
            ld = rup(c, step)                          # the only row's stride says nothing
        if (n and c and (rows is None or n == rows) and (d is None or c == d) and t.get_device() == torch._C._cuda_getDevice()
                and (one == 1 or c == 1) and ld >= c and ld % step == 0 and t.data_ptr() % 16 == 0):
            return ld
    return _refuse_mat(t, what, rows, d, dtypes)


def _refuse_mat(t, what, rows, d, dtypes):
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"vita_amd: {what} must be a 2-D tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"vita_amd: {what} has dtype {t.dtype}, expected one of {[str(x) for x in dtypes]}")
    if t.shape[0] == 0 or t.shape[1] == 0:
        raise ValueError(f"vita_amd: {what} is empty: {tuple(t.shape)}")
    if (rows is not None and t.shape[0] != rows) or (d is not None and t.shape[1] != d):
        raise ValueError(f"vita_amd: {what} has shape {tuple(t.shape)}, expected {(rows, d)}")
    _on_current_device(t, what)
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"vita_amd: {what} must be contiguous along its last dimension (strides {t.stride()})")
    raise ValueError(f"vita_amd: rows of {what} must start on 16-byte boundaries and must not overlap (strides {t.stride()}, "
                     f"address % 16 = {t.data_ptr() % 16}); pad the row length to a multiple of {_STEP[t.dtype]}")


def _vec(t, what, n):
    """Checks an fp32 vector of n elements and returns its address (None passes)."""
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"vita_amd: {what} must be a contiguous float32 tensor of {n} elements, got {t.dtype} {tuple(t.shape)}")
    if not t.is_cuda or t.get_device() != torch._C._cuda_getDevice():
        _on_current_device(t, what)
    return t.data_ptr()


def _new_act(rows, d, device):
    """An empty checkpoint and what the C entries take of it: (Act8, (q pointer, ldq, scale pointer, lds))."""
    g = (d + 31) // 32
    q = torch.empty(rows, 32 * g, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty(rows, g, dtype=torch.float8_e8m0fnu, device=device)
    return Act8(q, scale, d), (q.data_ptr(), 32 * g, scale.data_ptr(), g)


def _act(a, what, rows=None):
    """Checks a checkpoint and returns (q pointer, ldq, scale pointer, lds)."""
    if isinstance(a, Act8) and a.d > 0:
        q, scale, d = a
        g = (d + 31) // 32
        if (q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float8_e8m0fnu and q.dim() == 2 and scale.dim() == 2 and q.is_cuda
                and scale.is_cuda):
            n = q.shape[0] if rows is None else rows
            (ldq, q1), (lds, s1) = q.stride(), scale.stride()
            if n == 1:
                ldq, lds = 32 * g, g
            if (n and tuple(q.shape) == (n, 32 * g) and tuple(scale.shape) == (n, g) and q1 == 1 and (s1 == 1 or g == 1) and ldq >= 32 * g
                    and lds >= g and ldq % 16 == 0 and q.data_ptr() % 16 == 0 and q.get_device() == scale.get_device() == torch._C._cuda_getDevice()):
                return q.data_ptr(), ldq, scale.data_ptr(), lds
    return _refuse_act(a, what, rows)


def _refuse_act(a, what, rows):
    if not isinstance(a, Act8):
        raise TypeError(f"vita_amd: {what} must be an Act8")
    if a.d < 1:
        raise ValueError(f"vita_amd: {what} is empty")
    g = rup(a.d, 32) // 32
    for t, n, dt, name in ((a.q, 32 * g, torch.float8_e4m3fn, "codes"), (a.scale, g, torch.float8_e8m0fnu, "scales")):
        if t.dtype != dt or t.dim() != 2 or t.shape[1] != n or t.shape[0] == 0 or t.shape[0] != (rows if rows is not None else a.q.shape[0]):
            raise ValueError(f"vita_amd: {name} of {what} must be {dt} [{rows if rows is not None else 'rows'}, {n}], got {t.dtype} "
                             f"{tuple(t.shape)}")
    for t, name in ((a.q, "codes"), (a.scale, "scales")):
        _on_current_device(t, f"{name} of {what}")
    raise ValueError(f"vita_amd: rows of {what} must be contiguous, must not overlap, and code rows must start on 16-byte boundaries (strides "
                     f"{a.q.stride()}, {a.scale.stride()})")


def _ld_out(ld, d, step, what):
    if ld is None:
        return (d + step - 1) // step * step
    if ld < d or ld % step:
        raise ValueError(f"vita_amd: {what} = {ld} must be a multiple of {step} and at least {d}")
    return int(ld)


def act8_pack(x) -> Act8:
    """x bf16 | fp32 [rows, d] -> its 8-bit checkpoint."""
    ld = _mat(x, "x")
    rows, d = x.shape
    a, ap = _new_act(rows, d, x.device)
    check(_lib.lib().vita_act8_pack(x.data_ptr(), _dt(x), ld, rows, d, *ap, _s()), "act8_pack")
    return a


def act8_unpack(act: Act8, gamma=None, beta=None, dtype=torch.bfloat16, ldo=None):
    """The values of a checkpoint (* gamma + beta per column) as [rows, ldo], zero behind column d.  bf16 without gamma is exact."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"vita_amd: unsupported dtype {dtype}")
    if beta is not None and gamma is None:
        raise ValueError("vita_amd: beta needs gamma")
    q = _act(act, "act")
    rows, d = act.q.shape[0], act.d
    ldo = _ld_out(ldo, d, 8, "ldo")
    gp, bp = _vec(gamma, "gamma", d), _vec(beta, "beta", d)
    y = torch.empty(rows, ldo, dtype=dtype, device=act.q.device)
    check(_lib.lib().vita_act8_unpack(*q, rows, d, gp, bp, y.data_ptr(), _dt(y), ldo, _s()), "act8_unpack")
    return y


def gelu_act8_fwd(z, ldg=None):
    """z bf16 | fp32 [rows, d] -> (GELU(z) bf16 [rows, ldg] with zero pads, the 8-bit checkpoint of z)."""
    ld = _mat(z, "z")
    rows, d = z.shape
    ldg = _ld_out(ldg, d, 8, "ldg")
    g = torch.empty(rows, ldg, dtype=torch.bfloat16, device=z.device)
    a, ap = _new_act(rows, d, z.device)
    check(_lib.lib().vita_gelu_act8_fwd(z.data_ptr(), _dt(z), ld, rows, d, g.data_ptr(), ldg, *ap, _s()), "gelu_act8_fwd")
    return g, a


def gelu_act8_bwd(dg, act: Act8, want_g=True, ldo=None):
    """(dg * GELU'(z) bf16 [rows, ldo], GELU(z) bf16 [rows, ldo] or None), z from its checkpoint; zero pads."""
    q = _act(act, "act")
    rows, d = act.q.shape[0], act.d
    ld = _mat(dg, "dg", rows, d, _BF16)
    ldo = _ld_out(ldo, d, 8, "ldo")
    dz = torch.empty(rows, ldo, dtype=torch.bfloat16, device=dg.device)
    g = torch.empty_like(dz) if want_g else None
    check(_lib.lib().vita_gelu_act8_bwd(dg.data_ptr(), ld, *q, rows, d, dz.data_ptr(), ldo, _p(g), ldo if want_g else 0, _s()),
          "gelu_act8_bwd")
    return dz, g


def act8_wgrad(dy, act: Act8, out=None):
    """dW fp32 [m, d] = dy^T x over the rows, from x's checkpoint; dy bf16 [rows, m].  out: a contiguous fp32 [m, d] to ADD it to."""
    q = _act(act, "act")
    k, n = act.q.shape[0], act.d
    m = dy.shape[-1]
    ld = _mat(dy, "dy", k, m, _BF16)
    if out is not None and out.shape != (m, n):
        raise ValueError(f"vita_amd: out has shape {tuple(out.shape)}, expected {(m, n)}")
    _vec(out, "out", m * n)
    dw = torch.empty(m, n, dtype=torch.float32, device=dy.device) if out is None else out
    qp, ldq, sp, lds = q
    # the kernel's offsets inside a call are 32 bits: longer sums go in several calls (whole K-tiles, five of them to spare)
    most = max(0x7ffffe00 // max(2 * ld, ldq, lds) // 64 * 64 - 320, 64)
    with _Timed("act8_wgrad", 2.0 * m * n * k):
        for r in range(0, k, most):
            rows = min(most, k - r)
            ws_bytes = _lib.lib().vita_act8_wgrad_ws_bytes(m, n, rows)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dy.device) if ws_bytes else None
            check(_lib.lib().vita_act8_wgrad(dy.data_ptr() + 2 * r * ld, ld, qp + r * ldq, ldq, sp + r * lds, lds, dw.data_ptr(), n, m, n,
                                             rows, int(out is not None or r > 0), _p(ws), ws_bytes, _s()), "act8_wgrad")
    return dw


def addnorm_fwd(x, gamma=None, beta=None, residual=None, kind="rms", eps=1e-6, y_dtype=torch.bfloat16, sum_dtype=None, pack=None,
                ldy=None) -> AddNorm:
    """Norm of x (+ residual) over the last dimension, kind "rms" or "layer": y_dtype bf16 | fp32 | None, sum_dtype to also get the
    sum, pack "normed" (the rows before gamma: addnorm_bwd's source) or "output" (y itself) for an 8-bit copy."""
    if kind not in _KINDS or pack not in _PACKS:
        raise ValueError(f"vita_amd: kind {kind!r} / pack {pack!r}: expected kind in {list(_KINDS)}, pack in {list(_PACKS)}")
    if beta is not None and gamma is None:
        raise ValueError("vita_amd: beta needs gamma")
    if sum_dtype is not None and residual is None:
        raise ValueError("vita_amd: sum_dtype needs a residual")
    if y_dtype is None and pack is None:
        raise ValueError("vita_amd: nothing to compute (no y, no pack)")
    for t in (y_dtype, sum_dtype):
        if t not in (None, torch.bfloat16, torch.float32):
            raise TypeError(f"vita_amd: unsupported dtype {t}")
    ldx = _mat(x, "x")
    rows, d = x.shape
    dev = x.device
    ldr = 0 if residual is None else _mat(residual, "residual", rows, d)
    gp, bp = _vec(gamma, "gamma", d), _vec(beta, "beta", d)
    ld = _ld_out(ldy, d, 8, "ldy")
    y = torch.empty(rows, ld, dtype=y_dtype, device=dev) if y_dtype is not None else None
    s = torch.empty(rows, ld, dtype=sum_dtype, device=dev) if sum_dtype is not None else None
    a, ap = _new_act(rows, d, dev) if pack is not None else (None, (None, 0, None, 0))
    rstd = torch.empty(rows, dtype=torch.float32, device=dev)
    mean = torch.empty(rows, dtype=torch.float32, device=dev) if kind == "layer" else None
    c = AddNormFwdDesc(x.data_ptr(), _p(residual), _p(s), gp, bp, _p(y), ap[0], ap[2], _p(mean), rstd.data_ptr(), rows, d,
                       ldx, ldr, ld, ld, ap[1], ap[3], _KINDS[kind], _PACKS[pack], _dt(x), _dt(residual) if residual is not None else 0,
                       _dt(s) if s is not None else 0, _dt(y) if y is not None else 0, eps)
    check(_lib.lib().vita_addnorm_fwd(C.byref(c), _s()), "addnorm_fwd")
    return AddNorm(y, s, a, mean, rstd)


def addnorm_bwd(dy, src, rstd, gamma=None, kind="rms", mean=None, dx_in=None, dx_dtype=torch.float32, lddx=None, want_bf16=False,
                want_dgamma=True, want_dbeta=None, acc=None):
    """(dx [rows, lddx], dgamma, dbeta) of addnorm_fwd; src = its Act8 ("normed") or its sum (then with mean for "layer").
    dx is the gradient of x and of the residual, dx_in [rows, d] of type dx_dtype is added to it.  want_bf16: dx becomes the pair
    (dx, bf16 copy).  acc = (dgamma_buf, dbeta_buf or None): fp32 [d] buffers the sums are ADDED to; None is returned for them."""
    if kind not in _KINDS:
        raise ValueError(f"vita_amd: kind {kind!r}: expected one of {list(_KINDS)}")
    if dx_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"vita_amd: unsupported dtype {dx_dtype}")
    sp = mp = None
    ldx = src_dt = 0
    ap = (None, 0, None, 0)
    if isinstance(src, Act8):
        ap = _act(src, "src")
        rows, d = src.q.shape[0], src.d
    else:
        ldx = _mat(src, "src")
        rows, d = src.shape
        sp, src_dt = src.data_ptr(), _dt(src)
        if kind == "layer":
            if mean is None:
                raise ValueError("vita_amd: the layer norm's gradient from the sum needs mean")
            mp = _vec(mean, "mean", rows)
    lddy = _mat(dy, "dy", rows, d)
    dev = dy.device
    rp, gp = _vec(rstd, "rstd", rows), _vec(gamma, "gamma", d)
    if rp is None:
        raise ValueError("vita_amd: rstd is missing")
    ldin = 0 if dx_in is None else _mat(dx_in, "dx_in", rows, d, (dx_dtype,))
    ld = _ld_out(lddx, d, 8, "lddx")
    dgamma = dbeta = None
    if acc is not None:
        dg, db = acc
    else:
        want_dbeta = kind == "layer" if want_dbeta is None else want_dbeta
        dg = dgamma = torch.empty(d, dtype=torch.float32, device=dev) if want_dgamma else None
        db = dbeta = torch.empty(d, dtype=torch.float32, device=dev) if want_dbeta else None
    if kind == "rms" and db is not None:
        raise ValueError("vita_amd: the rms norm has no beta")
    dgp, dbp = _vec(dg, "dgamma", d), _vec(db, "dbeta", d)
    dx = torch.empty(rows, ld, dtype=dx_dtype, device=dev)
    dxb = torch.empty(rows, ld, dtype=torch.bfloat16, device=dev) if want_bf16 else None
    partial = None
    if dg is not None or db is not None:
        partial = torch.empty(2 * _lib.lib().vita_addnorm_bwd_nblk(rows, d) * d, dtype=torch.float32, device=dev)
    c = AddNormBwdDesc(dy.data_ptr(), sp, ap[0], ap[2], mp, rp, gp, _p(dx_in), dx.data_ptr(), _p(dxb), dgp, dbp, _p(partial), rows, d,
                       lddy, ldx, ap[1], ap[3], ldin, ld, ld, _KINDS[kind], int(acc is not None), _dt(dy), src_dt, _dt(dx))
    check(_lib.lib().vita_addnorm_bwd(C.byref(c), _s()), "addnorm_bwd")
    return (dx, dxb) if want_bf16 else dx, dgamma, dbeta
