"""RMSNorm with the adaLN modulation fused in (forward and backward), the head's LayerNorm, and RMSNorm with the
residual's addition (bf16 or MXFP8 output, and its gradient).

Forward  h = bf16( w * x * rstd * (1 + scale[g]) + shift[g] ),  rstd = 1 / sqrt(mean(x^2) + eps),  g = row // rows_per_group
Backward with u = w * x * rstd:
    d_shift[g] = sum_rows dh          d_scale[g] = sum_rows dh * u           du = dh * (1 + scale[g])
    d_w        = sum_all_rows du * x * rstd                                    dxn = du * w
    dx         = rstd * (dxn - x * rstd * mean(dxn * x * rstd)) (+ d_residual)
Column sums are deterministic: fixed-order partials per chunk of rows, then a fixed-order reduction.

Reference sites: RMSNorm (baselines/PixelGen/src/models/layers/rmsnorm.py:5-20, fp32 math cast back) composed with
`modulate` (JiT_T2I.py:75-76) in FlattenDiTBlock/TextRefineBlock (JiT_T2I.py:201-210, 279-293), and the Triton fused
norm of the reference's lever K (baselines/PixelGen/src/models/layers/fused_norm.py:64-140), which does the same sums.
"""
import torch

from .._ext import ext
from .elementwise import Segments, _rows


def rms_mod_fwd(x, w, shift=None, scale=None, rows_per_group=1, eps=1e-6):
    """x [M, C] bf16, w [C] fp32, shift/scale [G, C] bf16 views (row stride free) or None.
    Returns (h [M, C] bf16, rstd [M] fp32)."""
    M, C = x.shape
    if not x.is_cuda:
        xf = x.float()
        rstd = torch.rsqrt(xf.pow(2).mean(-1) + eps)
        u = w.float() * xf * rstd[:, None]
        if scale is not None:
            sc = _rows(rows_per_group, scale.float(), M)
            sh = _rows(rows_per_group, shift.float(), M)
            u = u * (1 + sc) + sh
        return u.to(torch.bfloat16), rstd
    h = torch.empty_like(x)
    rstd = torch.empty(M, device=x.device, dtype=torch.float32)
    if isinstance(rows_per_group, Segments):
        ext().rms_mod_fwd(x, w, shift, scale, h, rstd, 1, eps, rows_per_group.seg)
    else:
        ext().rms_mod_fwd(x, w, shift, scale, h, rstd, rows_per_group, eps, None)
    return h, rstd


def rms_mod_fwd_mx(x, w, shift=None, scale=None, rows_per_group=1, eps=1e-6):
    """rms_mod_fwd that also returns h's MXFP8 copy (ops.mx.MX) from the same kernel: (h, rstd, hq). C % 128 == 0."""
    from . import mx
    if not x.is_cuda:
        h, rstd = rms_mod_fwd(x, w, shift, scale, rows_per_group, eps)
        return h, rstd, mx.quant(h)
    M, C = x.shape
    h = torch.empty_like(x)
    rstd = torch.empty(M, device=x.device, dtype=torch.float32)
    q = torch.empty(M, C, device=x.device, dtype=torch.uint8)
    rp = mx.rows_pad(M)
    shape = (rp // 128, C // 128, 512)
    if rp == M:
        sf = torch.empty(shape, device=x.device, dtype=torch.uint8)
    else:  # rows past M (up to the 256-row padding) keep scale 1
        sf = torch.full(shape, 127, device=x.device, dtype=torch.uint8)
    ext().rms_mod_fwd_mx(x, w, shift, scale, h, rstd, q, sf, rows_per_group, eps)
    return h, rstd, mx.MX(q, sf)


def rms_mod_bwd(dh, x, rstd, w, scale=None, rows_per_group=1, dres=None, dw_acc=None, dshift=None, dscale=None):
    """Backward of rms_mod_fwd. Returns dx [M, C] bf16 (plus dres when given).
    dw_acc [C] fp32: d_w is added into it. dshift/dscale [G, C] fp32 views: overwritten (None: not computed).
    rows_per_group may be a Segments (packed rows): rows of no sample then get dx = 0 and add nothing to d_w."""
    M, C = x.shape
    seg = rows_per_group if isinstance(rows_per_group, Segments) else None
    if not x.is_cuda:
        xf, dhf = x.float(), dh.float()
        if seg is not None:
            dhf = dhf * seg.owned(M, dhf.device)[:, None].float()
        xn = xf * rstd[:, None]
        u = w.float() * xn
        if scale is not None:
            G = scale.shape[0]
            sc = _rows(rows_per_group, scale.float(), M)
            du = dhf * (1 + sc)
            if dshift is not None:
                if seg is not None:
                    dshift[:seg.groups].copy_(seg.sum_rows(dhf))
                else:
                    dshift.copy_(dhf.view(G, rows_per_group, C).sum(1))
            if dscale is not None:
                if seg is not None:
                    dscale[:seg.groups].copy_(seg.sum_rows(dhf * u))
                else:
                    dscale.copy_((dhf * u).view(G, rows_per_group, C).sum(1))
        else:
            du = dhf
        if dw_acc is not None:
            dw_acc.add_((du * xn).sum(0))
        dxn = du * w.float()
        dx = rstd[:, None] * (dxn - xn * (dxn * xn).mean(-1, keepdim=True))
        if dres is not None:
            dx = dx + dres.float()
        if seg is not None:
            dx = dx * seg.owned(M, dx.device)[:, None].float()
        return dx.to(torch.bfloat16)
    if seg is not None:
        dx = torch.zeros_like(x)  # rows of no sample keep a zero gradient
        ext().rms_mod_bwd(dh, x, rstd, w, scale, dres, dx, dw_acc, dshift, dscale, 1, seg.cu, seg.max_rows)
        return dx
    dx = torch.empty_like(x)
    ext().rms_mod_bwd(dh, x, rstd, w, scale, dres, dx, dw_acc, dshift, dscale, rows_per_group, None, 0)
    return dx


def _add_rms_check(x, res, w):
    M, C = x.shape
    if C % 8 or not 0 < C <= 16384:
        raise RuntimeError(f"add_rms: the width must be a multiple of 8 up to 16384, got {C}")
    if res.shape != x.shape or w.shape != (C,):
        raise RuntimeError(f"add_rms: res must be {list(x.shape)} and w [{C}], got {list(res.shape)}, {list(w.shape)}")
    if res.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError("add_rms: res must be bf16 or fp32")


def _add_rms_cpu(x, res, w, eps):
    _add_rms_check(x, res, w)
    s = res.float() + x.float()
    rstd = torch.rsqrt(s.pow(2).mean(-1) + eps)
    return s * rstd[:, None] * w.float(), s.to(res.dtype), rstd


def add_rms_fwd(x, res, w, eps=1e-6):
    """RMSNorm with the residual's addition in front (the pre-norm blocks of a language model), one pass:
        s = res + x,  rstd = 1 / sqrt(mean(s^2) + eps),  h = bf16(w * s * rstd)
    x [M, C] bf16 and res [M, C] bf16 or fp32 (the residual stream), row strides free, rows 16-byte aligned; w [C]
    fp32;
    C a multiple of 8 up to 16384. Returns (h [M, C] bf16, s [M, C] in res's type, rstd [M] fp32). h and rstd come from
    the unrounded fp32 sum."""
    if not x.is_cuda:
        h, s, rstd = _add_rms_cpu(x, res, w, eps)
        return h.to(torch.bfloat16), s, rstd
    return tuple(ext().add_rms_fwd(x, res, w, eps, False))


def add_rms_fwd_mx(x, res, w, eps=1e-6):
    """add_rms_fwd with h in MXFP8 (ops.mx.MX, the input of mx.linear) instead of bf16: (hq, s, rstd). C % 128 == 0.
    h is rounded once, from fp32 (rms_mod_fwd_mx rounds through bf16, to equal a separate quantisation)."""
    from . import mx
    if not x.is_cuda:
        if x.shape[1] % 128:
            raise RuntimeError(f"add_rms: the MXFP8 output needs a width that is a multiple of 128, got {x.shape[1]}")
        h, s, rstd = _add_rms_cpu(x, res, w, eps)
        return mx.quant(h), s, rstd
    q, sf, s, rstd = ext().add_rms_fwd(x, res, w, eps, True)
    return mx.MX(q, sf), s, rstd


def add_rms_bwd(dh, ds, s, rstd, w, dw_acc=None):
    """Gradient of add_rms_fwd: dh [M, C] bf16 (of h), ds [M, C] in s's type (of s as the later blocks read it) or None,
    s and rstd as the forward returned them. Returns dx [M, C] in s's type, the gradient of x and of res alike:
        xn = s * rstd, dxn = dh * w, dx = rstd * (dxn - xn * mean(dxn * xn)) + ds
    dw_acc [C] fp32: sum over rows of dh * xn is added into it (fixed order: the same inputs give the same bits). For a
    bf16 stream this is rms_mod_bwd without modulation, dres = ds."""
    if not dh.is_cuda:
        _add_rms_check(dh, s, w)
        xn = s.float() * rstd[:, None]
        if dw_acc is not None:
            dw_acc.add_((dh.float() * xn).sum(0))
        dxn = dh.float() * w.float()
        dx = rstd[:, None] * (dxn - xn * (dxn * xn).mean(-1, keepdim=True))
        if ds is not None:
            dx = dx + ds.float()
        return dx.to(s.dtype)
    return ext().add_rms_bwd(dh, ds, s, rstd, w, dw_acc)


def layernorm_fwd(x, eps=1e-6):
    """LayerNorm without affine parameters (the head's norm_final, JiT_T2I.py:345-357): fp32 statistics.
    x [M, C] bf16 -> (h [M, C] bf16, mean [M], rstd [M])."""
    if not x.is_cuda:
        xf = x.float()
        mu = xf.mean(-1)
        var = (xf - mu[:, None]).pow(2).mean(-1)
        rstd = torch.rsqrt(var + eps)
        return ((xf - mu[:, None]) * rstd[:, None]).to(torch.bfloat16), mu, rstd
    M, C = x.shape
    h = torch.empty_like(x)
    mu = torch.empty(M, device=x.device, dtype=torch.float32)
    rstd = torch.empty(M, device=x.device, dtype=torch.float32)
    ext().layernorm_fwd(x, h, mu, rstd, eps)
    return h, mu, rstd


def layernorm_bwd(dh, x, mu, rstd):
    """dx = rstd * (dh - mean(dh) - xhat * mean(dh * xhat)) for LayerNorm without affine."""
    if not x.is_cuda:
        xh = (x.float() - mu[:, None]) * rstd[:, None]
        d = dh.float()
        dx = rstd[:, None] * (d - d.mean(-1, keepdim=True) - xh * (d * xh).mean(-1, keepdim=True))
        return dx.to(torch.bfloat16)
    dx = torch.empty_like(x)
    ext().layernorm_bwd(dh, x, mu, rstd, dx)
    return dx
