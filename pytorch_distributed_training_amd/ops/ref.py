"""Pure-PyTorch fp32 reference implementation of every engine op.

This backend has two jobs: it is the numerical oracle the HIP kernels are tested
against (same signatures, same tensor layouts), and it is what the engine runs on when
there is no GPU (CPU / gloo plumbing tests).  Every function up-casts its inputs to fp32,
computes with stock ``torch`` ops and rounds the result to the activation dtype.

Layouts: activations are NHWC ``[B, H, W, C]`` contiguous; convolution weights are OHWI
``[Cout, R, S, Cin]``; per-channel vectors are fp32.

The ops correspond to the kernels PyTorch dispatches implicitly for the upstream trainer's
``model(img)`` / ``loss.backward()`` / ``optimizer.step()`` (reference
``train_distributed.py:274-277``): convolution forward / data-gradient / weight-gradient,
(Sync)BatchNorm statistics / apply / backward-reduce / backward-elementwise
(``torch/nn/modules/_functions.py:39-179``), max/avg pooling, the classifier GEMM,
softmax cross-entropy, SGD with momentum (``torch/optim/sgd.py:322-367``) and top-k.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

name = "ref"
# conv_dgrad reads the forward weights ``w`` (an update of them must wait until backward is over)
dgrad_reads_forward_weights = True

MASK_NONE = 0       # dy = g
MASK_TENSOR = 1     # dy = g * (mask_src > 0)
MASK_RECOMPUTE = 2  # dy = g * (y * scale + shift > 0)


def _nchw(x: torch.Tensor) -> torch.Tensor:
    return x.permute(0, 3, 1, 2)


def _nhwc(x: torch.Tensor) -> torch.Tensor:
    return x.permute(0, 2, 3, 1).contiguous()


def _w_oihw(w: torch.Tensor) -> torch.Tensor:
    return w.permute(0, 3, 1, 2)


def channel_moments(y32: torch.Tensor, shift: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[2, C]``: per-channel SHIFTED moments ``E[y - s]`` and ``E[(y - s)^2]``.

    ``s`` is a per-channel shift (the BatchNorm running mean; zero when ``None``).  Shifted
    moments are what ranks exchange for SyncBatchNorm: running means are identical on all
    ranks and per-rank counts are equal, so the global moments are the plain average of the
    local ones -- ONE sum all-reduce of ``2C`` floats -- and the variance
    ``E[(y-s)^2] - E[y-s]^2`` only suffers cancellation if the batch mean is many standard
    deviations away from the running mean.
    """
    flat = y32.reshape(-1, y32.shape[-1])
    if shift is not None:
        flat = flat - shift
    var, mean = torch.var_mean(flat, dim=0, unbiased=False)
    return torch.stack([mean, var + mean * mean])


# ---------------------------------------------------------------------------- input
def input_transform(img: torch.Tensor, mean: torch.Tensor, std: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Loader batch -> stem input.

    ``img`` is either float NCHW, already normalised (the upstream loader contract,
    reference ``train_distributed.py:272``), or uint8 NHWC raw pixels, normalised here
    with ``(x/255 - mean) / std``.  Returns NHWC ``[B, H, W, 3]`` in ``dtype``.
    """
    if img.dtype == torch.uint8:
        x = img.float().div_(255.0)
        x = (x - mean.view(1, 1, 1, 3)) / std.view(1, 1, 1, 3)
        return x.to(dtype).contiguous()
    return _nhwc(img.float()).to(dtype)


def crop_resize_flip(src: torch.Tensor, boxes: torch.Tensor, out_size: int) -> torch.Tensor:
    """``src [B, S, S, 3]`` uint8, ``boxes [B, 5]`` int32 ``(x, y, w, h, flip)`` -> ``[B, out, out, 3]`` uint8:
    bilinear resize (half-pixel centres, no antialiasing) of each box, then the horizontal flip."""
    outs = []
    for img, (x, y, w, h, flip) in zip(src, boxes.tolist()):
        crop = img[y:y + h, x:x + w].permute(2, 0, 1).unsqueeze(0).float()
        r = F.interpolate(crop, size=(out_size, out_size), mode="bilinear", align_corners=False)
        r = (r + 0.5).floor().clamp_(0, 255).to(torch.uint8)[0].permute(1, 2, 0)
        outs.append(r.flip(1) if flip else r)
    return torch.stack(outs).contiguous()


def prepare_stem_weight(w: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Compute-side stem weights from the ``[64, 7, 7, 3]`` compute-dtype view (identity here)."""
    return w


def stem_fprop(x0: torch.Tensor, w: torch.Tensor, stat_shift: Optional[torch.Tensor] = None):
    return conv_fprop(x0, w, 7, 7, 2, 3, stat_shift)


def stem_wgrad(x0: torch.Tensor, dy: torch.Tensor, dw: torch.Tensor) -> None:
    conv_wgrad(x0, dy, 7, 7, 2, 3, dw)


# ---------------------------------------------------------------------------- convolution
def conv_fprop(x: torch.Tensor, w: torch.Tensor, R: int, S: int, stride: int, pad: int,
               stat_shift: Optional[torch.Tensor] = None, **_) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``y = conv(x, w)``; when ``stat_shift`` is given also the shifted per-channel moments of
    the result (see :func:`channel_moments`).  Here they are taken from the fp32 result; a
    backend may take them from the rounded ``y`` it stores instead (the HIP kernel does: that is
    what a separate statistics pass over the output tensor would see)."""
    y32 = F.conv2d(_nchw(x.float()), _w_oihw(w.float()), None, stride, pad)
    y32 = _nhwc(y32)
    stats = channel_moments(y32, stat_shift) if stat_shift is not None else None
    return y32.to(x.dtype), stats


def conv_dgrad(dy: torch.Tensor, w: torch.Tensor, wt: Optional[torch.Tensor], in_shape, R: int, S: int,
               stride: int, pad: int, addend: Optional[torch.Tensor] = None,
               relu_mask: Optional[torch.Tensor] = None, relu_bits: Optional[torch.Tensor] = None,
               addend_half: bool = False, out_sums: bool = False, **_) -> torch.Tensor:
    """``dx = (conv_transpose(dy, w) [+ addend]) [* (relu_mask > 0)]`` ; ``in_shape = (B, Hi, Wi, Ci)``.
    ``relu_bits``: the same mask in packed form (see :func:`bn_apply`).

    ``addend`` accumulates the other gradient path of a residual block; ``relu_mask`` (the
    post-ReLU tensor this gradient belongs to) applies that ReLU's backward right here, so the
    consumers of ``dx`` -- the BatchNorm backward passes of the previous block -- need no mask.
    The sum is rounded to the activation dtype before the mask, like a separate add would."""
    B, Hi, Wi, Ci = in_shape
    dx = torch.nn.grad.conv2d_input((B, Ci, Hi, Wi), _w_oihw(w.float()), _nchw(dy.float()), stride, pad)
    dx = _nhwc(dx)
    dx = dx.to(dy.dtype)
    if addend is not None:
        if addend_half:          # given at the output pixels with two even coordinates only, zero elsewhere
            full = torch.zeros_like(dx)
            full[:, ::2, ::2] = addend
            addend = full
        dx = (dx.float() + addend.float()).to(dy.dtype)
    if relu_bits is not None:
        dx = dx * _unpack_bits(relu_bits)
    elif relu_mask is not None:
        dx = dx * (relu_mask > 0)
    if out_sums:         # per-channel sums of the stored result, collected by grad_sums
        _grad_sums[Ci] = dx.float().reshape(-1, Ci).sum(0)
    return dx


_grad_sums = {}


def grad_sums(C: int, device=None) -> torch.Tensor:
    """``[C]`` sums left by the last ``conv_dgrad(out_sums=True)`` with ``C`` output channels."""
    return _grad_sums.pop(C)


def colsum_take(slot: str, C: int, device=None):
    """(fused backends: the sums ``bn_apply(colsum_slot=slot)`` left behind; nothing is kept here)"""
    return None


def subsample2(x: torch.Tensor) -> torch.Tensor:
    """``x[:, ::2, ::2]`` of an NHWC tensor, dense: the pixels a stride-2 1x1 convolution reads."""
    return x[:, ::2, ::2].contiguous()


def zeros_f32(shape, device) -> torch.Tensor:
    return torch.zeros(shape, dtype=torch.float32, device=device)


def conv_wgrad(x: torch.Tensor, dy: torch.Tensor, R: int, S: int, stride: int, pad: int, dw: torch.Tensor,
               **_) -> None:
    """``dw[Cout, R, S, Cin] += x (*) dy`` (fp32 accumulate into the flat gradient buffer)."""
    Co, Ci = dy.shape[-1], x.shape[-1]
    g = torch.nn.grad.conv2d_weight(_nchw(x.float()), (Co, Ci, R, S), _nchw(dy.float()), stride, pad)
    dw.add_(g.permute(0, 2, 3, 1))


def transpose_weights(w: torch.Tensor, wt: Optional[torch.Tensor]) -> None:
    """Fill the data-gradient weight copy ``wt[Cin, R, S, Cout]`` (unused by this backend)."""
    if wt is not None:
        wt.copy_(w.permute(3, 1, 2, 0))


# ---------------------------------------------------------------------------- batch norm
def bn_stats(y: torch.Tensor, shift: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stand-alone shifted per-channel moments of an NHWC tensor."""
    return channel_moments(y.float(), shift)


def bn_finalize(moments: torch.Tensor, inv_world: float, gamma: torch.Tensor, beta: torch.Tensor,
                running_mean: torch.Tensor, running_var: torch.Tensor, momentum: float, eps: float, count: int):
    """Summed moments -> ``(scale, shift, mean, invstd)``; updates running stats in place.

    ``moments`` is the (all-reduced) SUM over ranks of the local moments shifted by
    ``running_mean`` (its value BEFORE this update) and ``inv_world = 1 / world_size`` turns
    it into the global moments.  ``scale = gamma * invstd``, ``shift = beta - mean * scale``.
    The running variance uses the unbiased estimate with the GLOBAL element count
    ``count``, as ``SyncBatchNorm`` does (``torch/nn/modules/_functions.py:106-115``).
    """
    m0 = moments[0] * inv_world
    mean = running_mean + m0
    var = (moments[1] * inv_world - m0 * m0).clamp_min(0.0)
    invstd = torch.rsqrt(var + eps)
    scale = gamma * invstd
    shift = beta - mean * scale
    unbiased = var * (count / max(count - 1, 1))
    running_mean.mul_(1.0 - momentum).add_(mean, alpha=momentum)
    running_var.mul_(1.0 - momentum).add_(unbiased, alpha=momentum)
    return scale, shift, mean, invstd


def bn_eval_affine(gamma, beta, running_mean, running_var, eps: float):
    invstd = torch.rsqrt(running_var + eps)
    scale = gamma * invstd
    return scale, beta - running_mean * scale


relu_bits = True             # bn_apply/bn_apply2(bits_out=...) and conv_dgrad(relu_bits=...)
half_addend = True           # conv_dgrad(addend_half=True)
_BIT_WEIGHTS = (1, 2, 4, 8, 16, 32, 64, 128)


def new_relu_bits(like: torch.Tensor) -> torch.Tensor:
    """Destination for the packed ReLU mask of a tensor shaped like ``like``: one byte per 8 channels."""
    return torch.empty(*like.shape[:-1], like.shape[-1] // 8, dtype=torch.uint8, device=like.device)


def _pack_bits(out: torch.Tensor, bits_out: torch.Tensor) -> None:
    w = torch.tensor(_BIT_WEIGHTS, dtype=torch.int32, device=out.device)
    on = (out > 0).to(torch.int32).reshape(*out.shape[:-1], out.shape[-1] // 8, 8)
    bits_out.copy_((on * w).sum(-1).to(torch.uint8))


def _unpack_bits(bits: torch.Tensor) -> torch.Tensor:
    w = torch.tensor(_BIT_WEIGHTS, dtype=torch.int32, device=bits.device)
    on = (bits.to(torch.int32).unsqueeze(-1) & w) != 0
    return on.reshape(*bits.shape[:-1], bits.shape[-1] * 8)


def bn_apply(y: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, residual: Optional[torch.Tensor],
             relu: bool, bits_out: Optional[torch.Tensor] = None, colsum_slot: Optional[str] = None) -> torch.Tensor:
    """``bits_out``: also receives ``[out > 0]``, bit k of byte j = channel ``8j + k``.  ``colsum_slot``: a fused
    backend leaves the per-channel sums of the result under that name for :func:`conv_wgrad_folded`; this backend
    recomputes them there."""
    out = y.float() * scale + shift
    if residual is not None:
        out = out + residual.float()
    if relu:
        out = torch.relu(out)
    out = out.to(y.dtype)
    if bits_out is not None:
        _pack_bits(out, bits_out)
    return out


def _masked(g, y32, scale, shift, mask_src, mask_mode):
    dy = g.float()
    if mask_mode == MASK_TENSOR:
        dy = dy * (mask_src.float() > 0)
    elif mask_mode == MASK_RECOMPUTE:
        dy = dy * ((y32 * scale + shift) > 0)
    return dy


def bn_apply2(y, scale, shift, y2, scale2, shift2, relu: bool, bits_out: Optional[torch.Tensor] = None):
    """``relu(y*scale + shift + y2*scale2 + shift2)`` -- a block's main path and its projection
    shortcut normalised, added and activated in one pass (one rounding to the compute dtype)."""
    out = y.float() * scale + shift + y2.float() * scale2 + shift2
    if relu:
        out = torch.relu(out)
    out = out.to(y.dtype)
    if bits_out is not None:
        _pack_bits(out, bits_out)
    return out


def bn_bwd_reduce(g, y, mean, invstd, scale, shift, mask_src, mask_mode: int,
                  dgamma: Optional[torch.Tensor] = None, dbeta: Optional[torch.Tensor] = None,
                  pool_idx=None) -> torch.Tensor:
    """``[2, C]``: local ``sum(dy)`` and ``sum(dy * xhat)`` with ``xhat = (y - mean) * invstd``.

    When given, ``dbeta += sum(dy)`` and ``dgamma += sum(dy * xhat)`` (the LOCAL sums are the
    parameter gradients; the bucketed all-reduce averages them over ranks later).
    ``pool_idx``: ``g`` is the gradient of the 3x3/s2 max pooling that follows this layer's ReLU
    (with the pooling's index tensor), not of the activation itself.
    """
    if pool_idx is not None:
        g = maxpool_bwd(g, pool_idx, tuple(y.shape))
    y32 = y.float()
    dy = _masked(g, y32, scale, shift, mask_src, mask_mode)
    xhat = (y32 - mean) * invstd
    C = y.shape[-1]
    sums = torch.stack([dy.reshape(-1, C).sum(0), (dy * xhat).reshape(-1, C).sum(0)])
    if dbeta is not None:
        dbeta.add_(sums[0])
    if dgamma is not None:
        dgamma.add_(sums[1])
    return sums


def bn_bwd_elemt(g, y, mean, invstd, scale, shift, sums, inv_count: float, mask_src, mask_mode: int,
                 pool_idx=None) -> torch.Tensor:
    """``dx = (dy - s0 - xhat * s1) * scale`` with ``[s0, s1] = sums * inv_count``.

    ``sums`` are the (all-reduced) global sums from :func:`bn_bwd_reduce` and ``inv_count`` is
    one over the GLOBAL number of elements per channel
    (``torch/nn/modules/_functions.py:170-179``).  ``pool_idx``: as in :func:`bn_bwd_reduce`.
    """
    if pool_idx is not None:
        g = maxpool_bwd(g, pool_idx, tuple(y.shape))
    y32 = y.float()
    dy = _masked(g, y32, scale, shift, mask_src, mask_mode)
    xhat = (y32 - mean) * invstd
    dx = (dy - sums[0] * inv_count - xhat * (sums[1] * inv_count)) * scale
    return dx.to(y.dtype)



# ---------------------------------------------------------------------------- folded BatchNorm backward
bn_fold = True
BN_FOLD_MAX_C = 512


class BnFold:
    __slots__ = ("wfold", "bias", "coef", "C", "N")

    def __init__(self, wfold, bias, coef, C: int, N: int) -> None:
        self.wfold, self.bias, self.coef, self.C, self.N = wfold, bias, coef, C, N

    def tensors(self):
        return self.wfold, self.bias, self.coef


def bn_fold_prepare(sums, scale, invstd, mean, inv_count: float, w: torch.Tensor, wt=None) -> BnFold:
    """BatchNorm backward folded into the 1x1 / stride 1 convolution ``y = a . w^T`` in front of it.

    With the reduced sums of :func:`bn_bwd_reduce`, the gradient w.r.t. the conv output is, per channel n,
    ``d = A g + B y + K`` with ``A = scale``, ``B = -scale * invstd * sums[1] * inv_count``,
    ``K = -scale * sums[0] * inv_count - B * mean`` (:func:`bn_bwd_elemt` written out).  Because ``y`` is a
    product with ``w`` itself, both gradient products of the convolution can be formed from ``g`` and ``a``
    alone -- neither ``d`` nor ``y`` is touched:

    * data gradient ``d . w = g . (A o w) + a . S + bias`` with ``S = w^T diag(B) w`` (``[C, C]``) and
      ``bias = K . w``: :func:`conv_dgrad_folded`;
    * weight gradient ``d^T a = A o (g^T a) + B o (w . (a^T a)) + K (x) colsum(a)``: :func:`conv_wgrad_folded`.

    Returns the folded data-gradient weights ``[C, N + C]`` (``[(A o w)^T | S]``, compute dtype), ``bias [C]``
    and ``coef = [A, B, K]`` (``[3, N]``).  ``y`` here is the exact product; a backend's stored ``y`` is that
    product rounded to the compute dtype, so results agree with :func:`bn_bwd_elemt` + :func:`conv_dgrad` /
    :func:`conv_wgrad` up to that rounding (and are free of the rounding of ``d``).
    """
    N, C = w.shape[0], w.shape[-1]
    w2 = w.reshape(N, C).float()
    k0, k1 = sums[0] * inv_count, sums[1] * inv_count
    A = scale.float()
    Bc = -A * k1 * invstd
    K = -A * k0 - Bc * mean
    S = w2.t() @ (Bc[:, None] * w2)
    wfold = torch.cat([(w2 * A[:, None]).t(), S], dim=1).to(w.dtype).contiguous()
    return BnFold(wfold, K @ w2, torch.stack([A, Bc, K]).contiguous(), C, N)


def bn_fold_sums(prod: torch.Tensor, w: torch.Tensor, s0: torch.Tensor, mean, invstd, dgamma=None, dbeta=None):
    """``[s0, s1]`` with ``s1 = sum g * xhat = invstd * (sum_c w[n, c] prod[n, c] - mean * s0)`` from the unscaled
    weight-gradient product ``prod = g^T a`` -- because ``y = a . w^T``, ``sum_m g y`` needs neither ``g`` nor
    ``y`` again.  ``dbeta += s0``, ``dgamma += s1`` (local sums, like :func:`bn_bwd_reduce`)."""
    N, C = w.shape[0], w.shape[-1]
    s1 = invstd * ((w.reshape(N, C).float() * prod.reshape(N, C)).sum(1) - mean * s0)
    if dbeta is not None:
        dbeta.add_(s0)
    if dgamma is not None:
        dgamma.add_(s1)
    return torch.stack([s0, s1])


def conv_dgrad_folded(g: torch.Tensor, a_in: torch.Tensor, fold: BnFold, bwd_stats=None,
                      out: Optional[torch.Tensor] = None, **_) -> torch.Tensor:
    """``g . (A o w) + a_in . S + bias`` (see :func:`bn_fold_prepare`); ``bwd_stats`` is a fused backend's
    business (ignored here like in :func:`conv_dgrad`)."""
    N, C = fold.N, fold.C
    wf = fold.wfold.float()
    dx = g.float().reshape(-1, N) @ wf[:, :N].t() + a_in.float().reshape(-1, C) @ wf[:, N:].t() + fold.bias
    dx = dx.reshape(a_in.shape).to(g.dtype)
    if out is not None:
        out.copy_(dx)
        return out
    return dx


def gram_and_means(a: torch.Tensor, colsum_slot: Optional[str] = None):
    """``(a^T a, [column means, column means of squares])`` of an NHWC tensor seen as ``[rows, C]`` (fp32)."""
    a2 = a.float().reshape(-1, a.shape[-1])
    return a2.t() @ a2, torch.stack([a2.mean(0), (a2 * a2).mean(0)])


def bn_stats_from_gram(w: torch.Tensor, gram: torch.Tensor, mom: torch.Tensor, rows: int,
                       stat_shift: Optional[torch.Tensor], **_) -> torch.Tensor:
    """Shifted moments (see :func:`channel_moments`) of ``y = a . w^T`` from the Gram matrix and column means of
    ``a`` alone: ``E[y_n] = w_n . mean(a)``, ``E[y_n^2] = w_n (a^T a / rows) w_n^T`` -- the batch statistics of a
    1x1 convolution's output are known before the convolution has run."""
    N, C = w.shape[0], w.shape[-1]
    w2 = w.reshape(N, C).float()
    mean = w2 @ mom[0]
    # centred first: the variance as a quadratic form of its own, not the difference of two numbers ~ mean^2
    var = ((w2 @ (gram / rows - torch.outer(mom[0], mom[0]))) * w2).sum(1)
    off = mean - stat_shift if stat_shift is not None else mean
    return torch.stack([off, var + off * off])


def bn_fuse_fprop_weights(w, scale, shift, w2=None, scale2=None, shift2=None):
    """``([scale o w | scale2 o w2], shift + shift2)`` (rows = output channels; ``w2`` optional, both 1x1)."""
    N = w.shape[0]
    parts = [w.reshape(N, -1).float() * scale[:, None]]
    sh = shift.clone()
    if w2 is not None:
        parts.append(w2.reshape(N, -1).float() * scale2[:, None])
        sh = sh + shift2
    return torch.cat(parts, dim=1).to(w.dtype).contiguous(), sh


def conv_fprop_fused_tail(a: torch.Tensor, wf: torch.Tensor, shift: torch.Tensor, addend: Optional[torch.Tensor] = None,
                          in2: Optional[torch.Tensor] = None, bits_out: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None, **_) -> torch.Tensor:
    """``relu(a . wf[:, :C]^T + in2 . wf[:, C:]^T + shift + addend)`` (+ packed sign mask): a residual block's tail
    as one product, see :func:`bn_fuse_fprop_weights`."""
    C = a.shape[-1]
    N = wf.shape[0]
    wf32 = wf.float()
    y = a.float().reshape(-1, C) @ wf32[:, :C].t() + shift
    if in2 is not None:
        y = y + in2.float().reshape(-1, in2.shape[-1]) @ wf32[:, C:].t()
    y = y.reshape(*a.shape[:-1], N)
    if addend is not None:
        y = y + addend.float()
    y = torch.relu(y).to(a.dtype)
    if bits_out is not None:
        _pack_bits(y, bits_out)
    if out is not None:
        out.copy_(y)
        return out
    return y


def channel_sums(g: torch.Tensor) -> torch.Tensor:
    return g.float().reshape(-1, g.shape[-1]).sum(0)


def conv_wgrad_folded(a_in: torch.Tensor, g: torch.Tensor, fold: BnFold, w: torch.Tensor, dw: torch.Tensor,
                      prod: Optional[torch.Tensor] = None, amean_slot: Optional[str] = None, gram=None,
                      mom=None) -> None:
    """``dw += A o (g^T a) + B o (w . (a^T a)) + K (x) colsum(a)`` (see :func:`bn_fold_prepare`); ``prod``: the
    product ``g^T a`` when it has been formed already (:func:`bn_fold_sums`)."""
    N, C = fold.N, fold.C
    a2, g2 = a_in.float().reshape(-1, C), g.float().reshape(-1, N)
    A, Bc, K = fold.coef[0], fold.coef[1], fold.coef[2]
    gram = a2.t() @ a2
    p2 = prod.reshape(N, C) if prod is not None else g2.t() @ a2
    upd = A[:, None] * p2 + Bc[:, None] * (w.reshape(N, C).float() @ gram) + K[:, None] * a2.sum(0)[None, :]
    dw.add_(upd.reshape(dw.shape))

# ---------------------------------------------------------------------------- pooling
def maxpool_fwd(x: torch.Tensor):
    """3x3 / stride 2 / pad 1 max pooling; returns ``(out, idx)`` with an opaque index tensor."""
    out, idx = F.max_pool2d(_nchw(x.float()), 3, 2, 1, return_indices=True)
    return _nhwc(out).to(x.dtype), idx


pool_winners = True


def bn_relu_maxpool_fwd(y, scale, shift, winners: bool = False):
    """``maxpool3x3s2(relu(y*scale + shift))``: the stem's BatchNorm-apply and pooling in one op.  ``winners``: also
    ``y`` at every window's winner, and the packed sign mask of the pooled result attached to it."""
    out, idx = maxpool_fwd(bn_apply(y, scale, shift, None, True))
    if not winners:
        return out, idx
    B, H, W, C = y.shape
    ywin = _nhwc(_nchw(y.float()).reshape(B, C, -1).gather(2, idx.reshape(B, C, -1)).view(idx.shape)).to(y.dtype)
    bits = new_relu_bits(out)
    _pack_bits(out, bits)
    out._pdt_relu_bits = bits
    return out, idx, ywin


def maxpool_bwd(dout: torch.Tensor, idx: torch.Tensor, in_shape) -> torch.Tensor:
    B, H, W, C = in_shape
    # Overlapping 3x3/s2 windows can select the same input element twice and the gradient
    # must then be the SUM of both, so scatter-add (max_unpool2d would overwrite).
    dx = torch.zeros(B, C, H * W, dtype=torch.float32, device=dout.device)
    dx.scatter_add_(2, idx.reshape(B, C, -1), _nchw(dout.float()).reshape(B, C, -1))
    return _nhwc(dx.view(B, C, H, W)).to(dout.dtype)


def avgpool_fwd(x: torch.Tensor) -> torch.Tensor:
    return x.float().mean(dim=(1, 2)).to(x.dtype)


def avgpool_bwd(dp: torch.Tensor, H: int, W: int, relu_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    B, C = dp.shape
    dx = (dp.float() / (H * W)).view(B, 1, 1, C).expand(B, H, W, C).contiguous().to(dp.dtype)
    if relu_mask is not None:
        dx = dx * (relu_mask > 0)
    return dx


# ---------------------------------------------------------------------------- classifier + loss
def linear_fwd(a: torch.Tensor, w: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    return (a.float() @ w.float().t() + bias).to(a.dtype)


def linear_bwd(a, dlogits, w, wt, dw: torch.Tensor, dbias: torch.Tensor) -> torch.Tensor:
    d32 = dlogits.float()
    dw.add_(d32.t() @ a.float())
    dbias.add_(d32.sum(0))
    return (d32 @ w.float()).to(a.dtype)


def softmax_ce(logits: torch.Tensor, labels: torch.Tensor, grad_scale: float = 1.0):
    """Mean cross-entropy and its gradient ``(softmax - onehot) * grad_scale / B`` in one pass."""
    l32 = logits.float()
    logp = torch.log_softmax(l32, dim=1)
    B = l32.shape[0]
    loss = -logp.gather(1, labels.view(-1, 1).long()).mean()
    d = torch.exp(logp)
    d.scatter_add_(1, labels.view(-1, 1).long(), torch.full((B, 1), -1.0, device=d.device))
    return loss, (d * (grad_scale / B)).to(logits.dtype)


def ce_metrics(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """``[loss_sum, correct@1, correct@5, n]`` (fp32) for a validation batch."""
    l32 = logits.float()
    lab = labels.view(-1, 1).long()
    logp = torch.log_softmax(l32, dim=1)
    loss_sum = -logp.gather(1, lab).sum()
    rank = (l32 > l32.gather(1, lab)).sum(dim=1)
    n = torch.tensor(float(l32.shape[0]), device=l32.device)
    return torch.stack([loss_sum, (rank < 1).sum().float(), (rank < 5).sum().float(), n])


# ---------------------------------------------------------------------------- linear with activation and residual
LINEAR_ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
MAX_ROWS = 2 ** 31 - 65                 # of any operand: row numbers are 32-bit
MAX_WIDTH = 2 ** 22 - 64                # of a layer: 256 rows of an operand stay below 2 GiB of 32-bit offsets


def _check_rows(what: str, name: str, t: torch.Tensor, shape) -> None:
    if t.dtype not in (torch.bfloat16, torch.float32) or (t.is_cuda and t.dtype != torch.bfloat16):
        raise TypeError(f"{what}: {name} must be bf16 (the CPU path also takes fp32), got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{what}: {name} must have unit column stride")


def _check_vector(what: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be fp32, got {t.dtype}")
    if tuple(t.shape) != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what}: {name} must be contiguous [{n}], got {tuple(t.shape)}")


def _check_product(what: str, a: torch.Tensor, w: torch.Tensor, act: str):
    if act not in LINEAR_ACTS:
        raise ValueError(f"{what}: act must be one of {sorted(LINEAR_ACTS)}, got {act!r}")
    if a.dim() != 2 or w.dim() != 2 or a.shape[1] != w.shape[1] or a.shape[1] < 1 or w.shape[0] < 1:
        raise ValueError(f"{what}: a [M, K] and w [N, K] with K, N >= 1, got {tuple(a.shape)}, {tuple(w.shape)}")
    if max(a.shape[1], w.shape[0]) > MAX_WIDTH or a.shape[0] > MAX_ROWS:
        raise ValueError(f"{what}: K and N are at most {MAX_WIDTH}, M fits 31 bits, got {tuple(a.shape)}, {tuple(w.shape)}")
    _check_rows(what, "a", a, a.shape)
    _check_rows(what, "w", w, w.shape)
    return a.shape[0], w.shape[0], a.shape[1]


def check_linear_act_fwd(a, w, bias, act: str, residual) -> None:
    M, N, _ = _check_product("linear_act_fwd", a, w, act)
    if bias is not None:
        _check_vector("linear_act_fwd", "bias", bias, N)
    if residual is not None:
        _check_rows("linear_act_fwd", "residual", residual, (M, N))


def check_linear_act_bwd(a, w, dy, z, act: str, dw, dbias) -> None:
    what = "linear_act_bwd"
    M, N, K = _check_product(what, a, w, act)
    _check_rows(what, "dy", dy, (M, N))
    if act != "none":
        if z is None:
            raise ValueError(f"{what}: act {act!r} needs z, the pre-activation that linear_act_fwd(save=True) returns")
        _check_rows(what, "z", z, (M, N))
    if dw is not None:
        if dw.dtype != torch.float32:
            raise TypeError(f"{what}: dw, where given, is a fp32 gradient buffer to add to, got {dw.dtype}")
        if tuple(dw.shape) != (N, K) or (K > 1 and dw.stride(1) != 1) or (N > 1 and dw.stride(0) < K):
            raise ValueError(f"{what}: dw must be [{N}, {K}] with unit column stride, got {tuple(dw.shape)}")
    if dbias is not None:
        _check_vector(what, "dbias", dbias, N)


def _act_value(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.relu(z)
    if act == "gelu":
        return torch.where(z == -torch.inf, torch.zeros_like(z), 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5))
    if act == "silu":
        return torch.where(z == -torch.inf, torch.zeros_like(z), z * torch.sigmoid(z))
    return z


def _act_slope(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.where(z.isnan(), z, (z > 0).to(z.dtype))
    big = z.isinf()
    zf = torch.where(big, torch.zeros_like(z), z)
    if act == "gelu":
        slope = 0.5 * torch.special.erfc(-zf * 0.5 ** 0.5) + zf * torch.exp(-0.5 * zf * zf) * (0.5 / torch.pi) ** 0.5
    else:
        s = torch.sigmoid(zf)
        slope = s * (1 + zf * (1 - s))
    return torch.where(big, (z > 0).to(z.dtype), slope)


def linear_act_fwd(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
                   residual: Optional[torch.Tensor] = None, save: bool = False):
    """``(y, z)``: ``z = a w^T + bias``, ``y = act(z) + residual``, each rounded once from fp32; ``a[M, K]``, ``w[N, K]``,
    ``residual[M, N]`` in the compute dtype with unit column stride and any row stride, ``bias[N]`` fp32; K and N up to
    ``MAX_WIDTH``, M up to ``MAX_ROWS``.

    ``act``: none, relu, gelu (the exact one) or silu; on the GPU gelu and silu are zero where the factor of ``z`` is below 2^-126
    (``z`` below -13 and -87).  ``z`` is returned with ``save`` (what :func:`linear_act_bwd` needs where
    there is an activation) and is None without it or with act none.  On the GPU ``y`` and ``z`` are views of rows padded to a
    multiple of 64 columns, as :func:`linear_fwd` returns them, the padding zero."""
    check_linear_act_fwd(a, w, bias, act, residual)
    z = a.float() @ w.float().t()
    if bias is not None:
        z = z + bias
    y = _act_value(z, act)
    if residual is not None:
        y = y + residual.float()
    return y.to(a.dtype), (z.to(a.dtype) if save and act != "none" else None)


def linear_act_bwd(a: torch.Tensor, w: torch.Tensor, dy: torch.Tensor, z: Optional[torch.Tensor] = None, act: str = "none",
                   dw: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None, need_da: bool = True):
    """Gradients ``(da, dw, dbias)`` of :func:`linear_act_fwd` for the gradient ``dy`` of its ``y`` (the residual's gradient is
    ``dy`` itself): ``dz = dy act'(z)``, ``da = dz w``, ``dw = dz^T a``, ``dbias = sum of dz over the rows``.

    ``dw`` / ``dbias`` given: fp32 gradient buffers, added to.  Not given: new tensors, ``dw`` in the compute dtype, ``dbias``
    fp32.  ``need_da=False`` (a first layer): ``da`` is None.  On the GPU ``dz`` is rounded to bf16 before the products, as their
    operand; ``dbias`` sums it unrounded.  Sums run in a fixed order: the same bits from run to run."""
    check_linear_act_bwd(a, w, dy, z, act, dw, dbias)
    dz = dy.float()
    if act != "none":
        dz = dz * _act_slope(z.float(), act)
    da = (dz @ w.float()).to(a.dtype) if need_da else None
    gw, gb = dz.t() @ a.float(), dz.sum(0)
    dw = gw.to(a.dtype) if dw is None else dw.add_(gw)
    dbias = gb if dbias is None else dbias.add_(gb)
    return da, dw, dbias


# ---------------------------------------------------------------------------- distillation
MAX_TOP = 512                # slots per row
MAX_CLASSES = 262144
_LOGIT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_INDEX_DTYPES = (torch.int32, torch.int64)


def _check_logits(what: str, logits: torch.Tensor, temperature: float):
    shape = logits.shape
    if logits.dtype not in _LOGIT_DTYPES:
        raise TypeError(f"{what}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if len(shape) != 2 or not 1 <= shape[1] <= MAX_CLASSES or shape[0] > MAX_ROWS:
        raise ValueError(f"{what}: logits must be [rows, classes] with 1 to {MAX_CLASSES} classes and at most {MAX_ROWS} rows, "
                         f"got {tuple(shape)}")
    if logits.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f"{what}: logits must have unit column stride")
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"{what}: temperature must lie in [0.001, 1000], got {temperature}")
    return shape


def check_top_logits(logits: torch.Tensor, k: int, temperature: float) -> None:
    N = _check_logits("top_logits", logits, temperature)[1]
    if not 1 <= k <= min(MAX_TOP, N):
        raise ValueError(f"top_logits: k must lie in [1, {min(MAX_TOP, N)}], got {k}")


def _check_per_row(name: str, t: torch.Tensor, dtypes, B: int) -> None:
    if t.dtype not in dtypes:
        raise TypeError(f"distill_ce: {name} must be one of {dtypes}, got {t.dtype}")
    if t.dim() != 1 or t.shape[0] != B or not t.is_contiguous():
        raise ValueError(f"distill_ce: {name} must be [{B}] and contiguous, got {tuple(t.shape)}")


def check_distill_ce(logits, labels, values, indices, temperature: float, alpha: float, lse) -> None:
    B = _check_logits("distill_ce", logits, temperature)[0]
    shape = values.shape
    if values.dtype not in _LOGIT_DTYPES or indices.dtype not in _INDEX_DTYPES:
        raise TypeError(f"distill_ce: values must be bf16 / fp16 / fp32 and indices int32 / int64, got {values.dtype}, {indices.dtype}")
    if len(shape) != 2 or shape[0] != B or shape != indices.shape or not 1 <= shape[1] <= MAX_TOP:
        raise ValueError(f"distill_ce: values and indices must both be [{B}, k] with k in [1, {MAX_TOP}], got "
                         f"{tuple(shape)}, {tuple(indices.shape)}")
    if labels is not None:
        _check_per_row("labels", labels, _INDEX_DTYPES, B)
    if lse is not None:
        _check_per_row("lse", lse, (torch.float32,), B)
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"distill_ce: alpha must lie in [0, 1], got {alpha}")


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0):
    """What a teacher hands to :func:`distill_ce`: ``(values[B, k], indices[B, k] int32, lse[B] fp32)``.

    The ``k`` largest logits of each row in falling order, ties to the lower class, a NaN before every number; a class at
    ``-inf`` is never chosen (slots left over hold value ``-inf``, class ``-1``).  ``lse`` is ``logsumexp(logits / T)`` over the
    whole row (``-inf`` for a row that is ``-inf`` throughout).  ``logits``: bf16, fp16 or fp32, unit column stride, any row
    stride; up to ``MAX_TOP`` slots, ``MAX_CLASSES`` classes and ``MAX_ROWS`` rows."""
    check_top_logits(logits, k, temperature)
    l32 = logits.float()
    order = torch.where(l32.isnan(), torch.full_like(l32, torch.inf), l32)
    # a NaN sorts before +inf: two stable passes, the second by "is a NaN"
    idx = torch.sort(order, dim=1, descending=True, stable=True).indices
    nan_first = torch.sort(l32.gather(1, idx).isnan().to(torch.uint8), dim=1, descending=True, stable=True).indices
    idx = idx.gather(1, nan_first)[:, :k]
    values = logits.gather(1, idx)
    idx = torch.where(values == -torch.inf, torch.full_like(idx, -1), idx)
    return values, idx.to(torch.int32), torch.logsumexp(l32.double() / temperature, dim=1).float()


def distill_ce(logits: torch.Tensor, labels: Optional[torch.Tensor], values: torch.Tensor, indices: torch.Tensor,
               temperature: float = 1.0, alpha: float = 0.5, lse: Optional[torch.Tensor] = None, grad_scale: float = 1.0):
    """Distillation from a teacher's top logits: mean loss and its gradient in one pass.

    A row's loss is ``(1 - alpha) * hard + alpha * T^2 * soft``.  ``hard`` is the cross-entropy with ``labels`` (None: left out),
    ``soft`` the divergence KL(P || q) of ``q = softmax(logits / T)`` from the teacher's ``P``: ``exp(values / T - L)`` at the classes
    ``indices``.  With ``lse`` (the teacher's logsumexp at ``T``, see :func:`top_logits`) ``L = lse`` and what either distribution has
    outside the listed classes is compared as one class more; without it ``L`` is the logsumexp over the slots, and ``P`` sums to 1
    over them.  The gradient is that of ``grad_scale * loss``, in the logits' type (on the GPU: in rows padded to a multiple of 64
    columns, the padding zero, as ``linear_bwd`` takes them).

    Left out of the mean's numerator, never of its ``B``: the hard term of a row whose label is no class, the soft term of a row
    without slots, everything of a row whose logits are all ``-inf``, and a term whose weight is 0 (``alpha`` 0 or 1).  A slot is
    empty if its index is no class or its value is ``-inf``; slots of one class are added up.  Where the student has nothing outside
    the listed classes there is no rest to compare.  NaN and +inf in the logits or in a slot reach the loss through the terms that
    count; a row without any has a gradient of zero, whatever it holds."""
    check_distill_ce(logits, labels, values, indices, temperature, alpha, lse)
    B, N = logits.shape
    l32 = logits.float()
    if B == 0:
        return torch.zeros((), device=logits.device), torch.zeros_like(logits)
    some = ~(l32 == -torch.inf).all(dim=1, keepdim=True)
    l32 = torch.where(some, l32, torch.zeros_like(l32))
    idx = indices.long()
    filled = (idx >= 0) & (idx < N) & (values != -torch.inf)
    taught = filled.any(dim=1, keepdim=True) & some & (alpha != 0.0)
    # the teacher's distribution in 64 bits: its rest is 1 minus the listed mass
    t = torch.where(filled, values.double() / temperature, torch.full_like(values, -torch.inf, dtype=torch.float64))
    total = lse.double()[:, None] if lse is not None else torch.logsumexp(t, dim=1, keepdim=True)
    p64 = torch.where(filled, torch.exp(t - total), torch.zeros_like(t))
    p = p64.float()
    at = torch.where(filled, idx, torch.full_like(idx, N))                    # one column more: a bin for empty slots
    P = torch.zeros(B, N + 1, device=l32.device).scatter_add_(1, at, p)[:, :N]
    log_q = torch.log_softmax(l32 / temperature, dim=1)
    q = log_q.exp()
    soft = torch.where(P == 0, torch.zeros_like(P), P * (P.log() - log_q)).sum(dim=1, keepdim=True)
    mass = P.sum(dim=1, keepdim=True)
    g = mass * q - P
    if lse is not None:
        listed = torch.zeros(B, N + 1, dtype=torch.bool, device=l32.device).scatter_(1, at, True)[:, :N]
        log_r = torch.logsumexp(torch.where(listed, torch.full_like(log_q, -torch.inf), log_q), dim=1, keepdim=True)
        p_r = (1.0 - p64.sum(dim=1, keepdim=True)).clamp_min(0.0).float()
        has = log_r != -torch.inf
        mass = mass + torch.where(has, p_r, torch.zeros_like(p_r))
        soft = soft + torch.where(has & (p_r > 0), p_r * (p_r.log() - log_r), torch.zeros_like(p_r))
        g = torch.where(listed, mass * q - P, torch.where(has, mass * q - p_r * torch.exp(log_q - log_r), torch.zeros_like(q)))
    loss = torch.where(taught, alpha * temperature * temperature * soft, torch.zeros_like(soft))
    d = torch.where(taught, alpha * temperature * g, torch.zeros_like(g))
    if labels is not None and alpha != 1.0:
        lab = labels.long()[:, None]
        known = (lab >= 0) & (lab < N) & some
        lab = torch.where(known, lab, torch.zeros_like(lab))
        logp = torch.log_softmax(l32, dim=1)
        loss = loss + torch.where(known, -(1.0 - alpha) * logp.gather(1, lab), torch.zeros_like(loss))
        h = logp.exp().scatter_add_(1, lab, torch.full_like(loss, -1.0))
        d = d + torch.where(known, (1.0 - alpha) * h, torch.zeros_like(h))
    return loss.mean(), (d * (grad_scale / B)).to(logits.dtype)


# ---------------------------------------------------------------------------- optimizer
def sgd_step(p: torch.Tensor, g: torch.Tensor, m: torch.Tensor, pc: Optional[torch.Tensor], lr: float,
             momentum: float, weight_decay: float, grad_scale: float, nesterov: bool = False,
             dampening: float = 0.0, first_step: bool = False) -> None:
    """Flat SGD: ``g = g*grad_scale + wd*p; m = mu*m + (1-damp)*g; p -= lr*(m | g+mu*m)``.

    Zeroes ``g`` afterwards (weight-gradient kernels accumulate into it) and refreshes the
    compute-dtype mirror ``pc`` when it is a separate buffer.  On the first step the
    momentum buffer is initialised to the gradient, like ``torch.optim.SGD``.
    """
    grad = g * grad_scale
    if weight_decay != 0.0:
        grad = grad + weight_decay * p
    if momentum != 0.0:
        if first_step:
            m.copy_(grad)
        else:
            m.mul_(momentum).add_(grad, alpha=1.0 - dampening)
        step = grad + momentum * m if nesterov else m
    else:
        step = grad
    p.add_(step, alpha=-lr)
    g.zero_()
    if pc is not None and pc.data_ptr() != p.data_ptr():
        pc.copy_(p)
