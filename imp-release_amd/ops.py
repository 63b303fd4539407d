"""Operators with gradients, for training and scoring next to the matcher (kernels: csrc/attention_grad.hip, norm_act.hip, log_probs.hip).

    attention(q, k, v)            multi-head attention, forward and backward        (nets/layers.py:121-131)
    group_norm_act(x, groups)     group norm + activation, channels last            (nets/layers.py:59-77: groups == channels)
    match_log_probs(logits, ids)  log probability of given matches, entropy, the best alternatives (nets/layers.py:20-24)

They take and return CUDA tensors (float32, float16, bfloat16), work on the current stream of the tensors' device, and are differentiable by autograd once (the gradients
are no autograd functions themselves).  Nothing waits for the GPU and nothing is kept between calls, so they can be captured into a graph: forward, and backward with
``torch.autograd.grad`` inside the capture.  Errors: ``ValueError`` / ``TypeError`` for arguments, ``ImpError`` from the library.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ACT_IDS, DTYPE_IDS, ImpAttnDesc, ImpError, _ptr

OP_ACT_IDS = {**ACT_IDS, 'silu': 3, 'none': 4}


def _check(rc):
    if rc != 0:
        raise ImpError(rc, _lib.lib().imp_last_error().decode())


def _tensor(t, name, dtypes=tuple(DTYPE_IDS), device=None, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{name} must be a tensor')
    if t.dtype not in dtypes:
        raise TypeError(f'{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must have shape {tuple(shape)}, got {tuple(t.shape)}')
    if device is None and not t.is_cuda:
        raise ValueError(f'{name} must live on the GPU (got {t.device}); libimp_hip has no CPU path')
    if device is not None and t.device != device:
        raise ValueError(f'{name} must live on {device} (got {t.device})')
    return t


def _lens(t, name, batch, device):
    if t is None:
        return None
    return _tensor(t, name, (torch.int32, torch.int64), device, (batch,)).to(torch.int32).contiguous()


def _scratch(nbytes, device):
    """scratch memory of one call, from torch's allocator: it belongs to the current stream (or to the graph that is being captured)"""
    return torch.empty((int(nbytes) + 15) // 16 * 2, device=device, dtype=torch.int64) if nbytes else None


def _where(t):
    """(device index, its current stream)"""
    return t.device.index, C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _aligned(t):
    return t.data_ptr() % 16 == 0


# --------------------------------------------------------------------------------------------------------------------------- attention
def _rows(t):
    """t [batch, tokens, heads, channels] as the kernels take it: channels contiguous, everything else in steps of 16 bytes (a copy if it is not)"""
    unit = 16 // t.element_size()
    ok = (t.shape[3] == 1 or t.stride(3) == 1) and _aligned(t) and all(t.shape[i] == 1 or (t.stride(i) % unit == 0 and t.stride(i) > 0) for i in range(3))
    return t if ok else t.contiguous()


def _strides(t):
    return (C.c_int64 * 3)(*[0 if t.shape[i] == 1 else t.stride(i) for i in range(3)])


def _desc(q, k, v, mask, q_lens, k_lens, scale):
    d = ImpAttnDesc()
    d.dtype, d.batch, d.nq, d.nk, d.heads, d.kv_heads, d.head_dim = DTYPE_IDS[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3]
    d.scale = scale
    d.q_stride, d.k_stride, d.v_stride = _strides(q), _strides(k), _strides(v)
    d.key_mask, d.q_lens, d.k_lens = (None if t is None else t.data_ptr() for t in (mask, q_lens, k_lens))
    return d


def _attn_forward(q, k, v, mask, q_lens, k_lens, scale, want_lse):
    L = _lib.lib()
    q, k, v = _rows(q), _rows(k), _rows(v)
    d = _desc(q, k, v, mask, q_lens, k_lens, scale)
    need = C.c_uint64()
    _check(L.imp_attn_workspace(C.byref(d), 0, C.byref(need)))
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = torch.empty(q.shape[0], q.shape[2], q.shape[1], device=q.device, dtype=torch.float32) if want_lse else None
    ws = _scratch(need.value, q.device)
    _check(L.imp_attn_forward(C.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(ws), need, *_where(q)))
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, q_lens, k_lens, scale):
        out, lse = _attn_forward(q, k, v, mask, q_lens, k_lens, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, mask, q_lens, k_lens)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse, mask, q_lens, k_lens = ctx.saved_tensors
        L = _lib.lib()
        q, k, v = _rows(q), _rows(k), _rows(v)
        dout = dout.to(out.dtype).contiguous()
        dout = dout if _aligned(dout) else dout.clone()
        d = _desc(q, k, v, mask, q_lens, k_lens, ctx.scale)
        need = C.c_uint64()
        _check(L.imp_attn_workspace(C.byref(d), 1, C.byref(need)))
        dq = torch.empty(q.shape, device=q.device, dtype=q.dtype) if ctx.needs_input_grad[0] else None
        kv = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dk = torch.empty(k.shape, device=k.device, dtype=k.dtype) if kv else None
        dv = torch.empty(v.shape, device=v.device, dtype=v.dtype) if kv else None
        ws = _scratch(need.value, q.device)
        _check(L.imp_attn_backward(C.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(dout), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), need, *_where(q)))
        return dq, dk if ctx.needs_input_grad[1] else None, dv if ctx.needs_input_grad[2] else None, None, None, None, None


def attention(q, k, v, key_mask: Optional[torch.Tensor] = None, q_lens=None, k_lens=None, scale: Optional[float] = None, return_lse: bool = False):
    """softmax(scale q k^T) v over the kept keys.

    q [batch, nq, heads, head_dim]; k, v [batch, nk, kv_heads, head_dim] with heads a multiple of kv_heads (query head h reads key head h // (heads // kv_heads)) and
    head_dim a multiple of 8 up to 128.  Views of a packed projection are taken without a copy.  key_mask [batch, nk] bool / uint8, True = keep; q_lens, k_lens [batch]
    int32: counts of a ragged batch.  scale: 1 / sqrt(head_dim) unless given.  -> out [batch, nq, heads, head_dim] (and lse float32 [batch, heads, nq], which carries no
    gradient).  A query without a key, or past its count, gives 0 and -inf and has no gradient."""
    _tensor(q, 'q')
    if q.dim() != 4:
        raise ValueError(f'q must be [batch, tokens, heads, head_dim], got {tuple(q.shape)}')
    b, nq, h, dh = q.shape
    for t, name in ((k, 'k'), (v, 'v')):
        _tensor(t, name, (q.dtype,), q.device)
        if t.dim() != 4 or t.shape[0] != b or t.shape[3] != dh or t.shape != k.shape:
            raise ValueError(f'{name} must be [batch, tokens, kv_heads, head_dim] like q {tuple(q.shape)}, got {tuple(t.shape)}')
    nk, kv = k.shape[1], k.shape[2]
    if dh < 8 or dh > 128 or dh % 8:
        raise ValueError(f'head_dim must be a multiple of 8 up to 128, got {dh}')
    if kv < 1 or h < 1 or h % kv:
        raise ValueError(f'heads ({h}) must be a multiple of kv_heads ({kv})')
    if key_mask is not None:
        key_mask = _tensor(key_mask, 'key_mask', (torch.bool, torch.uint8), q.device, (b, nk)).contiguous()
        key_mask = key_mask.view(torch.uint8)
    q_lens, k_lens = _lens(q_lens, 'q_lens', b, q.device), _lens(k_lens, 'k_lens', b, q.device)
    scale = float(dh) ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError('scale must be finite')
    if b == 0 or nq == 0 or nk == 0:        # nothing to attend to: zeros that still belong to the graph
        out = q.masked_fill(torch.ones((), device=q.device, dtype=torch.bool), 0.0) + (k.sum() + v.sum()) * 0
        lse = torch.full((b, h, nq), -math.inf, device=q.device)
        return (out, lse) if return_lse else out
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _Attention.apply(q, k, v, key_mask, q_lens, k_lens, scale)
    else:
        out, lse = _attn_forward(q, k, v, key_mask, q_lens, k_lens, scale, return_lse)
    return (out, lse) if return_lse else out


# -------------------------------------------------------------------------------------------------------------------------- group norm
def _norm_forward(x, weight, bias, lens, groups, eps, act):
    L = _lib.lib()
    b, n, c = x.shape
    need = C.c_uint64()
    _check(L.imp_group_norm_act_workspace(DTYPE_IDS[x.dtype], b, n, c, groups, 0, C.byref(need)))
    y = torch.empty_like(x)
    stats = torch.empty(b, groups, 4, device=x.device, dtype=torch.float32)
    ws = _scratch(need.value, x.device)
    _check(L.imp_group_norm_act_forward(DTYPE_IDS[x.dtype], b, n, c, groups, _ptr(x), _ptr(weight), _ptr(bias), _ptr(lens), eps, act, _ptr(y), _ptr(stats), _ptr(ws),
                                        need, *_where(x)))
    return y, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lens, groups, eps, act):
        y, stats = _norm_forward(x, weight, bias, lens, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, lens, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, lens, stats = ctx.saved_tensors
        L = _lib.lib()
        b, n, c = x.shape
        dy = dy.to(x.dtype).contiguous()
        dy = dy if _aligned(dy) else dy.clone()
        need = C.c_uint64()
        _check(L.imp_group_norm_act_workspace(DTYPE_IDS[x.dtype], b, n, c, ctx.groups, 1, C.byref(need)))
        dx = torch.empty_like(x)
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        ws = _scratch(need.value, x.device)
        _check(L.imp_group_norm_act_backward(DTYPE_IDS[x.dtype], b, n, c, ctx.groups, _ptr(x), _ptr(weight), _ptr(bias), _ptr(lens), ctx.act, _ptr(stats), _ptr(dy),
                                             _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), need, *_where(x)))
        return dx if ctx.needs_input_grad[0] else None, dw, db, None, None, None, None


def group_norm_act(x, groups: int, weight=None, bias=None, eps: float = 1e-3, act: str = 'relu', lens=None):
    """act(weight * (x - mean) / sqrt(var + eps) + bias) on channels-last data.

    x [batch, ..., channels]; mean and (biased) variance over everything between batch and channels and over the channels of a group (``groups`` groups of neighbouring
    channels; groups == channels is InstanceNorm).  weight, bias: float32 [channels], optional.  act: 'relu', 'gelu', 'lrelu' (slope 0.1), 'silu' or 'none'.  lens [batch]
    int32: only the first tokens of each element exist (x must then be [batch, tokens, channels]); the others are not read and give 0.  eps is the matcher's 1e-3."""
    _tensor(x, 'x')
    if x.dim() < 3:
        raise ValueError(f'x must be [batch, ..., channels], got {tuple(x.shape)}')
    b, c = x.shape[0], x.shape[-1]
    if not isinstance(groups, int) or groups < 1 or c < 1 or c % groups:
        raise ValueError(f'channels ({c}) must be a positive multiple of groups ({groups})')
    if act not in OP_ACT_IDS:
        raise ValueError(f'act must be one of {sorted(OP_ACT_IDS)}, got {act!r}')
    eps = float(eps)
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError('eps must be positive')
    if lens is not None and x.dim() != 3:
        raise ValueError('lens needs x [batch, tokens, channels]')
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is not None:
            _tensor(t, name, (torch.float32,), x.device, (c,))
    lens = _lens(lens, 'lens', b, x.device)
    if x.numel() == 0:
        return x + sum(t.sum() * 0 for t in (weight, bias) if t is not None)
    flat = x.reshape(b, -1, c).contiguous()
    flat = flat if _aligned(flat) else flat.clone()
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        y = _GroupNormAct.apply(flat, weight, bias, lens, groups, eps, OP_ACT_IDS[act])
    else:
        y, _ = _norm_forward(flat, weight, bias, lens, groups, eps, OP_ACT_IDS[act])
    return y.view(x.shape)


# ------------------------------------------------------------------------------------------------------------------- log probabilities
def _logp_forward(x, targets, bin_score, top):
    L = _lib.lib()
    rows, cols = x.shape
    dev = x.device
    need = C.c_uint64()
    _check(L.imp_log_probs_workspace(rows, cols, top, 0, C.byref(need)))
    logp, entropy = torch.empty(rows, device=dev), torch.empty(rows, device=dev)
    stats = torch.empty(rows, 2, device=dev)
    top_logp, top_ids = torch.empty(rows, top, device=dev), torch.empty(rows, top, device=dev, dtype=torch.int64)
    ws = _scratch(need.value, dev)
    _check(L.imp_log_probs_forward(DTYPE_IDS[x.dtype], rows, cols, _ld(x), _ptr(x), _ptr(bin_score), _ptr(targets), top, _ptr(logp), _ptr(entropy), _ptr(stats),
                                   _ptr(top_logp) if top else None, _ptr(top_ids) if top else None, _ptr(ws), need, *_where(x)))
    return logp, entropy, stats, top_logp, top_ids


def _ld(x):
    return x.shape[1] if x.shape[0] == 1 else x.stride(0)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bin_score, targets, top):
        logp, entropy, stats, top_logp, top_ids = _logp_forward(x, targets, bin_score, top)
        ctx.save_for_backward(x, bin_score, targets, entropy, stats)
        ctx.mark_non_differentiable(top_logp, top_ids)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, _, __):
        x, bin_score, targets, entropy, stats = ctx.saved_tensors
        if dlogp is None and dentropy is None:
            return None, None, None, None
        L = _lib.lib()
        rows, cols = x.shape
        dlogp, dentropy = (None if t is None else t.float().contiguous() for t in (dlogp, dentropy))
        dx = torch.empty(rows, cols, device=x.device, dtype=x.dtype) if ctx.needs_input_grad[0] else None
        dbin = torch.empty_like(bin_score) if bin_score is not None and ctx.needs_input_grad[1] else None
        need = C.c_uint64()
        _check(L.imp_log_probs_workspace(rows, cols, 0, 1, C.byref(need)))
        ws = _scratch(need.value, x.device) if dbin is not None else None
        if dx is not None or dbin is not None:
            _check(L.imp_log_probs_backward(DTYPE_IDS[x.dtype], rows, cols, _ld(x), _ptr(x), _ptr(bin_score), _ptr(targets), _ptr(entropy), _ptr(stats), _ptr(dlogp),
                                            _ptr(dentropy), _ptr(dx), _ptr(dbin), _ptr(ws), need if ws is not None else 0, *_where(x)))
        return dx, dbin, None, None


def match_log_probs(logits, targets, bin_score=None, top: int = 0):
    """Log probability of each row's given match under the row softmax, the row's entropy, and its best alternatives.

    logits [..., cols]; targets int64 [...]: the matched column, -1 = unmatched (as the matcher's ``indices0``: the dustbin when bin_score is given, otherwise no target),
    -2 = no target; other values give NaN.  bin_score: float32 scalar tensor, the score of the dustbin, one more column of every row.
    -> (logp, entropy) float32 [...], (top_logp float32, top_ids int64) [..., top] with top <= 16: the most probable columns, ties to the lower index (the dustbin is
    column ``cols``; -inf / -1 where there are no more).  logp is 0 where there is no target.  logp and entropy have gradients for logits and bin_score.  A logit of -inf is
    masked; a row of nothing else gives -inf, entropy 0 and no gradient; a NaN or +inf makes its row NaN."""
    _tensor(logits, 'logits')
    if logits.dim() < 1:
        raise ValueError('logits must be [..., cols]')
    lead, cols = logits.shape[:-1], logits.shape[-1]
    _tensor(targets, 'targets', (torch.int64,), logits.device, lead)
    if not isinstance(top, int) or not 0 <= top <= 16:
        raise ValueError(f'top must be between 0 and 16, got {top!r}')
    if bin_score is not None:
        _tensor(bin_score, 'bin_score', (torch.float32,), logits.device)
        if bin_score.numel() != 1:
            raise ValueError('bin_score must be a scalar tensor')
    elif cols == 0:
        raise ValueError('logits need at least one column, or a bin_score')
    rows = targets.numel()
    if rows == 0:
        z = logits.sum(-1).float() * 0 + (0 if bin_score is None else bin_score.sum() * 0)
        return z, z * 1, logits.new_empty(*lead, top, dtype=torch.float32), logits.new_empty(*lead, top, dtype=torch.int64)
    x = logits.reshape(rows, cols)
    if (cols > 1 and x.stride(1) != 1) or (rows > 1 and x.stride(0) < cols):
        x = x.contiguous()
    t = targets.reshape(rows).contiguous()
    if torch.is_grad_enabled() and (logits.requires_grad or (bin_score is not None and bin_score.requires_grad)):
        logp, entropy, top_logp, top_ids = _LogProbs.apply(x, bin_score, t, top)
    else:
        logp, entropy, _, top_logp, top_ids = _logp_forward(x, t, bin_score, top)
    return logp.view(lead), entropy.view(lead), top_logp.view(*lead, top), top_ids.view(*lead, top)
