"""GPU: the operators with gradients (imp_release_amd.ops) against plain implementations in 64 bits.

Tolerances, fixed before the first run.  A result is compared relative to the largest value of its tensor: fp32 outputs within F32 = 3e-6 for sums of up to a few thousand
terms (each product and addition is off by at most 2^-24 = 6e-8 of its operands' size; sums of n terms by about sqrt(n) / 2 of that; the factors of a backward pass
multiply three such results).  fp16 / bf16 outputs: half a step of the output's own rounding (2^-11, 2^-8) plus the roundings of P and dS to the operand type inside bf16
kernels, each half a step (2^-9 relative to its own value, so at most 2^-8 of the largest result after both): 2.5 half steps in all."""
import math

import pytest
import torch

from imp_release_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32 = 3e-6
TOL = {torch.float32: F32, torch.float16: 2.5 * 2.0 ** -11, torch.bfloat16: 2.5 * 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def close(got, want, tol, what=''):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f'{what}: finite in other places'
    f = torch.isfinite(want)
    if not f.any():
        return
    err, top = (got - want)[f].abs().max().item(), want[f].abs().max().item()
    assert err <= tol * max(top, 1e-30), f'{what}: off by {err:.3e} where the largest is {top:.3e} ({err / max(top, 1e-30):.2e} > {tol:.2e})'


# ------------------------------------------------------------------------------------------------------------------------ attention
def attention64(q, k, v, key_mask=None, q_lens=None, k_lens=None, scale=None):
    b, nq, h, dh = q.shape
    nk, kv = k.shape[1:3]
    scale = dh ** -0.5 if scale is None else scale
    keep = torch.ones(b, nk, dtype=torch.bool, device=q.device) if key_mask is None else key_mask.bool()
    if k_lens is not None:
        keep = keep & (torch.arange(nk, device=q.device) < k_lens[:, None])
    live = torch.ones(b, nq, dtype=torch.bool, device=q.device)
    if q_lens is not None:
        live = torch.arange(nq, device=q.device) < q_lens[:, None]
    live = live & keep.any(1, keepdim=True)
    q, k, v = q.double(), k.double(), v.double()
    k = torch.where(keep[:, :, None, None], k, 0.0).repeat_interleave(h // kv, 2)
    v = torch.where(keep[:, :, None, None], v, 0.0).repeat_interleave(h // kv, 2)
    q = torch.where(live[:, :, None, None], q, 0.0)
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * scale
    s = s.masked_fill(~keep[:, None, None, :], -1e300)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None]).masked_fill(~keep[:, None, None, :], 0.0) * live[:, None, :, None]
    out = torch.matmul(p, v.transpose(1, 2)).transpose(1, 2)
    return out, lse.masked_fill(~live[:, None, :], -math.inf)


def attention_case(q, k, v, dout, tol, cancel=0.0, **masks):
    """out, lse and the three gradients against 64 bits; cancel: an absolute error that dq and dk may have besides"""
    got = [t.detach().requires_grad_() for t in (q, k, v)]
    out, lse = ops.attention(*got, return_lse=True, **masks)
    ref = [t.detach().double().requires_grad_() for t in (q, k, v)]
    rout, rlse = attention64(*ref, **masks)
    close(out, rout, tol, 'out')
    close(lse, rlse, 1e-5, 'lse')
    gg = torch.autograd.grad(out, got, dout)
    rg = torch.autograd.grad(rout, ref, torch.where(torch.isfinite(dout), dout, torch.zeros_like(dout)).double())
    for a, b, n in zip(gg, rg, ('dq', 'dk', 'dv')):
        close(a, b, tol + (0.0 if n == 'dv' else cancel / b.abs().max().item()), n)
    plain = ops.attention(q, k, v, **masks)
    assert torch.equal(plain, out.detach()), 'the same without autograd'
    return out.detach(), gg


SIZES = [(1, 1, 1, 1, 1, 8), (1, 1, 5, 4, 4, 64), (2, 33, 65, 4, 2, 32), (1, 128, 128, 4, 4, 64), (2, 129, 31, 4, 1, 48), (3, 64, 257, 6, 3, 128), (1, 300, 512, 4, 4, 80),
         (2, 1000, 333, 4, 4, 64), (1, 7, 2049, 8, 2, 16), (1, 2048, 40, 2, 2, 96)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,nq,nk,h,kv,dh', SIZES)
def test_attention(dtype, b, nq, nk, h, kv, dh):
    q, k, v = rand(b, nq, h, dh, seed=1, dtype=dtype), rand(b, nk, kv, dh, seed=2, dtype=dtype), rand(b, nk, kv, dh, seed=3, dtype=dtype)
    # one key: dq and dk are zero, what is left is the cancellation of two equal sums; compare the rest
    if nk == 1:
        out, lse = ops.attention(q, k, v, return_lse=True)
        close(out, v.repeat_interleave(h // kv, 2).expand(b, nq, h, dh), TOL[dtype], 'out')
        return
    attention_case(q, k, v, rand(b, nq, h, dh, seed=4, scale=0.1, dtype=dtype), TOL[dtype])


@pytest.mark.parametrize('dtype', DTYPES)
def test_attention_ragged_masks_and_garbage(dtype):
    """counts (0 and beyond the tensor among them), a masked-out pair, and NaN / inf / the type's lowest value in everything that does not exist"""
    b, nq, nk, h, kv, dh = 6, 150, 200, 4, 2, 64
    q, k, v = rand(b, nq, h, dh, seed=1, dtype=dtype), rand(b, nk, kv, dh, seed=2, dtype=dtype), rand(b, nk, kv, dh, seed=3, dtype=dtype)
    dout = rand(b, nq, h, dh, seed=4, dtype=dtype)
    q_lens = torch.tensor([150, 149, 1, 0, 1000, 77], dtype=torch.int32, device=DEV)
    k_lens = torch.tensor([200, 1, 130, 64, -5, 199], dtype=torch.int32, device=DEV)
    mask = torch.rand(b, nk, generator=torch.Generator().manual_seed(5)).to(DEV) < 0.6
    mask[1, 0] = True
    mask[5] = False                                   # no key left
    dead = ~(mask & (torch.arange(nk, device=DEV) < k_lens[:, None]))
    gone = torch.arange(nq, device=DEV) >= q_lens[:, None]
    low = torch.finfo(dtype).min
    for t, where in ((q, gone), (k, dead), (v, dead), (dout, gone)):
        for i, val in enumerate((math.nan, math.inf, low)):
            sel = where & (torch.arange(where.shape[1], device=DEV) % 3 == i)
            t[sel] = val
    masks = dict(key_mask=mask, q_lens=q_lens, k_lens=k_lens)
    # Pair 1 has one key: P = 1 and dS is the difference of two equal sums of dh products, 0 but for their roundings.  A partial sum is about |dO| |v| / sqrt(dh) =
    # sqrt(dh) large and is rounded some 24 times by half a step 2^-24: dS is off by sqrt(dh) sqrt(24) 2^-24 = 2.3e-6, and dk, the sum of 300 of them times scale and a q of up
    # to 4, by scale sqrt(300) 4 times that.
    cancel = dh ** -0.5 * 300 ** 0.5 * 4 * dh ** 0.5 * 24 ** 0.5 * 2.0 ** -24
    out, (dq, dk, dv) = attention_case(q, k, v, dout, TOL[dtype], cancel, **masks)
    assert (out[3] == 0).all() and (out[4] == 0).all() and (out[5] == 0).all() and (out[1, 149:] == 0).all()
    assert (dk[dead] == 0).all() and (dv[dead] == 0).all() and (dq[gone] == 0).all() and (dq[5] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,nq,nk,h,kv,dh', [(1, 70, 90, 6, 2, 32), (2, 5, 3001, 3, 1, 64), (1, 300, 400, 7, 1, 128), (1, 1000, 70, 10, 2, 64)])
def test_attention_head_groups_of_any_size(dtype, b, nq, nk, h, kv, dh):
    """3, 5 and 7 query heads per key head, and byte masks of any nonzero value"""
    q, k, v = rand(b, nq, h, dh, seed=1, dtype=dtype), rand(b, nk, kv, dh, seed=2, dtype=dtype), rand(b, nk, kv, dh, seed=3, dtype=dtype)
    mask = torch.randint(0, 3, (b, nk), generator=torch.Generator().manual_seed(5), dtype=torch.uint8).to(DEV) * 127
    out, _ = attention_case(q, k, v, rand(b, nq, h, dh, seed=4, scale=0.1, dtype=dtype), TOL[dtype], key_mask=mask)
    assert torch.equal(out, ops.attention(q, k, v, key_mask=mask != 0))


@pytest.mark.parametrize('dtype', DTYPES)
def test_attention_packed_projection_and_strides(dtype):
    """q | k | v side by side, [batch, heads, tokens, channels] storage, and views that need a copy: the same bits as contiguous operands"""
    b, n, h, dh = 2, 77, 4, 32
    qkv = rand(b, n, 3, h, dh, seed=1, dtype=dtype)
    q, k, v = qkv.unbind(2)
    want = ops.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(ops.attention(q, k, v), want)
    bhnd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(ops.attention(*bhnd), want)
    odd = rand(b, n, h, dh + 3, seed=2, dtype=dtype)[..., 3:]
    assert torch.equal(ops.attention(odd, k, v), ops.attention(odd.contiguous(), k, v))
    wide = torch.stack([q, q], -1).reshape(b, n, h, dh, 2)[..., 0]                  # channel stride 2
    assert torch.equal(ops.attention(wide, k, v), want)
    x = qkv.detach().requires_grad_()
    a = ops.attention(*x.unbind(2))
    g = torch.autograd.grad(a.sum(), x)[0]                                          # an expanded gradient
    y = [t.contiguous().detach().requires_grad_() for t in (q, k, v)]
    gy = torch.autograd.grad(ops.attention(*y), y, torch.ones_like(want))
    assert torch.equal(g, torch.stack(gy, 2))


def test_attention_large_scores_and_scales():
    """scores of +- 1e4 (a hard maximum), tiny and huge operands: fp32 has no operand limit"""
    q, k, v = rand(1, 60, 4, 64, seed=1, scale=60), rand(1, 70, 4, 64, seed=2, scale=60), rand(1, 70, 4, 64, seed=3)
    out = ops.attention(q, k, v)
    ref, _ = attention64(q, k, v)
    # |S| ~ 3e4: a score is off by about 2^-24 |q| |k| / 8 = 2e-3, and with it the weight of a runner-up
    close(out, ref, 4e-3, 'hard maximum')
    for s in (1e-18, 1e18):
        q, k, v = rand(1, 60, 4, 64, seed=1, scale=s), rand(1, 70, 4, 64, seed=2, scale=1 / s), rand(1, 70, 4, 64, seed=3, scale=s)
        attention_case(q, k, v, rand(1, 60, 4, 64, seed=4, scale=1 / s), F32)
    attention_case(*(rand(1, 40, 2, 64, seed=i) for i in (1, 2, 3)), rand(1, 40, 2, 64, seed=4), F32, scale=-0.3)


def test_attention_half_gradients_far_below_the_type():
    """fp16: dS of 1e-7 keeps its bits, the gradients that fit the type come out right"""
    q, k, v = (rand(1, 256, 4, 64, seed=i, dtype=torch.float16) for i in (1, 2, 3))
    dout = rand(1, 256, 4, 64, seed=4, scale=3e-3, dtype=torch.float16)
    g = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(ops.attention(*g), g, dout)
    r = [t.detach().double().requires_grad_() for t in (q, k, v)]
    for a, b, n in zip((dq, dk, dv), torch.autograd.grad(attention64(*r)[0], r, dout.double()), 'qkv'):
        # one more term: the outputs themselves are near the end of the type's range (steps of 2^-24)
        assert (a.double() - b).abs().max().item() <= 2.5 * 2 ** -11 * b.abs().max().item() + 2.0 ** -25, n


def test_attention_gradient_against_differences():
    """directional derivative of a scalar of the outputs by central differences of the operator itself"""
    q, k, v = rand(2, 50, 4, 32, seed=1), rand(2, 60, 2, 32, seed=2), rand(2, 60, 2, 32, seed=3)
    w = rand(2, 50, 4, 32, seed=4).double()
    mask = torch.rand(2, 60, generator=torch.Generator().manual_seed(1)).to(DEV) < 0.7
    f = lambda a, b, c: (ops.attention(a, b, c, key_mask=mask).double() * w).sum().item()  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.attention(*leaves, key_mask=mask), leaves, w.float())
    for i, g in enumerate(grads):
        d = rand(*g.shape, seed=10 + i)
        h = 1e-2
        hi, lo = [q, k, v], [q, k, v]
        hi[i], lo[i] = hi[i] + h * d, lo[i] - h * d
        num, ana = (f(*hi) - f(*lo)) / (2 * h), (g.double() * d).sum().item()
        # third derivative: h^2 / 6 of it; rounding: 2^-24 * sqrt(terms) / h
        assert abs(num - ana) <= 2e-3 * max(1.0, abs(ana)), (i, num, ana)


def test_attention_repeats_bit_for_bit_and_on_other_streams():
    q, k, v = rand(2, 400, 4, 64, seed=1), rand(2, 500, 2, 64, seed=2), rand(2, 500, 2, 64, seed=3)
    dout = rand(2, 400, 4, 64, seed=4)

    def once():
        g = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*g)
        return (out.detach(),) + torch.autograd.grad(out, g, dout)
    first = once()
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for s in side:
        with torch.cuda.stream(s):
            results.append(once())
    torch.cuda.synchronize()
    for r in results + [once()]:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_attention_refusals():
    q, k = rand(2, 5, 4, 16), rand(2, 7, 2, 16)
    for bad in (lambda: ops.attention(q, k, k[:, :5]), lambda: ops.attention(q, k[:1], k[:1]), lambda: ops.attention(q[0], k, k), lambda: ops.attention(q[..., :12], k[..., :12], k[..., :12]),
                lambda: ops.attention(q[:, :, :3], k, k), lambda: ops.attention(q, k.half(), k.half()), lambda: ops.attention(q, k, k, key_mask=torch.ones(2, 6, device=DEV, dtype=torch.bool)),
                lambda: ops.attention(q, k, k, key_mask=torch.ones(2, 7, device=DEV)), lambda: ops.attention(q, k, k, q_lens=torch.ones(3, device=DEV, dtype=torch.int32)),
                lambda: ops.attention(q, k, k, k_lens=torch.ones(2, dtype=torch.int32)), lambda: ops.attention(q, k, k.cpu()), lambda: ops.attention(q, k, k, scale=math.inf)):
        with pytest.raises((ValueError, TypeError)):
            bad()


def test_attention_empty_tensors():
    for nq, nk in ((0, 5), (5, 0)):
        q, k, v = (rand(2, n, 4, 16).requires_grad_() for n in (nq, nk, nk))
        out, lse = ops.attention(q, k, v, return_lse=True)
        assert out.shape == (2, nq, 4, 16) and (out == 0).all() and (lse == -math.inf).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out.sum(), (q, k, v)))


def test_second_derivative_is_refused():
    q, k, v = (rand(1, 8, 2, 16, seed=i).requires_grad_() for i in range(3))
    g = torch.autograd.grad(ops.attention(q, k, v).sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), k)


# ----------------------------------------------------------------------------------------------------------------------- group norm
def norm64(x, groups, weight=None, bias=None, eps=1e-3, act='relu', lens=None):
    b, c = x.shape[0], x.shape[-1]
    flat = x.double().reshape(b, -1, groups, c // groups)
    n = flat.shape[1]
    live = torch.ones(b, n, dtype=torch.bool, device=x.device) if lens is None else torch.arange(n, device=x.device) < lens[:, None]
    w = live.double()[:, :, None, None]
    flat = torch.where(live[:, :, None, None], flat, 0.0)
    count = (w.sum(1, keepdim=True) * (c // groups)).clamp_min(1)
    mean = (flat * w).sum((1, 3), keepdim=True) / count
    var = ((flat - mean) ** 2 * w).sum((1, 3), keepdim=True) / count
    z = ((flat - mean) / torch.sqrt(var + eps)).reshape(b, n, c)
    z = z if weight is None else z * weight.double()
    z = z if bias is None else z + bias.double()
    f = torch.nn.functional
    y = {'relu': torch.relu, 'gelu': f.gelu, 'lrelu': lambda t: f.leaky_relu(t, 0.1), 'silu': f.silu, 'none': lambda t: t}[act](z)
    return torch.where(live[:, :, None], y, 0.0).reshape(x.shape)


def norm_case(x, groups, dy, tol, weight=None, bias=None, **kw):
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    rleaves = [t.detach().double().requires_grad_() for t in (x, weight, bias) if t is not None]
    it, rt = iter(leaves), iter(rleaves)
    args = [next(it), next(it) if weight is not None else None, next(it) if bias is not None else None]
    rargs = [next(rt), next(rt) if weight is not None else None, next(rt) if bias is not None else None]
    y = ops.group_norm_act(args[0], groups, args[1], args[2], **kw)
    ry = norm64(rargs[0], groups, rargs[1], rargs[2], **kw)
    close(y, ry, tol, 'y')
    g = torch.autograd.grad(y, leaves, dy)
    r = torch.autograd.grad(ry, rleaves, torch.nan_to_num(dy, 0, 0, 0).double())
    close(g[0], r[0], tol, 'dx')
    for a, b in zip(g[1:], r[1:]):
        close(a, b, 1e-5, 'dweight / dbias')
    assert torch.equal(ops.group_norm_act(x, groups, weight, bias, **kw), y.detach())
    return y.detach(), g


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,n,c,g,act,affine', [(1, 4, 8, 8, 'relu', False), (2, 97, 64, 64, 'relu', False), (3, 300, 32, 4, 'gelu', True), (1, 1000, 30, 5, 'lrelu', True),
                                                (2, 2048, 512, 512, 'relu', False), (1, 50, 7, 7, 'silu', True), (2, 33, 1100, 4, 'none', True), (4, 5000, 48, 1, 'silu', False),
                                                (1, 9, 2100, 2100, 'gelu', True), (1, 70000, 64, 8, 'relu', True)])
def test_group_norm_act(dtype, b, n, c, g, act, affine):
    x = rand(b, n, c, seed=1, dtype=dtype) + rand(c, seed=2, dtype=dtype)
    w, bias = (1 + 0.2 * rand(c, seed=3), 0.3 * rand(c, seed=4)) if affine else (None, None)
    norm_case(x, g, rand(b, n, c, seed=5, dtype=dtype), TOL[dtype], w, bias, act=act)


@pytest.mark.parametrize('dtype', DTYPES)
def test_group_norm_single_values_and_constants(dtype):
    """one token of one channel per group, and constant groups: the normalised value is 0, the bias remains, the gradient of the input is 0"""
    x = rand(2, 1, 16, seed=1, dtype=dtype)
    bias = rand(16, seed=2)
    assert torch.equal(ops.group_norm_act(x, 16, None, bias, act='none').float(), bias.to(dtype).float().expand(2, 1, 16))
    for t in (x, torch.full((2, 40, 16), 7.25, device=DEV, dtype=dtype)):
        t = t.requires_grad_()
        y = ops.group_norm_act(t, 16, act='none')
        assert (y == 0).all()
        assert (torch.autograd.grad(y, t, torch.ones_like(y))[0] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_group_norm_ragged_and_garbage(dtype):
    b, n, c = 5, 130, 24
    x, dy = rand(b, n, c, seed=1, dtype=dtype), rand(b, n, c, seed=2, dtype=dtype)
    lens = torch.tensor([130, 1, 0, 500, 64], dtype=torch.int32, device=DEV)
    gone = torch.arange(n, device=DEV) >= lens[:, None]
    x[gone] = math.nan
    dy[gone] = math.inf
    w, bias = 1 + 0.2 * rand(c, seed=3), 0.3 * rand(c, seed=4)
    y, g = norm_case(x, 6, dy, TOL[dtype], w, bias, act='gelu', lens=lens)
    assert (y[gone] == 0).all() and (g[0][gone] == 0).all()


def test_group_norm_far_from_zero_and_outliers():
    """a mean of 1e4 deviations, and a first element that is an outlier: nothing cancels"""
    x = rand(2, 500, 32, seed=1) + 1e4                # the inputs' own steps are 1e-3: compare with what they are
    norm_case(x, 8, rand(2, 500, 32, seed=2), 1e-5, act='none')
    x = rand(2, 500, 32, seed=1)
    x[:, 0] = 1e5
    norm_case(x, 32, rand(2, 500, 32, seed=2), 1e-5, act='lrelu')


def test_group_norm_shapes_strides_and_instance_norm():
    x = rand(2, 6, 10, 12, seed=1)
    y = ops.group_norm_act(x, 3, act='silu')
    assert torch.equal(y.view(2, 60, 12), ops.group_norm_act(x.view(2, 60, 12), 3, act='silu'))
    nchw = x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)       # channels not innermost
    assert torch.equal(ops.group_norm_act(nchw, 3, act='silu'), y)
    off = rand(2 * 60 * 12 + 1, seed=1)[1:].view(2, 60, 12)             # not aligned to 16 bytes
    assert torch.equal(ops.group_norm_act(off, 3), ops.group_norm_act(off.clone(), 3))
    z = rand(2, 200, 64, seed=3)
    inst = torch.relu(torch.nn.functional.instance_norm(z.transpose(1, 2), eps=1e-3)).transpose(1, 2)
    close(ops.group_norm_act(z, 64), inst, F32, 'InstanceNorm + ReLU')
    assert ops.group_norm_act(z[:, :0], 64).shape == (2, 0, 64)


def test_group_norm_slope_next_to_zero():
    """values a few steps from the mean: the slope of relu is the one of the exact normalised value"""
    x = torch.full((1, 64, 4), 3.0, device=DEV)
    x[0, 0::2] = torch.nextafter(torch.tensor(3.0), torch.tensor(4.0)).item()
    norm_case(x, 4, rand(1, 64, 4, seed=1), 1e-4, act='relu')


def test_group_norm_gradient_against_differences():
    x, w, bias, dy = rand(2, 60, 16, seed=1), 1 + 0.2 * rand(16, seed=2), 0.3 * rand(16, seed=3), rand(2, 60, 16, seed=4).double()
    f = lambda a, b, c: (ops.group_norm_act(a, 4, b, c, act='gelu').double() * dy).sum().item()  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
    grads = torch.autograd.grad(ops.group_norm_act(leaves[0], 4, leaves[1], leaves[2], act='gelu'), leaves, dy.float())
    for i, g in enumerate(grads):
        d, h = rand(*g.shape, seed=20 + i), 1e-2
        hi, lo = [x, w, bias], [x, w, bias]
        hi[i], lo[i] = hi[i] + h * d, lo[i] - h * d
        num, ana = (f(*hi) - f(*lo)) / (2 * h), (g.double() * d).sum().item()
        assert abs(num - ana) <= 2e-3 * max(1.0, abs(ana)), (i, num, ana)


def test_group_norm_refusals():
    x = rand(2, 5, 12)
    for bad in (lambda: ops.group_norm_act(x, 5), lambda: ops.group_norm_act(x, 0), lambda: ops.group_norm_act(x[0], 3), lambda: ops.group_norm_act(x, 3, act='tanh'),
                lambda: ops.group_norm_act(x, 3, eps=0.0), lambda: ops.group_norm_act(x, 3, rand(11)), lambda: ops.group_norm_act(x, 3, rand(12).half()),
                lambda: ops.group_norm_act(x, 3, rand(12).cpu()), lambda: ops.group_norm_act(x.double(), 3), lambda: ops.group_norm_act(x[None], 3, lens=torch.ones(1, device=DEV, dtype=torch.int32)),
                lambda: ops.group_norm_act(x, 3, lens=torch.ones(3, device=DEV, dtype=torch.int32))):
        with pytest.raises((ValueError, TypeError)):
            bad()


# ---------------------------------------------------------------------------------------------------------------- log probabilities
def logp64(x, t, bin_score=None, top=0):
    rows, cols = x.shape
    x = x.double()
    full = x if bin_score is None else torch.cat([x, bin_score.double().reshape(1, 1).expand(rows, 1)], 1)
    none = (full == -math.inf).all(1)
    safe = torch.where(none[:, None], torch.zeros_like(full), full)
    lp = torch.log_softmax(safe, 1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * torch.where(p > 0, lp, 0.0), 0.0).sum(1)
    entropy = torch.where(none, 0.0, entropy)
    col = torch.where(t == -1, torch.full_like(t, cols), t) if bin_score is not None else t
    has = (col >= 0) & (col < full.shape[1])
    logp = torch.where(has, torch.where(none, -math.inf, lp.gather(1, col.clamp(0, full.shape[1] - 1)[:, None])[:, 0]), 0.0)
    ids = torch.sort(full, dim=1, descending=True, stable=True)[1][:, :top]
    tops = torch.where(none[:, None], -math.inf, lp.gather(1, ids))
    if ids.shape[1] < top:
        ids = torch.nn.functional.pad(ids, (0, top - ids.shape[1]), value=-1)
        tops = torch.nn.functional.pad(tops, (0, top - tops.shape[1]), value=-math.inf)
    ids = torch.where(tops == -math.inf, -1, ids)
    return logp, entropy, tops, ids


def logp_case(x, t, bin_score=None, top=0, tol=F32):
    leaves = [a.detach().requires_grad_() for a in (x, bin_score) if a is not None]
    ref = [a.detach().double().requires_grad_() for a in (x, bin_score) if a is not None]
    logp, ent, tl, ti = ops.match_log_probs(leaves[0], t, *leaves[1:], top=top)
    rlogp, rent, rtl, rti = logp64(ref[0], t, *ref[1:], top=top)
    assert torch.equal(ti, rti), 'alternatives'
    for a, b, n in ((logp, rlogp, 'logp'), (ent, rent, 'entropy'), (tl, rtl, 'top')):
        close(a, b.detach(), F32, n)
    g, h = rand(x.shape[0], seed=8), rand(x.shape[0], seed=9)
    got = torch.autograd.grad((logp, ent), leaves, (g, h))
    fin = torch.isfinite(rlogp.detach())
    want = torch.autograd.grad((torch.where(fin, rlogp, 0.0), rent), ref, (g.double(), h.double()))
    want = [torch.where(torch.isfinite(w), w, 0.0) for w in want]
    if fin.all():
        close(got[0], want[0], max(tol, F32), 'dlogits')
        if len(got) > 1:
            close(got[1], want[1], 2e-5, 'dbin')
    return logp, ent, tl, ti, got


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cols,top,with_bin', [(1, 1, 1, False), (1, 1, 4, True), (3, 2, 8, False), (5, 7, 3, True), (257, 100, 1, True), (64, 513, 4, False),
                                                    (5000, 600, 16, True), (33, 4097, 8, True), (7, 9001, 0, False), (1, 65537, 8, True), (2, 131072, 16, False)])
def test_match_log_probs(dtype, rows, cols, top, with_bin):
    x = rand(rows, cols, seed=1, scale=3.0, dtype=dtype)
    t = torch.randint(-2, cols, (rows,), generator=torch.Generator().manual_seed(2)).to(DEV)
    logp_case(x, t, rand(1, seed=3)[0] if with_bin else None, top, TOL[dtype])


@pytest.mark.parametrize('dtype', DTYPES)
def test_log_probs_masked_columns_ties_and_lowest_values(dtype):
    rows, cols = 12, 700
    x = rand(rows, cols, seed=1, dtype=dtype)
    x[0] = -math.inf                                   # nothing left
    x[1] = -math.inf
    x[1, 300] = 0.5                                    # one column left
    x[2, ::2] = -math.inf
    x[3] = torch.finfo(dtype).min                      # the type's lowest value everywhere: uniform
    x[4] = 1.25                                        # all equal
    x[5, 100:600] = torch.finfo(dtype).min
    x[6, 50:500] = 9.0                                 # a run of equal maxima
    x[7] = -math.inf
    x[7, :3] = torch.finfo(dtype).min
    x[8, 699] = torch.finfo(dtype).max / 2             # sure
    t = torch.tensor([3, 300, 1, 699, 0, 5, 60, 1, 699, -1, -2, 0], device=DEV)
    logp, ent, tl, ti, g = logp_case(x, t, top=8, tol=TOL[dtype])
    assert logp[0] == -math.inf and ent[0] == 0 and (ti[0] == -1).all() and (g[0][0] == 0).all()
    assert logp[1] == 0 and ent[1] == 0 and ti[1].tolist() == [300] + [-1] * 7
    assert ti[4].tolist() == list(range(8)) and ti[6].tolist() == list(range(50, 58))
    assert logp[9] == 0 and logp[10] == 0
    fin = [i for i in range(rows) if i != 0]
    logp_case(x[fin], t[fin], rand(1, seed=3)[0], 4, TOL[dtype])


def test_log_probs_of_sure_matches():
    """logp near 0 keeps its relative precision, and with it the gradient 1 - p"""
    x = torch.zeros(4, 50, device=DEV)
    x[:, 7] = torch.tensor([10.0, 16.0, 30.0, 60.0], device=DEV)
    t = torch.full((4,), 7, device=DEV)
    lx = x.requires_grad_()
    logp, ent, _, _ = ops.match_log_probs(lx, t)
    rest = 49 * torch.exp(-x.detach()[:, 7].double())
    want = -torch.log1p(rest)
    # e^-d is formed as 2^(d log2 e) in 32 bits: the product and the constant are off by half a step each, 2 * 2^-24 d relative in the result
    tol = 1e-6 + x.detach()[:, 7].double() * 2.0 ** -23
    assert ((logp.double() - want).abs() <= tol * want.abs()).all()
    g = torch.autograd.grad(logp.sum(), lx)[0]
    wg = rest / (1 + rest)
    assert ((g[:, 7].double() - wg).abs() <= 1e-5 * wg).all()
    went = torch.log1p(rest) + rest / (1 + rest) * x.detach()[:, 7].double()
    assert ((ent.double() - went).abs() <= 1e-5 * went).all()


def test_log_probs_bad_targets_and_values():
    x = rand(6, 40, seed=1)
    x[2, 3], x[3, 9] = math.nan, math.inf
    t = torch.tensor([40, -3, 0, 0, 1 << 40, 5], device=DEV)
    lx = x.clone().requires_grad_()
    logp, ent, tl, ti = ops.match_log_probs(lx, t, top=2)
    assert torch.isnan(logp[[0, 1, 2, 3, 4]]).all() and torch.isfinite(logp[5])
    assert torch.isnan(ent[[2, 3]]).all() and torch.isfinite(ent[[0, 1, 4, 5]]).all()
    g = torch.autograd.grad(logp, lx, torch.ones_like(logp))[0]
    assert torch.isnan(g[[0, 1, 2, 3, 4]]).any(1).all() and torch.isfinite(g[5]).all()
    assert ((ti >= -1) & (ti < 40)).all()
    with_bin = ops.match_log_probs(x, torch.full((6,), 40, device=DEV), torch.tensor(1.0, device=DEV))[0]
    assert torch.equal(with_bin[[0, 1, 4, 5]], ops.match_log_probs(x, torch.full((6,), -1, device=DEV), torch.tensor(1.0, device=DEV))[0][[0, 1, 4, 5]])


@pytest.mark.parametrize('dtype', DTYPES)
def test_log_probs_strides_and_shapes(dtype):
    x = rand(4, 30, 45, seed=1, dtype=dtype)
    t = torch.randint(0, 29, (4, 45), generator=torch.Generator().manual_seed(1)).to(DEV)
    a = ops.match_log_probs(x.transpose(1, 2), t, top=3)                             # the other image's direction
    b = ops.match_log_probs(x.transpose(1, 2).contiguous(), t, top=3)
    assert all(torch.equal(i, j) for i, j in zip(a, b)) and a[2].shape == (4, 45, 3)
    wide = rand(50, 77, seed=2, dtype=dtype)
    sub = wide[:, 3:70]                                                             # rows apart, start not aligned
    lx = sub.detach().requires_grad_()
    tt = torch.randint(0, 67, (50,), generator=torch.Generator().manual_seed(2)).to(DEV)
    lc = sub.contiguous().requires_grad_()
    oa, ob = ops.match_log_probs(lx, tt), ops.match_log_probs(lc, tt)
    close(oa[0], ob[0], F32), close(oa[1], ob[1], F32)
    ga, gb = torch.autograd.grad(oa[0].sum(), lx)[0], torch.autograd.grad(ob[0].sum(), lc)[0]
    close(ga, gb, TOL[dtype])
    one = ops.match_log_probs(x[0, 0], torch.tensor(4, device=DEV), top=2)
    assert one[0].shape == () and one[3].shape == (2,)
    none = ops.match_log_probs(x[:0, 0], t[:0, 0], top=2)
    assert none[0].shape == (0,) and none[3].shape == (0, 2)


def test_log_probs_agree_with_the_dual_softmax_scores():
    """the matcher's dual-softmax scores are exp of the two directions' log probabilities (nets/layers.py:20-24)"""
    from helpers import eval_config, make_hip_model
    from imp_release_amd import synthetic
    cfg = eval_config(n_layers=2)
    ctx = make_hip_model('GM', cfg, synthetic.make_state_dict(cfg, model='GM', seed=5))._ensure_ctx()
    dist, z = rand(1, 60, 50, seed=1, scale=2.0), 0.7
    scores = ctx.compute_score(dist, z, 1, with_sinkhorn=False)
    bin_ = torch.tensor(z, device=DEV)
    for i in range(0, 60, 7):
        j = (i * 3) % 50
        row = ops.match_log_probs(dist[0, i], torch.tensor(j, device=DEV), bin_)[0]
        col = ops.match_log_probs(dist[0, :, j], torch.tensor(i, device=DEV), bin_)[0]
        # the dustbin row / column holds bin_score too: the column's log-softmax sees it as one more entry
        assert abs((row + col).exp().item() - scores[0, i, j].item()) <= 1e-5 * max(scores[0, i, j].item(), 1e-6) + 1e-9


def test_log_probs_refusals():
    x, t = rand(3, 5), torch.zeros(3, dtype=torch.int64, device=DEV)
    for bad in (lambda: ops.match_log_probs(x, t[:2]), lambda: ops.match_log_probs(x, t.int()), lambda: ops.match_log_probs(x, t.cpu()), lambda: ops.match_log_probs(x, t, top=17),
                lambda: ops.match_log_probs(x, t, top=-1), lambda: ops.match_log_probs(x, t, torch.zeros(2, device=DEV)), lambda: ops.match_log_probs(x[:, :0], t),
                lambda: ops.match_log_probs(x.double(), t), lambda: ops.match_log_probs(x, t, torch.zeros((), device=DEV).half())):
        with pytest.raises((ValueError, TypeError)):
            bad()


# ------------------------------------------------------------------------------------------------------------------------ far and many
def test_sizes_past_32_bits_are_refused():
    """a count that would wrap around in the library is refused, not taken modulo 2^32 (views without memory)"""
    n = 2 ** 32 + 5
    q = rand(1, 5, 2, 16)
    far = rand(1, 1, 2, 16).expand(1, n, 2, 16)
    for bad in (lambda: ops.attention(q, far, far), lambda: ops.attention(far, q, q), lambda: ops.group_norm_act(rand(1, 1, 8).expand(1, n, 8), 2),
                lambda: ops.match_log_probs(rand(1, 1).expand(1, n), torch.zeros(1, dtype=torch.int64, device=DEV)),
                lambda: ops.match_log_probs(rand(1, 1).expand(n, 1), torch.zeros(1, dtype=torch.int64, device=DEV).expand(n))):
        with pytest.raises(ValueError, match='at most'):
            bad()


def test_counts_in_64_bits():
    """a count beyond 2^32 is clamped to the tensor like any other that is too large"""
    q, k = rand(2, 9, 2, 16, seed=1), rand(2, 40, 2, 16, seed=2)
    big = torch.tensor([2 ** 32 + 3, -2 ** 33 - 7], device=DEV)
    want = torch.tensor([2 ** 31 - 1, 0], device=DEV, dtype=torch.int32)
    assert torch.equal(ops.attention(q, k, k, k_lens=big), ops.attention(q, k, k, k_lens=want))
    x = rand(2, 30, 8, seed=3)
    assert torch.equal(ops.group_norm_act(x, 4, lens=big), ops.group_norm_act(x, 4, lens=want))


@pytest.mark.parametrize('nq', [1, 70])
def test_attention_over_a_cache_past_32_bits(nq):
    """keys and values as views of a storage whose tokens lie 2^19 elements apart: offsets past 2^32 bytes"""
    nk, h, kv, dh, step = 4100, 4, 2, 64, 1 << 19
    store = torch.empty(nk * step, device=DEV, dtype=torch.bfloat16)
    k, v = (store.as_strided((1, nk, kv, dh), (nk * step, step, dh, 1), at) for at in (0, 4096))
    k.copy_(rand(1, nk, kv, dh, seed=1, dtype=torch.bfloat16))
    v.copy_(rand(1, nk, kv, dh, seed=2, dtype=torch.bfloat16))
    q, dout = rand(1, nq, h, dh, seed=3, dtype=torch.bfloat16), rand(1, nq, h, dh, seed=4, dtype=torch.bfloat16)

    def once(k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves)
        return (out.detach(),) + torch.autograd.grad(out, leaves, dout)
    for a, b in zip(once(k, v), once(k.contiguous(), v.contiguous())):
        assert torch.equal(a, b)


def test_group_norm_past_32_bits():
    n, c, tol = (1 << 25) + 7, 64, TOL[torch.float16]
    g = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.randn(1, n, c, generator=g, device=DEV, dtype=torch.float16) for _ in range(2))
    lx = x.detach().requires_grad_()
    y = ops.group_norm_act(lx, c, act='none')
    dx = torch.autograd.grad(y, lx, dy)[0]
    sums = torch.zeros(4, c, device=DEV, dtype=torch.float64)
    for i in range(0, n, 1 << 22):
        a, d = x[0, i:i + (1 << 22)].double(), dy[0, i:i + (1 << 22)].double()
        sums += torch.stack([a.sum(0), (a * a).sum(0), d.sum(0), (a * d).sum(0)])
    mean, sq, m1, md = sums / n
    r = 1 / (sq - mean * mean + 1e-3).sqrt()
    m2 = (md - mean * m1) * r
    for rows in (slice(0, 300), slice(n - 300, n)):
        xh = (x[0, rows].double() - mean) * r
        close(y[0, rows].detach(), xh, tol, 'y')
        close(dx[0, rows], (dy[0, rows].double() - m1 - xh * m2) * r, tol, 'dx')


def test_group_norm_of_many_elements():
    """more workgroups than the x dimension of a grid has threads for, and an affine gradient summed over all of them"""
    b, c = 65535, 2048
    x, w = rand(1, 1, c, seed=1).expand(b, 2, c) * torch.linspace(1, 2, 2, device=DEV)[:, None], rand(c, seed=2)
    lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = ops.group_norm_act(lx, 128, lw, act='none')
    dw, = torch.autograd.grad(y, lw, torch.ones_like(y))
    want = norm64(x[:1], 128, w, act='none')
    for i in (0, 32768, b - 1):
        close(y[i:i + 1].detach(), want, F32, f'element {i}')
    close(dw, (norm64(x[:1], 128, act='none').sum((0, 1)) * b), 2e-5, 'dw')            # (a sum of two normalised values of either sign: up to 4 times smaller than they are)


def test_log_probs_of_many_rows():
    """more rows than the x dimension of a grid has threads for"""
    rows = (1 << 26) + 5
    x = torch.randn(rows, 2, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    t = torch.randint(0, 2, (rows,), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    lx = x.detach().requires_grad_()
    logp, ent, _, ids = ops.match_log_probs(lx, t, top=1)
    dx = torch.autograd.grad(logp, lx, torch.ones_like(logp))[0]
    d = x.double()
    lp = d - torch.logsumexp(d, 1, keepdim=True)
    close(logp.detach(), lp.gather(1, t[:, None])[:, 0], F32, 'logp')
    close(ent.detach(), -(lp.exp() * lp).sum(1), F32, 'entropy')
    assert torch.equal(ids[:, 0], (d[:, 1] > d[:, 0]).long())
    close(dx, torch.nn.functional.one_hot(t, 2) - lp.exp(), TOL[torch.float16], 'dx')


def test_log_probs_of_rows_far_apart():
    store = torch.empty(4, 1 << 30, device=DEV, dtype=torch.float16)
    x = store[:, :700]
    x.copy_(rand(4, 700, seed=1, dtype=torch.float16))
    t = torch.tensor([0, 699, 5, -1], device=DEV)
    a, b = (ops.match_log_probs(v, t, top=3) for v in (x, x.contiguous()))
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_log_probs_of_the_dustbin_alone():
    z = torch.tensor(0.5, device=DEV, requires_grad=True)
    x = torch.empty(3, 0, device=DEV, requires_grad=True)
    t = torch.tensor([-1, 0, -2], device=DEV)
    logp, ent, tl, ti = ops.match_log_probs(x, t, z, top=2)
    assert (logp == 0).all() and (ent == 0).all() and (ti == torch.tensor([0, -1], device=DEV)).all() and (tl[:, 0] == 0).all() and (tl[:, 1] == -math.inf).all()
    dx, dz = torch.autograd.grad(logp.sum() + ent.sum(), (x, z))
    assert dx.shape == (3, 0) and dz == 0
    assert torch.autograd.grad(ops.match_log_probs(x, t, z.detach())[0].sum(), x)[0].shape == (3, 0)


# ------------------------------------------------------------------------------------------------------------------------- together
def layer_loss(lib, x, src, wqkv, wkv, w1, w2, targets, bin_score, lens):
    """one cross-attention propagation layer with its MLP, the match scores and the matching loss"""
    b, n, d = x.shape
    m = src.shape[1]
    q = (x @ wqkv).view(b, n, 4, d // 4)
    k, v = (src @ wkv).view(b, m, 2, 4, d // 4).unbind(2)
    msg = lib['attention'](q, k, v, k_lens=lens).reshape(b, n, d)
    hid = lib['norm'](torch.cat([x, msg], -1) @ w1, 2 * d)
    y = x + hid @ w2
    dist = torch.matmul(y, src.transpose(1, 2)) / d ** 0.5
    logp, ent = lib['logp'](dist, targets, bin_score)
    return -logp.mean() + 0.01 * ent.mean()


def test_a_training_step_of_a_layer():
    b, n, m, d = 2, 130, 150, 128
    args = [rand(b, n, d, seed=1), rand(b, m, d, seed=2), rand(d, d, seed=3, scale=0.1), rand(d, 2 * d, seed=4, scale=0.1), rand(2 * d, 2 * d, seed=5, scale=0.1),
            rand(2 * d, d, seed=6, scale=0.1)]
    targets = torch.randint(-1, m, (b, n), generator=torch.Generator().manual_seed(7)).to(DEV)
    lens = torch.tensor([150, 90], dtype=torch.int32, device=DEV)
    mine = {'attention': ops.attention, 'norm': ops.group_norm_act, 'logp': lambda a, t, z: ops.match_log_probs(a, t, z)[:2]}

    def plain_logp(a, t, z):
        full = torch.cat([a, z.reshape(1, 1, 1).expand(*a.shape[:2], 1)], 2)
        lp = torch.log_softmax(full, -1)
        return lp.gather(2, torch.where(t < 0, a.shape[2], t)[..., None])[..., 0], -(lp.exp() * lp).sum(-1)
    plain = {'attention': lambda *a, **k: attention64(*a, **k)[0], 'norm': norm64, 'logp': plain_logp}
    bin_ = torch.tensor(1.0, device=DEV)
    leaves = [a.clone().requires_grad_() for a in args + [bin_]]
    ref = [a.double().requires_grad_() for a in args + [bin_]]
    loss = layer_loss(mine, *leaves[:6], targets, leaves[6], lens)
    rloss = layer_loss(plain, *ref[:6], targets, ref[6], lens)
    assert abs(loss.item() - rloss.item()) <= 1e-5 * abs(rloss.item())
    for i, (a, r) in enumerate(zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(rloss, ref))):
        # torch's own fp32 products between the operators round as much again
        close(a, r, 3e-5, f'gradient {i}')


def test_the_operators_in_a_graph():
    """forward and backward captured and replayed on new inputs, with eager work between the replays, and two graphs at once"""
    b, n, d = 2, 200, 128
    shapes = [(b, n, 4, 32), (b, n, 4, 32), (b, n, 4, 32), (b, n, d)]
    lens = torch.tensor([200, 120], dtype=torch.int32, device=DEV)
    targets = torch.randint(0, n, (b * n,), generator=torch.Generator().manual_seed(1)).to(DEV)

    def step(q, k, v, x):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, x)]
        out = ops.attention(*leaves[:3], k_lens=lens)
        y = ops.group_norm_act(leaves[3] + out.reshape(b, n, d), 16, act='gelu')
        dist = torch.mm(y.reshape(-1, d), y[0].t().contiguous())
        logp, ent, _, ids = ops.match_log_probs(dist, targets, top=2)
        # the seeds of the backward pass are tensors: no library reduction in the captured graph
        return (out.detach(), y.detach(), logp.detach(), ids) + torch.autograd.grad((logp, ent), leaves, (torch.full_like(logp, -0.01), torch.full_like(ent, 0.001)))
    graphs = []
    for i in range(2):
        static = [rand(*s, seed=10 * i + j) for j, s in enumerate(shapes)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*static)
        graphs.append((g, static, res))
    for rep in range(4):
        for i, (g, static, res) in enumerate(graphs):
            new = [rand(*s, seed=100 * rep + 10 * i + j) for j, s in enumerate(shapes)]
            for a, t in zip(static, new):
                a.copy_(t)
            g.replay()
        torch.cuda.synchronize()
        for i, (g, static, res) in enumerate(graphs):
            want = step(*static)
            torch.cuda.synchronize()
            for j, (a, t) in enumerate(zip(res, want)):
                assert torch.equal(a, t), (rep, i, j)
