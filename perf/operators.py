"""What the training and scoring operators of ``imp_release_amd.ops`` are measured on.

Three operators that stand beside the matcher's own layers: multi-head attention with its gradients (``ops.attention``), group norm with an
activation on channels-last data with its gradients (``ops.group_norm_act``; one channel per group is the InstanceNorm + ReLU of every MLP of
the matcher), and the log probabilities of given matches with entropy and the best alternatives, with the gradient of the matching loss
(``ops.match_log_probs``).  ``own`` chooses between those calls and the same mathematics in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

if own:      # the tools set the flag after the import as well: run() imports on its own
    import imp_release_amd  # noqa: F401

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
SIZE = {'f32': 4, 'f16': 2, 'bf16': 2}
ACTS = ('relu', 'gelu', 'lrelu', 'silu', 'none')


# ---------------------------------------------------------------------------------------------------------------------------- cases
def _attn(name, dtype, b, nq, nk, h, kv, dh, train, ragged=False, packed=False):
    return {'name': name, 'op': 'attention', 'dtype': dtype, 'b': b, 'nq': nq, 'nk': nk, 'h': h, 'kv': kv, 'dh': dh, 'train': train, 'ragged': ragged,
            'packed': packed}


def _norm(name, dtype, b, n, c, g, act, affine, train, ragged=False):
    return {'name': name, 'op': 'norm', 'dtype': dtype, 'b': b, 'n': n, 'c': c, 'g': g, 'act': act, 'affine': affine, 'train': train, 'ragged': ragged}


def _logp(name, dtype, rows, v, top, bin_, train):
    return {'name': name, 'op': 'logp', 'dtype': dtype, 'rows': rows, 'v': v, 'top': top, 'bin': bin_, 'train': train}


def listed():
    return [
        # one new keypoint looked up in a map of 4096 (serving: a single query, latency)
        _attn('attn_one_query_bf16', 'bf16', 1, 1, 4096, 4, 4, 64, False),
        # one attention launch of the bench workload: 4 pairs = 8 images of 2048 keypoints, packed q | k | v projection, 32-bit inference
        _attn('attn_pairs_f32', 'f32', 8, 2048, 2048, 4, 4, 64, False, packed=True),
        # a ragged cross-attention batch of 16 in training, 128-channel descriptors (32 per head), odd sizes, keys masked
        _attn('attn_ragged_train_f16', 'f16', 16, 1531, 1777, 4, 4, 32, True, ragged=True),
        # the bench workload's layer in a training step, 32 bits
        _attn('attn_pairs_train_f32', 'f32', 8, 2048, 2048, 4, 4, 64, True),
        # a long set in mixed precision with shared key heads
        _attn('attn_long_train_bf16', 'bf16', 1, 8192, 8192, 16, 4, 128, True),
        # the keypoint encoder's second norm on one small pair (latency)
        _norm('norm_small_f32', 'f32', 2, 97, 64, 64, 'relu', False, False),
        # InstanceNorm + ReLU inside a layer's MLP, training step of 4 pairs of 2048
        _norm('norm_layer_train_f32', 'f32', 8, 2048, 512, 512, 'relu', False, True),
        # full-resolution feature maps of a 480 x 640 image, mixed precision, affine group norm
        _norm('norm_image_train_bf16', 'bf16', 4, 480 * 640, 64, 8, 'gelu', True, True),
        # a ragged batch of descriptors, grouped channels
        _norm('norm_ragged_f32', 'f32', 16, 4095, 256, 32, 'lrelu', True, False, ragged=True),
        # one row over a large set of candidates (retrieval over a map, or one generated token)
        _logp('logp_one_row_f32', 'f32', 1, 65537, 8, False, False),
        # match scores of 4 pairs of 2048 x 2048 with the dustbin: confidence, entropy and the runners-up of every keypoint
        _logp('logp_pairs_f32', 'f32', 4 * 2048, 2048, 4, True, False),
        # a training step over a large candidate set in mixed precision
        _logp('logp_large_train_bf16', 'bf16', 4096, 50001, 0, False, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'norm', 'logp'])
    dtype = rng.choice(['f32', 'f16', 'bf16'])
    train = rng.random() < 0.5
    if op == 'attention':
        kv = rng.choice([1, 2, 4])
        h = kv * rng.choice([1, 2, 4])
        dh = rng.choice([16, 32, 48, 64, 80, 96, 128])
        nk = _log_int(rng, 16 if train else 1, 8192)        # a row of one key has no gradient to compare
        nq = 1 if not train and rng.random() < 0.3 else _log_int(rng, 1, 8192)
        b = max(1, min(_log_int(rng, 1, 16), int(4e9 // (h * nq * nk * dh)) or 1))
        packed = nq == nk and kv == h
        c = _attn('', dtype, b, nq, nk, h, kv, dh, train, ragged=b > 1 and rng.random() < 0.5, packed=packed)
    elif op == 'norm':
        cg = rng.choice([1, 1, 2, 5, 8, 16])
        g = _log_int(rng, 1, 512 // cg)
        n = _log_int(rng, 8 if train else 1, 65536)        # the gradient of two values that are normalised together all but cancels
        b = max(1, min(_log_int(rng, 1, 16), int(4e7 // (n * g * cg)) or 1))
        c = _norm('', dtype, b, n, g * cg, g, rng.choice(ACTS), rng.random() < 0.5, train, ragged=rng.random() < 0.3)
    else:
        v = _log_int(rng, 2, 131072)
        rows = max(1, min(_log_int(rng, 1, 16384), int(1.5e8 // v)))
        c = _logp('', dtype, rows, v, 0 if train else rng.choice([0, 1, 4, 8]), rng.random() < 0.5, train)
    del c['name']
    return c


# --------------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = TYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dt)

    def lengths(b, n):
        return torch.randint((n + 1) // 2, n + 1, (b,), generator=g, device='cuda', dtype=torch.int32)

    s = {'case': case}
    if case['op'] == 'attention':
        b, nq, nk, h, kv, dh = (case[x] for x in ('b', 'nq', 'nk', 'h', 'kv', 'dh'))
        if case['packed']:       # one projection's output: q | k | v side by side in a row
            qkv = normal(b, nq, 3, h, dh, scale=1.3)
            s['q'], s['k'], s['v'] = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            s['q'], s['k'], s['v'] = normal(b, nq, h, dh, scale=1.3), normal(b, nk, kv, dh, scale=1.3), normal(b, nk, kv, dh)
        s['q_lens'] = lengths(b, nq) if case['ragged'] else None
        s['k_lens'] = lengths(b, nk) if case['ragged'] else None
        s['key_mask'] = torch.rand(b, nk, generator=g, device='cuda') < 0.8 if case['ragged'] else None
        if case['ragged']:
            s['key_mask'][0] = False       # one pair whose keys were all pruned
        s['dout'] = normal(b, nq, h, dh, scale=0.01) if case['train'] else None
    elif case['op'] == 'norm':
        b, n, c = case['b'], case['n'], case['c']
        s['x'] = normal(b, n, c) + torch.randn(c, generator=g, device='cuda').to(dt)
        s['weight'] = 1 + 0.1 * torch.randn(c, generator=g, device='cuda') if case['affine'] else None
        s['bias'] = 0.1 * torch.randn(c, generator=g, device='cuda') if case['affine'] else None
        s['lens'] = lengths(b, n) if case['ragged'] else None
        s['dy'] = normal(b, n, c, scale=0.01) if case['train'] else None
    else:
        rows, v = case['rows'], case['v']
        s['logits'] = normal(rows, v, scale=2.0)
        s['targets'] = torch.randint(0, v, (rows,), generator=g, device='cuda')
        s['targets'] = torch.where(torch.rand(rows, generator=g, device='cuda') < 0.2, torch.full_like(s['targets'], -1), s['targets'])
        s['logits'][torch.arange(rows, device='cuda'), s['targets'].clamp_min(0)] += 6.0
        s['bin_score'] = torch.randn((), generator=g, device='cuda') + 4.0 if case['bin'] else None
        if case['train']:
            s['dlogp'] = torch.full((rows,), -1.0 / rows, device='cuda') * (0.5 + torch.rand(rows, generator=g, device='cuda'))
            s['dentropy'] = torch.full((rows,), 0.01 / rows, device='cuda')
    return s


# ----------------------------------------------------------------------------------------------------- the framework's own operators
def _own(s):
    from imp_release_amd import ops
    c = s['case']
    if c['op'] == 'attention':
        masks = {'key_mask': s['key_mask'], 'q_lens': s['q_lens'], 'k_lens': s['k_lens']}
        if not c['train']:
            return ops.attention(s['q'], s['k'], s['v'], **masks)
        q, k, v = (s[x].detach().requires_grad_() for x in 'qkv')
        out = ops.attention(q, k, v, **masks)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), s['dout'])
    if c['op'] == 'norm':
        if not c['train']:
            return ops.group_norm_act(s['x'], c['g'], s['weight'], s['bias'], act=c['act'], lens=s['lens'])
        leaves = [s[x].detach().requires_grad_() for x in ('x', 'weight', 'bias') if s[x] is not None]
        y = ops.group_norm_act(leaves[0], c['g'], *leaves[1:], act=c['act'], lens=s['lens'])
        return (y.detach(),) + torch.autograd.grad(y, leaves, s['dy'])
    if not c['train']:
        return ops.match_log_probs(s['logits'], s['targets'], s['bin_score'], top=c['top'])
    leaves = [s[x].detach().requires_grad_() for x in ('logits', 'bin_score') if s[x] is not None]
    logp, entropy, _, _ = ops.match_log_probs(leaves[0], s['targets'], *leaves[1:])
    return (logp.detach(), entropy.detach()) + torch.autograd.grad((logp, entropy), leaves, (s['dlogp'], s['dentropy']))


# ------------------------------------------------------------------------------------------- the same in elementary torch operations
def _plain_attention(s):
    c = s['case']
    dt, rep = s['q'].dtype, c['h'] // c['kv']
    scale = 1.0 / math.sqrt(c['dh'])
    q = s['q'].float().transpose(1, 2).contiguous()
    k = s['k'].float().transpose(1, 2).repeat_interleave(rep, 1)
    v = s['v'].float().transpose(1, 2).repeat_interleave(rep, 1)
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    if c['ragged']:
        keep = s['key_mask'] & (torch.arange(c['nk'], device='cuda') < s['k_lens'][:, None])
        live = (torch.arange(c['nq'], device='cuda') < s['q_lens'][:, None])[:, None, :, None]
        p.masked_fill_(~keep[:, None, None, :], -math.inf)
        top = p.amax(-1, keepdim=True)
        p = torch.where(live & (top > -math.inf), (p - top.clamp_min(-3e38)).exp_(), 0.0)
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    else:
        p = p.sub_(p.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).to(dt)
    if not c['train']:
        return out
    do = s['dout'].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    shared = (c['b'], c['kv'], rep, c['nk'], c['dh'])
    dk, dv = dk.view(shared).sum(2), dv.view(shared).sum(2)
    return out, dq.transpose(1, 2).to(dt), dk.transpose(1, 2).to(dt), dv.transpose(1, 2).to(dt)


def _positive(s, live, count, eps):
    """whether the normalised value is above zero, in 64 bits: the slope of the activation jumps there"""
    c = s['case']
    x = s['x'].double().view(c['b'], c['n'], c['g'], -1)
    mean = torch.where(live, x, 0.0).sum((1, 3), keepdim=True) / count
    x = torch.where(live, x - mean, 0.0)
    z = (x * ((x * x).sum((1, 3), keepdim=True) / count + eps).rsqrt()).view(c['b'], c['n'], c['c'])
    return (z * s['weight'].double() + s['bias'].double() if c['affine'] else z) > 0


def _plain_norm(s, eps=1e-3):
    c = s['case']
    b, n, ch, g = c['b'], c['n'], c['c'], c['g']
    dt, act = s['x'].dtype, c['act']
    x = s['x'].float().view(b, n, g, ch // g)
    if c['ragged']:
        live = (torch.arange(n, device='cuda') < s['lens'][:, None])[:, :, None, None]
        count = (s['lens'].float() * (ch // g)).view(b, 1, 1, 1)
    else:
        live, count = torch.ones((), device='cuda', dtype=torch.bool), torch.full((), float(n * (ch // g)), device='cuda')
    mean = torch.where(live, x, 0.0).sum((1, 3), keepdim=True) / count
    xc = torch.where(live, x - mean, 0.0)
    rstd = ((xc * xc).sum((1, 3), keepdim=True) / count + eps).rsqrt()
    xh = (xc * rstd).view(b, n, ch)
    w = s['weight'] if c['affine'] else torch.ones(ch, device='cuda')
    z = xh * w + s['bias'] if c['affine'] else xh
    live3 = live.view(b, n, 1) if c['ragged'] else live
    one = torch.ones((), device='cuda')
    if act in ('relu', 'lrelu'):
        low = 0.0 if act == 'relu' else 0.1
        above = _positive(s, live, count, eps) if c['train'] else z > 0
        y, slope = torch.where(z > 0, z, low * z), torch.where(above, one, low * one)
    elif act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    elif act == 'silu':
        sg = 1 / (1 + torch.exp(-z))
        y, slope = z * sg, sg * (1 + z * (1 - sg))
    else:
        y, slope = z, one
    y = torch.where(live3, y, 0.0).to(dt)
    if not c['train']:
        return y
    dz = torch.where(live3, s['dy'].float() * slope, 0.0)
    dxh = (dz * w).view(b, n, g, ch // g)
    xg = xh.view(b, n, g, ch // g)
    m1 = dxh.sum((1, 3), keepdim=True) / count
    m2 = (dxh * xg).sum((1, 3), keepdim=True) / count
    dx = torch.where(live, (dxh - m1 - xg * m2) * rstd, 0.0).view(b, n, ch).to(dt)
    if not c['affine']:
        return y, dx
    return y, dx, (dz * xh).sum((0, 1)), dz.sum((0, 1))


def _plain_logp(s):
    c = s['case']
    x = s['logits'].float()
    if c['bin']:
        x = torch.cat([x, s['bin_score'].float().expand(c['rows'], 1)], 1)
    t = s['targets']
    col = torch.where(t < 0, torch.full_like(t, c['v']), t) if c['bin'] else t.clamp_min(0)
    has = torch.ones_like(t, dtype=torch.bool) if c['bin'] else t >= 0
    # the largest element is left out of the sum, which keeps the log probability of a sure answer (near 0) exact
    x0 = x - x.amax(-1, keepdim=True)
    e = x0.exp()
    rest = e.scatter(1, x0.argmax(-1, keepdim=True), 0.0).sum(-1, keepdim=True)
    lp = x0 - rest.log1p()
    p = e / (1 + rest)
    entropy = (rest.log1p() - (p * x0).sum(-1, keepdim=True))[:, 0]
    logp = torch.where(has, lp.gather(1, col[:, None])[:, 0], 0.0)
    if not c['train']:
        if c['top'] == 0:
            ids = torch.empty(c['rows'], 0, device='cuda', dtype=torch.int64)
        else:
            ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :c['top']].contiguous()
        tops = lp.gather(1, ids)
        if ids.shape[1] < c['top']:        # fewer columns than alternatives asked for
            ids = torch.nn.functional.pad(ids, (0, c['top'] - ids.shape[1]), value=-1)
            tops = torch.nn.functional.pad(tops, (0, c['top'] - tops.shape[1]), value=-math.inf)
        return logp, entropy, tops, ids
    gl = torch.where(has, s['dlogp'], 0.0)[:, None]
    ge = s['dentropy'][:, None]
    dx = -p * gl - ge * p * (lp + entropy[:, None])
    at = -gl * torch.expm1(lp) - ge * p * (lp + entropy[:, None])          # 1 - p without the cancellation
    dx.scatter_(1, col[:, None], torch.where(has[:, None], at.gather(1, col[:, None]), dx.gather(1, col[:, None])))
    grads = (dx[:, :c['v']].to(s['logits'].dtype),)
    if c['bin']:
        grads += (dx[:, c['v']].sum(),)
    return (logp, entropy) + grads


def run(state):
    if own:
        return _own(state)
    return {'attention': _plain_attention, 'norm': _plain_norm, 'logp': _plain_logp}[state['case']['op']](state)


# ----------------------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_attention(s):
    c = s['case']
    q, k, v = (s[x].detach().double().requires_grad_(c['train']) for x in 'qkv')
    grp = c['h'] // c['kv']
    qh = q.reshape(c['b'], c['nq'], c['kv'], grp, c['dh']).permute(0, 2, 3, 1, 4).reshape(c['b'], c['kv'], grp * c['nq'], c['dh'])
    kh, vh = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)
    score = (qh @ kh) / c['dh'] ** 0.5
    if c['ragged']:
        dead = ~s['key_mask'] | (torch.arange(c['nk'], device='cuda') >= s['k_lens'][:, None])
        score = score.masked_fill(dead[:, None, None, :], -1e300)
        prob = torch.softmax(score, -1).masked_fill(dead[:, None, None, :], 0.0)
    else:
        prob = torch.softmax(score, -1)
    o = (prob @ vh).reshape(c['b'], c['kv'], grp, c['nq'], c['dh']).permute(0, 3, 1, 2, 4).reshape(c['b'], c['nq'], c['h'], c['dh'])
    if c['ragged']:
        o = o.masked_fill((torch.arange(c['nq'], device='cuda') >= s['q_lens'][:, None])[:, :, None, None], 0.0)
    if not c['train']:
        return o
    return (o.detach(),) + torch.autograd.grad(o, (q, k, v), s['dout'].double())


def _exact_norm(s, eps=1e-3):
    c = s['case']
    x = s['x'].detach().double().requires_grad_(c['train'])
    leaves = [x]
    if c['affine']:
        w, bias = (s[i].detach().double().requires_grad_(c['train']) for i in ('weight', 'bias'))
        leaves += [w, bias]
    lens = s['lens'] if c['ragged'] else torch.full((c['b'],), c['n'], device='cuda')
    dead = torch.arange(c['n'], device='cuda')[None, :] >= lens[:, None]
    per = c['c'] // c['g']
    weight = (~dead).double() / (lens.double() * per)[:, None]
    xg = x.unflatten(2, (c['g'], per))
    mu = torch.einsum('bngc,bn->bg', xg, weight)
    var = torch.einsum('bngc,bn->bg', (xg - mu[:, None, :, None]) ** 2, weight)
    z = ((xg - mu[:, None, :, None]) / torch.sqrt(var + eps)[:, None, :, None]).flatten(2)
    if c['affine']:
        z = z * w + bias
    f = torch.nn.functional
    y = {'relu': torch.relu, 'gelu': f.gelu, 'silu': f.silu, 'lrelu': lambda t: f.leaky_relu(t, 0.1), 'none': lambda t: t}[c['act']](z)
    y = y.masked_fill(dead[:, :, None], 0.0)
    if not c['train']:
        return y
    return (y.detach(),) + torch.autograd.grad(y, leaves, s['dy'].double())


def _exact_logp(s):
    c = s['case']
    x = s['logits'].detach().double().requires_grad_(c['train'])
    leaves, full = [x], x
    if c['bin']:
        z = s['bin_score'].detach().double().requires_grad_(c['train'])
        leaves.append(z)
        full = torch.cat([x, z.expand(c['rows'], 1)], 1)
    t = s['targets']
    lp = torch.log_softmax(full, 1)
    entropy = torch.special.entr(lp.exp()).sum(1)
    picked = lp.gather(1, (t % (c['v'] + 1) if c['bin'] else t.clamp_min(0))[:, None]).squeeze(1)
    logp = picked if c['bin'] else torch.where(t < 0, torch.zeros_like(picked), picked)
    if c['train']:
        return (logp.detach(), entropy.detach()) + torch.autograd.grad((logp, entropy), leaves, (s['dlogp'].double(), s['dentropy'].double()))
    tops = lp.topk(min(c['top'], lp.shape[1]), 1)[0]
    if tops.shape[1] < c['top']:
        tops = torch.cat([tops, tops.new_full((c['rows'], c['top'] - tops.shape[1]), -math.inf)], 1)
    return logp, entropy, tops, None


def exact(case, seed):
    s = prepare(case, seed)
    return {'attention': _exact_attention, 'norm': _exact_norm, 'logp': _exact_logp}[case['op']](s)


# ------------------------------------------------------------------------------------------------------------- what a pass has to move
def work(case):
    e = SIZE[case['dtype']]
    if case['op'] == 'attention':
        b, nq, nk, h, kv, dh = (case[x] for x in ('b', 'nq', 'nk', 'h', 'kv', 'dh'))
        qb, kb = b * nq * h * dh * e, b * nk * kv * dh * e
        part = 0.75 * 0.75 * 0.8 if case['ragged'] else 1.0          # mean lengths of 3/4, four keys of five kept
        product = 2.0 * b * h * nq * nk * dh * part
        if case['train']:        # forward: two products; backward: five with the recomputed scores; reads q k v dout, writes out dq dk dv
            return {'bytes': 4 * qb + 4 * kb, 'flops': 7 * product}
        return {'bytes': 2 * qb + 2 * kb, 'flops': 2 * product}
    if case['op'] == 'norm':
        n = case['b'] * case['n'] * case['c'] * (0.75 if case['ragged'] else 1.0)
        out = case['b'] * case['n'] * case['c']
        return {'bytes': int((2 * n + 2 * out if case['train'] else n + out) * e), 'flops': (20 if case['train'] else 8) * n}
    n = case['rows'] * case['v']
    return {'bytes': n * e * (2 if case['train'] else 1) + case['rows'] * (16 + 12 * case['top']), 'flops': (10 if case['train'] else 5) * n}
