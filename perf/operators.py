"""Work cases of the token operators: softmax attention, matrix product with epilogue, channels-last group norm, each with its backward pass.

``run`` makes the calls of ``ops_tokens`` where ``own`` is true and computes the same outputs from elementary torch operations in 32 bits
where it is false; ``exact`` gives them from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, dtype, B, Tq, Tk, H, Hk, D, causal=False, mask='none', lens=False, train=True):
    c = {'op': 'attention', 'dtype': dtype, 'B': B, 'Tq': Tq, 'Tk': Tk, 'H': H, 'Hk': Hk, 'D': D, 'causal': causal, 'mask': mask, 'lens': lens,
         'train': train}
    return {'name': name, **c} if name else c


def _linear(name, dtype, M, N, K, act, bias=True, residual=False, train=True):
    c = {'op': 'linear', 'dtype': dtype, 'M': M, 'N': N, 'K': K, 'act': act, 'bias': bias, 'residual': residual, 'train': train}
    return {'name': name, **c} if name else c


def _group_norm(name, dtype, B, V, C, G, act, train=True):
    c = {'op': 'group_norm', 'dtype': dtype, 'B': B, 'V': V, 'C': C, 'G': G, 'act': act, 'train': train}
    return {'name': name, **c} if name else c


def listed():
    return [
        # training: the attention of HartleyMHASeg as it is published (1960 patches of the kept modes, 4 heads of 12 x 8 channels, fp32)
        _attention('attn_hartley_fp32', 'fp32', 1, 1960, 1960, 4, 4, 96),
        # training: a causal stack with four query heads to each key head
        _attention('attn_causal_bf16', 'bf16', 2, 4096, 4096, 16, 4, 128, causal=True),
        # training: a token grid with a visibility mask (windows, padding) of odd sizes
        _attention('attn_masked_bf16', 'bf16', 3, 777, 1033, 6, 2, 80, mask='full'),
        # inference: a long padded batch
        _attention('attn_long_bf16', 'bf16', 2, 8192, 8192, 8, 8, 64, lens=True, train=False),
        # serving: one new token per sequence against the keys and values so far
        _attention('attn_token_bf16', 'bf16', 4, 1, 8191, 16, 4, 128, lens=True, train=False),
        # inference: the wide product of an MLP with all of its epilogue
        _linear('linear_wide_bf16', 'bf16', 8192, 8192, 2048, 'gelu', residual=True, train=False),
        # training: an MLP's first layer over the tokens of two volumes
        _linear('linear_mlp_bf16', 'bf16', 3920, 1536, 384, 'silu'),
        # training in 32 bits, odd sizes
        _linear('linear_odd_fp32', 'fp32', 3001, 771, 387, 'elu', residual=True),
        # serving: a handful of rows
        _linear('linear_rows_bf16', 'bf16', 4, 2048, 2048, 'none', residual=True, train=False),
        # training: a convolution level of 80 x 96 x 64 voxels
        _group_norm('gn_level_bf16', 'bf16', 2, 80 * 96 * 64, 64, 8, 'elu'),
        # inference: the 65^3 working grid with 24 filters, fp32
        _group_norm('gn_grid_fp32', 'fp32', 1, 65 ** 3, 24, 6, 'selu', train=False),
        # training: the bottom of the pyramid, where latency counts
        _group_norm('gn_small_bf16', 'bf16', 2, 10 * 12 * 8, 256, 32, 'silu'),
    ]


def _activation(rng, dtype, train):
    # the slopes of selu and relu jump at 0: in 32 bits the gradient of a value next to 0 would go by the last bit of its sum
    return rng.choice(('none', 'elu', 'gelu', 'silu') + (() if train and dtype == 'fp32' else ('selu', 'relu')))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max(work(c)['flops'] for c in listed())
    while True:
        op = rng.choice(('attention', 'linear', 'group_norm'))
        dtype = rng.choice(('bf16', 'bf16', 'fp32'))
        train = rng.random() < 0.6
        if op == 'attention':
            Hk = rng.choice((1, 2, 3, 4, 8))
            H = Hk * rng.choice((1, 1, 2, 4))
            D = rng.choice((16, 24, 32, 40, 48, 64, 72, 80, 96, 112, 128))
            B = _log(rng, 1, 4)
            if rng.random() < 0.25:      # a few new tokens
                Tq, Tk, train = _log(rng, 1, 8), _log(rng, 16, 12000), False
                kind, lens = 'none', rng.random() < 0.5
                causal = rng.random() < 0.5
            else:
                Tq = _log(rng, 60, 4096 if dtype == 'bf16' else 2048)
                causal = rng.random() < 0.4
                Tk = Tq if causal or rng.random() < 0.5 else _log(rng, 60, 4096 if dtype == 'bf16' else 2048)
                kind = rng.choice(('none', 'none', 'full', 'key'))
                lens = kind == 'none' and rng.random() < 0.5
            case = _attention(None, dtype, B, Tq, Tk, H, Hk, D, causal, kind, lens, train)
        elif op == 'linear':
            big = 8192 if dtype == 'bf16' else 2500
            M, N, K = _log(rng, 1, big), _log(rng, 24, big // 2), _log(rng, 24, big // 2)
            if rng.random() < 0.5:
                N, K = N // 8 * 8, K // 8 * 8
            case = _linear(None, dtype, M, N, K, _activation(rng, dtype, train), rng.random() < 0.7, rng.random() < 0.5, train)
        else:
            G = rng.choice((1, 2, 4, 8, 16, 32))
            C = G * rng.choice((1, 2, 3, 4, 6, 8, 12))
            V = _log(rng, 1, max(2, (1 << 25) // C))
            B = _log(rng, 1, 4)
            if V * (C // G) < 4 or B * V * C > (1 << 26):
                continue
            case = _group_norm(None, dtype, B, V, C, G, _activation(rng, dtype, train), train)
        cost = work(case)
        if cost['flops'] * (8 if dtype == 'fp32' else 1) <= top and not any(all(c[k] == v for k, v in case.items()) for c in listed() if c['op'] == op):
            return case


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device='cuda') * scale + shift).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    dt = DTYPES[case['dtype']]
    s = {'case': case}
    train = case['train']
    if case['op'] == 'attention':
        B, Tq, Tk, H, Hk, D = (case[k] for k in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
        s['q'] = _normal(gen, (B, Tq, H, D), dt)
        s['k'] = _normal(gen, (B, Tk, Hk, D), dt)
        s['v'] = _normal(gen, (B, Tk, Hk, D), dt)
        s['g'] = _normal(gen, (B, Tq, H, D), dt, 0.01) if train else None
        s['mask'] = None
        if case['mask'] == 'full':       # two keys of three visible, and some rows without any
            m = torch.rand((B, 1, Tq, Tk), generator=gen, device='cuda') < 0.67
            s['mask'] = m & (torch.rand((B, 1, Tq, 1), generator=gen, device='cuda') < 0.98)
        elif case['mask'] == 'key':      # padding
            s['mask'] = torch.rand((B, 1, 1, Tk), generator=gen, device='cuda') < 0.9
        # lengths from half of the longest on; training and prompts keep at least one key
        s['lens'] = torch.randint(max(1, Tk // 2), Tk + 1, (B,), generator=gen, device='cuda', dtype=torch.int32) if case['lens'] else None
        leaves = ('q', 'k', 'v')
    elif case['op'] == 'linear':
        M, N, K = case['M'], case['N'], case['K']
        s['x'] = _normal(gen, (M, K), dt)
        s['w'] = _normal(gen, (N, K), dt, 1.0 / math.sqrt(K))
        s['b'] = _normal(gen, (N,), dt, 0.1) if case['bias'] else None
        s['r'] = _normal(gen, (M, N), dt) if case['residual'] else None
        s['g'] = _normal(gen, (M, N), dt, 0.01) if train else None
        leaves = ('x', 'w', 'b', 'r')
    else:
        B, V, C = case['B'], case['V'], case['C']
        s['x'] = (_normal(gen, (B, V, C), torch.float32, 1.5) + _normal(gen, (C,), torch.float32, 0.5)).to(dt)
        s['w'] = _normal(gen, (C,), torch.float32, 0.1, 1.0)
        s['b'] = _normal(gen, (C,), torch.float32, 0.1)
        s['g'] = _normal(gen, (B, V, C), dt, 0.01) if train else None
        leaves = ('x', 'w', 'b')
    if train:
        for k in leaves:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from multimodal_3d_image_segmentation_amd import ops_tokens as ot
    case = s['case']
    if case['op'] == 'attention':
        y = ot.attention(s['q'], s['k'], s['v'], causal=case['causal'], mask=s['mask'], kv_lens=s['lens'])
        leaves = ('q', 'k', 'v')
    elif case['op'] == 'linear':
        y = ot.linear(s['x'], s['w'], s['b'], act=case['act'], residual=s['r'])
        leaves = ('x', 'w', 'b', 'r')
    else:
        y = ot.group_norm(s['x'], case['G'], s['w'], s['b'], eps=1e-5, act=case['act'])
        leaves = ('x', 'w', 'b')
    out = {'y': y.detach()}
    if case['train']:
        names = [k for k in leaves if s[k] is not None]
        out.update(zip(('d' + k for k in names), torch.autograd.grad(y, [s[k] for k in names], s['g'])))
    return out


# ------------------------------------------------------------------------------------------------ the plain form
_SELU = (1.0507009873554804934193349852946, 1.6732632423543772848170429916717)


def _act(z, act):
    """act(z) and act'(z)"""
    if act == 'none':
        return z, torch.ones_like(z)
    if act == 'relu':
        on = z > 0
        return torch.where(on, z, 0.0), on.to(z.dtype)
    if act in ('selu', 'elu'):
        scale, alpha = _SELU if act == 'selu' else (1.0, 1.0)
        low = scale * alpha * torch.exp(torch.clamp(z, max=0.0))
        em1 = scale * alpha * torch.expm1(torch.clamp(z, max=0.0))
        return torch.where(z > 0, scale * z, em1), torch.where(z > 0, scale * torch.ones_like(z), low)
    if act == 'silu':
        sg = 1.0 / (1.0 + torch.exp(-z))
        return z * sg, sg * (1.0 + z * (1.0 - sg))
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_attention(s):
    case, dt = s['case'], s['q'].dtype
    B, Tq, Tk, H, Hk, D = (case[k] for k in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
    n = H // Hk
    q = s['q'].detach().float().transpose(1, 2)                                        # (B, H, Tq, D)
    k, v = (s[x].detach().float().transpose(1, 2).repeat_interleave(n, dim=1) for x in ('k', 'v'))
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    scale = 1.0 / math.sqrt(D)
    i, j = torch.arange(Tq, device='cuda').view(1, 1, Tq, 1), torch.arange(Tk, device='cuda').view(1, 1, 1, Tk)
    length = s['lens'].view(B, 1, 1, 1) if s['lens'] is not None else torch.full((1, 1, 1, 1), Tk, device='cuda')
    seen = j < length
    if case['causal']:
        seen = seen & (j <= i + (length - Tq))
    if s['mask'] is not None:
        seen = seen & s['mask']
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    sc = torch.where(seen, sc, -math.inf)
    top = sc.amax(dim=3, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p, v)
    out = {'y': o.transpose(1, 2).contiguous().to(dt)}
    if case['train']:
        g = s['g'].float().transpose(1, 2).contiguous()
        dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
        dp = torch.matmul(g, v.transpose(2, 3).contiguous())
        ds = p * (dp - (p * dp).sum(dim=3, keepdim=True))
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
        out['dq'] = dq.transpose(1, 2).contiguous().to(dt)
        for name, t in (('dk', dk), ('dv', dv)):
            out[name] = t.view(B, Hk, n, Tk, D).sum(dim=2).transpose(1, 2).contiguous().to(dt)
    return out


def _plain_linear(s):
    case, dt = s['case'], s['x'].dtype
    x, w = s['x'].detach().float(), s['w'].detach().float()
    z = torch.matmul(x, w.t())
    if s['b'] is not None:
        z = z + s['b'].detach().float()
    y, slope = _act(z, case['act'])
    if s['r'] is not None:
        y = y + s['r'].detach().float()
    out = {'y': y.to(dt)}
    if case['train']:
        dz = s['g'].float() * slope
        out['dx'] = torch.matmul(dz, w).to(dt)
        out['dw'] = torch.matmul(dz.t(), x).to(dt)
        if s['b'] is not None:
            out['db'] = dz.sum(dim=0).to(dt)
        if s['r'] is not None:
            out['dr'] = s['g'].clone()
    return out


def _plain_group_norm(s):
    case, dt = s['case'], s['x'].dtype
    B, V, C, G = (case[k] for k in ('B', 'V', 'C', 'G'))
    x = s['x'].detach().float().view(B, V, G, C // G)
    w, b = s['w'].detach().view(G, C // G), s['b'].detach().view(G, C // G)
    mean = x.mean(dim=(1, 3), keepdim=True)
    var = ((x - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(var + 1e-5)
    xh = (x - mean) * rstd
    y, slope = _act(xh * w + b, case['act'])
    out = {'y': y.view(B, V, C).to(dt)}
    if case['train']:
        du = s['g'].float().view(B, V, G, C // G) * slope
        t = du * w
        dx = rstd * (t - t.mean(dim=(1, 3), keepdim=True) - xh * (t * xh).mean(dim=(1, 3), keepdim=True))
        out['dx'] = dx.view(B, V, C).to(dt)
        out['dw'] = (du * xh).sum(dim=(0, 1)).view(C)
        out['db'] = du.sum(dim=(0, 1)).view(C)
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {'attention': _plain_attention, 'linear': _plain_linear, 'group_norm': _plain_group_norm}[state['case']['op']](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _visible_pairs(case):
    Tq, Tk = case['Tq'], case['Tk']
    if not case['causal']:
        return Tq * Tk
    first = Tk - Tq + 1                                   # keys that the first row sees (where positive)
    lo, hi = max(first, 0), Tk
    rows = hi - lo + 1 if first > 0 else Tk
    return (lo + hi) * rows // 2


def work(case):
    size = 2 if case['dtype'] == 'bf16' else 4
    train = case['train']
    if case['op'] == 'attention':
        B, Tq, Tk, H, Hk, D = (case[k] for k in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
        share = 0.75 if case['lens'] else 1.0             # lengths are drawn between a half and the whole
        nq, nk = B * Tq * H * D, B * Tk * Hk * D * share
        masks = {'none': 0, 'full': B * Tq * Tk, 'key': B * Tk}[case['mask']]
        pairs = B * H * _visible_pairs(case) * share * 2 * D
        if train:                                         # q, k, v, g in; y, dq, dk, dv out
            return {'bytes': int(size * (4 * nq + 4 * nk) + masks), 'flops': int(7 * pairs)}
        return {'bytes': int(size * (2 * nq + 2 * nk) + masks), 'flops': int(2 * pairs)}
    if case['op'] == 'linear':
        M, N, K = case['M'], case['N'], case['K']
        r, b = int(case['residual']), N * int(case['bias'])
        if train:
            return {'bytes': size * (2 * M * K + 2 * N * K + 2 * b + (2 + 2 * r) * M * N), 'flops': 6 * M * N * K}
        return {'bytes': size * (M * K + N * K + b + (1 + r) * M * N), 'flops': 2 * M * N * K}
    n, C = case['B'] * case['V'] * case['C'], case['C']
    if train:                                             # x, g in; y, dx out
        return {'bytes': 4 * n * size + 16 * C, 'flops': 30 * n}
    return {'bytes': 2 * n * size + 8 * C, 'flops': 10 * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def _act64(z, act):
    F = torch.nn.functional
    return {'none': lambda t: t, 'relu': F.relu, 'selu': F.selu, 'elu': F.elu, 'gelu': F.gelu, 'silu': F.silu}[act](z)


def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: None if t is None else t.detach().double().requires_grad_(True)  # noqa: E731
    if case['op'] == 'attention':
        B, Tq, Tk, H, Hk, D = (case[k] for k in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
        leaves = {'q': up(s['q']), 'k': up(s['k']), 'v': up(s['v'])}
        q = leaves['q'].reshape(B, Tq, Hk, H // Hk, D).permute(0, 2, 3, 1, 4)           # (B, Hk, n, Tq, D)
        k = leaves['k'].permute(0, 2, 1, 3)[:, :, None]
        v = leaves['v'].permute(0, 2, 1, 3)[:, :, None]
        kept = torch.ones((B, 1, 1, Tq, Tk), dtype=torch.bool, device='cuda')
        ends = s['lens'].long() if s['lens'] is not None else torch.full((B,), Tk, device='cuda')
        at = torch.arange(Tk, device='cuda')
        kept &= (at[None] < ends[:, None])[:, None, None, None]
        if case['causal']:
            rows = torch.arange(Tq, device='cuda')
            kept &= (at[None, None] - rows[None, :, None] <= (ends - Tq)[:, None, None])[:, None, None]
        if s['mask'] is not None:
            kept &= s['mask'][:, None]
        logits = (q @ k.transpose(-1, -2)) / math.sqrt(D)
        p = torch.softmax(logits.masked_fill(~kept, -1e300), dim=-1) * kept
        y = (p @ v).permute(0, 3, 1, 2, 4).reshape(B, Tq, H, D)
    elif case['op'] == 'linear':
        leaves = {x: up(s[x]) for x in ('x', 'w', 'b', 'r') if s[x] is not None}
        y = _act64(torch.nn.functional.linear(leaves['x'], leaves['w'], leaves.get('b')), case['act'])
        if 'r' in leaves:
            y = y + leaves['r']
    else:
        leaves = {x: up(s[x]) for x in ('x', 'w', 'b')}
        u = torch.nn.functional.group_norm(leaves['x'].transpose(1, 2), case['G'], leaves['w'], leaves['b'], 1e-5)
        y = _act64(u.transpose(1, 2), case['act'])
    out = {'y': y.detach()}
    if case['train']:
        grads = torch.autograd.grad(y, list(leaves.values()), s['g'].double())
        out.update(zip(('d' + k for k in leaves), grads))
    return out
