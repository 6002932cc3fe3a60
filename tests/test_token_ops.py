"""The token operators (ops_tokens: attention, linear, group_norm) against their definitions in float64.

Tolerances are bounds by arithmetic, element by element, computed next to the float64 result: E = 2^-24 for each fp32 operation (n E for a sum of n
terms), U = half a step of the operand type (bf16 2^-8, fp32 E) for each value that is rounded to it: the probabilities and score gradients that are
operands of a second product, the kept argument of an activation, the result."""
import gc
import math

import pytest
import torch
import torch.nn.functional as F

E = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: E}
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope='module')
def ot():
    import multimodal_3d_image_segmentation_amd as pkg
    return pkg.ops_tokens


def rand(shape, dtype, seed, scale=1.0, shift=0.0, device='cuda'):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + shift).to(dtype).to(device)


def close(name, got, want, bound):
    got, bound = got.double(), bound + 1e-30
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f'{name}: not finite'
    ratio = ((got - want).abs() / bound).max() if got.numel() else torch.tensor(0.0)
    print(f'{name}: worst error is {float(ratio):.3f} of its bound')
    assert ratio <= 1.0, (name, float(ratio))


# ------------------------------------------------------------------------------------------------ attention
def attention_reference(q, k, v, g, causal=False, mask=None, lens=None, scale=None):
    """float64 results and the bounds of the kernels' errors: {name: (value, bound)}"""
    u = HALF[q.dtype]
    B, Tq, H, Dk = q.shape
    Tk, Hk, Dv = v.shape[1:]
    n = H // Hk
    scale = 1.0 / math.sqrt(Dk) if scale is None else scale
    q, g = q.detach().double().transpose(1, 2), g.double().transpose(1, 2)
    k, v = (t.detach().double().transpose(1, 2).repeat_interleave(n, 1) for t in (k, v))
    L = torch.full((B,), Tk, device=q.device) if lens is None else lens.long().clamp(0, Tk)
    j, i = torch.arange(Tk, device=q.device), torch.arange(Tq, device=q.device)
    on = (j[None, None] < L[:, None, None]).expand(B, Tq, Tk)
    if causal:
        on = on & (j[None, None] <= i[None, :, None] + (L - Tq)[:, None, None])
    on = on[:, None].expand(B, H, Tq, Tk)
    if mask is not None:
        on = on & mask
    # rows of k and v that nobody sees may hold anything
    seen = on.any(dim=2)[..., None]
    k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)
    rows = on.any(dim=3, keepdim=True)
    q, g = torch.where(rows, q, 0.0), torch.where(rows, g, 0.0)
    T = lambda t: t.transpose(2, 3)  # noqa: E731
    s = (q @ T(k)) * scale
    s = s.masked_fill(~on, -1e300)
    p = torch.softmax(s, -1) * on if Tk else s
    o = p @ v
    dp = g @ T(v)
    D = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - D)
    # ---- bounds
    size = (s.abs() * on).amax(-1, keepdim=True) if Tk else torch.zeros_like(o[..., :1])
    ss = ((q.abs() @ T(k.abs())) * scale * on).amax(-1, keepdim=True) if Tk else size
    rp = 2 * (Dk + 6) * E * ss + E * (32 + 8 * size + Tk)                       # relative error of a probability
    pv = p @ v.abs()
    eo = (2 * u + rp + Tk * E) * pv
    eD = (g.abs() * eo).sum(-1, keepdim=True) + (Dv + 4) * E * (g.abs() * (o.abs() + pv)).sum(-1, keepdim=True)
    eds = ds.abs() * (rp + u + 4 * E) + p * ((Dv + 4) * E * (g.abs() @ T(v.abs())) + eD)
    dq, edq = (ds @ k) * scale, scale * ((eds + Tk * E * ds.abs()) @ k.abs())
    dk, edk = (T(ds) @ q) * scale, scale * (T(eds + Tq * n * E * ds.abs()) @ q.abs())
    dv, edv = T(p) @ g, T((u + rp + Tq * n * E) * p) @ g.abs()
    fold = lambda t: t.unflatten(1, (Hk, n)).sum(2)  # noqa: E731
    out = {'y': (o, eo), 'dq': (dq, edq), 'dk': (fold(dk), fold(edk)), 'dv': (fold(dv), fold(edv))}
    return {x: (a.transpose(1, 2), (e + (u + 4 * E) * a.abs()).transpose(1, 2)) for x, (a, e) in out.items()}


def check_attention(ot, q, k, v, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    B, Tq, H, _ = q.shape
    g = rand((B, Tq, H, v.shape[3]), q.dtype, 77, 0.5)
    y = ot.attention(q, k, v, **kw)
    grads = torch.autograd.grad(y, (q, k, v), g)
    kw['lens'] = kw.pop('kv_lens', None)
    want = attention_reference(q, k, v, g, **kw)
    for name, t in zip(('y', 'dq', 'dk', 'dv'), (y.detach(),) + grads):
        assert t.dtype == q.dtype
        close(name, t, *want[name])
    with torch.no_grad():
        kw['kv_lens'] = kw.pop('lens')
        assert torch.equal(ot.attention(q, k, v, **kw), y)          # nothing that only a backward pass reads changes the result


# B, Tq, Tk, H, Hk, Dk, Dv, causal
ATTENTION = [(1, 1, 1, 1, 1, 32, 32, False), (2, 5, 7, 4, 2, 16, 16, True), (1, 64, 64, 2, 2, 64, 64, False), (2, 130, 65, 3, 1, 40, 40, False),
             (1, 257, 257, 4, 1, 128, 128, True), (2, 33, 300, 2, 2, 96, 96, True), (1, 300, 33, 2, 1, 80, 80, True), (3, 1, 700, 8, 2, 128, 128, False),
             (1, 129, 191, 2, 1, 7, 13, False), (2, 70, 90, 2, 2, 33, 128, True), (1, 1, 4099, 2, 1, 64, 64, True), (2, 200, 0, 2, 1, 32, 32, False),
             (1, 700, 1200, 1, 1, 64, 64, False), (1, 3, 1000, 6, 3, 48, 24, True)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('B,Tq,Tk,H,Hk,Dk,Dv,causal', ATTENTION)
def test_attention_sizes(ot, B, Tq, Tk, H, Hk, Dk, Dv, causal, dtype):
    q, k, v = rand((B, Tq, H, Dk), dtype, 1), rand((B, Tk, Hk, Dk), dtype, 2), rand((B, Tk, Hk, Dv), dtype, 3)
    check_attention(ot, q, k, v, causal=causal)


# packed heads over several tiles; runs of a long axis on either side, few and many; a long causal triangle; one query of many heads
ATTENTION_RUNS = [(1, 100, 260, 8, 2, 64, 64, True), (2, 127, 130, 3, 1, 128, 128, False), (1, 2100, 70, 2, 2, 64, 64, False), (1, 300, 5000, 2, 1, 96, 96, False),
                  (1, 1100, 1300, 2, 1, 32, 32, True), (1, 1500, 900, 2, 2, 128, 128, True), (2, 1, 3000, 16, 2, 80, 80, False), (1, 4, 9000, 4, 4, 32, 32, True)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('B,Tq,Tk,H,Hk,Dk,Dv,causal', ATTENTION_RUNS)
def test_attention_runs(ot, B, Tq, Tk, H, Hk, Dk, Dv, causal, dtype):
    q, k, v = rand((B, Tq, H, Dk), dtype, 31), rand((B, Tk, Hk, Dk), dtype, 32), rand((B, Tk, Hk, Dv), dtype, 33)
    check_attention(ot, q, k, v, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('D', [32, 96, 128])
def test_attention_mask_lengths_and_causal_together(ot, D, causal, dtype):
    B, Tq, Tk, H, Hk = 3, 140, 230, 4, 2
    q, k, v = rand((B, Tq, H, D), dtype, 34), rand((B, Tk, Hk, D), dtype, 35), rand((B, Tk, Hk, D), dtype, 36)
    gen = torch.Generator().manual_seed(37)
    mask = (torch.rand((B, H, Tq, Tk), generator=gen) < 0.6).cuda()
    mask[1, :, 20:90] = False                                           # rows that see nothing
    lens = torch.tensor([230, 97, 0], device='cuda', dtype=torch.int32)
    check_attention(ot, q, k, v, causal=causal, mask=mask, kv_lens=lens)
    check_attention(ot, q, k, v, causal=causal, mask=mask[:, :1, :1], kv_lens=lens)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('Tq', [1, 40, 150])
def test_attention_lengths(ot, Tq, causal, dtype):
    """padded keys: lengths of zero, one, the whole and beyond it; what lies behind a length is not looked at"""
    Tk, lens = 150, [0, 1, 31, 64, 150, 400, -3]
    q, k, v = rand((7, Tq, 4, 64), dtype, 4), rand((7, Tk, 2, 64), dtype, 5), rand((7, Tk, 2, 64), dtype, 6)
    for b, n in enumerate(lens):
        k[b, max(n, 0):], v[b, max(n, 0):] = math.nan, math.inf
    for t in (torch.int32, torch.int64):
        check_attention(ot, q, k, v, causal=causal, kv_lens=torch.tensor(lens, device='cuda', dtype=t))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', [(2, 4, 100, 170), (2, 1, 100, 170), (1, 1, 100, 170), (100, 170), (2, 1, 1, 170), (2, 4, 1, 170), (2, 1, 100, 1), (170,)])
@pytest.mark.parametrize('causal', [False, True])
def test_attention_masks(ot, shape, causal, dtype):
    q, k, v = rand((2, 100, 4, 48), dtype, 7), rand((2, 170, 2, 48), dtype, 8), rand((2, 170, 2, 48), dtype, 9)
    m = torch.rand(shape, generator=torch.Generator().manual_seed(10)) < 0.6
    if m.shape[-1] > 1:
        m[..., 64:128] = False                                         # a whole tile of keys without any
    if m.ndim >= 2 and m.shape[-2] > 1:
        m[..., 17, :] = False                                          # an empty row
        m[..., 64:100, :] = False                                      # and a run of them
    m = m.cuda()
    if shape == (2, 1, 1, 170):                                        # a padding mask: the hidden keys and values may hold anything
        k = torch.where(m[:, 0, 0, :, None, None], k, math.nan)
        v = torch.where(m[:, 0, 0, :, None, None], v, math.inf)
    check_attention(ot, q, k, v, causal=causal, mask=m)
    if len(shape) == 4:
        check_attention(ot, q, k, v, causal=causal, mask=m.transpose(2, 3).contiguous().transpose(2, 3), kv_lens=torch.tensor([160, 33], device='cuda'))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_attention_empty_rows_are_zero_and_nan_in_them_stays_out(ot, dtype):
    q, k, v = (rand((1, 90, 2, 64), dtype, s).requires_grad_(True) for s in (11, 12, 13))
    m = torch.ones(1, 1, 90, 90, dtype=torch.bool, device='cuda')
    m[:, :, 40:72] = False
    bad = q.detach().clone()
    bad[:, 40:72] = math.nan
    g = rand((1, 90, 2, 64), dtype, 14)
    runs = []
    for x in (q, bad.requires_grad_(True)):
        y = ot.attention(x, k, v, mask=m)
        runs.append((y,) + torch.autograd.grad(y, (x, k, v), g))
        assert (y[:, 40:72] == 0).all() and (runs[-1][1][:, 40:72] == 0).all()
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('D', [40, 13])
def test_attention_strides_and_alignment(ot, D, dtype):
    """packed projections, head-major and channel-major storage, odd offsets: the same values, the same results"""
    B, T, H = 2, 75, 3
    flat = rand((B, T, 3, H, D), dtype, 15)
    q, k, v = flat.unbind(2)
    want = ot.attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    g = rand((B, T, H, D), dtype, 16)
    forms = {'packed': flat, 'head-major': flat.permute(2, 0, 3, 1, 4).contiguous().permute(1, 3, 0, 2, 4),
             'channel-major': flat.permute(0, 2, 3, 4, 1).contiguous().permute(0, 4, 1, 2, 3)}
    odd = torch.empty(flat.numel() + 1, device='cuda', dtype=dtype)[1:].view(flat.shape)
    odd.copy_(flat)
    forms['odd offset'] = odd
    ref = None
    for name, f in forms.items():
        f = f.detach().requires_grad_(True)
        y = ot.attention(*f.unbind(2), causal=True)
        assert torch.equal(y, want), name
        (gf,) = torch.autograd.grad(y, f, g if name != 'packed' else g.transpose(0, 1).contiguous().transpose(0, 1))
        ref = gf if ref is None else ref
        assert torch.equal(gf, ref), name


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_attention_one_sharp_key(ot, dtype):
    """scores of hundreds: the weights are 0 and 1, and the score gradients cancel"""
    q, k, v = rand((1, 66, 2, 64), dtype, 17, 30.0), rand((1, 130, 2, 64), dtype, 18, 8.0), rand((1, 130, 2, 64), dtype, 19)
    check_attention(ot, q, k, v, scale=1.0)


@pytest.mark.gpu
def test_attention_far_rows(ot):
    """offsets beyond 32 bits: the last batch entry starts 2^31 elements in (the storage is never touched as a whole)"""
    B, Tk, Hk, D = 2, 40, 1, 64
    store = torch.empty((1 << 31) + 4096 + Tk * Hk * D, device='cuda', dtype=torch.bfloat16)
    k = store.as_strided((B, Tk, Hk, D), ((1 << 31) + 4096, Hk * D, D, 1))
    k.copy_(rand((B, Tk, Hk, D), torch.bfloat16, 20))
    q, v = rand((B, 9, 2, D), torch.bfloat16, 21), rand((B, Tk, Hk, D), torch.bfloat16, 22)
    assert torch.equal(ot.attention(q, k, v), ot.attention(q, k.contiguous(), v))
    t = store.as_strided((1, 3, 1, D), (0, 1 << 30, 0, 1))              # and tokens that lie 2^30 elements apart
    t.copy_(rand((1, 3, 1, D), torch.bfloat16, 23))
    assert torch.equal(ot.attention(q[:1], t, t), ot.attention(q[:1], t.contiguous(), t.contiguous()))


# ------------------------------------------------------------------------------------------------ linear
ACT64 = {None: lambda z: z, 'selu': F.selu, 'elu': F.elu, 'relu': F.relu, 'gelu': F.gelu, 'silu': F.silu}


def slope64(z, act):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(ACT64[act](z).sum(), z)[0] if act else torch.ones_like(z)


def check_linear(ot, x, w, b, r, act):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    x, w = leaves[:2]
    b = leaves[2] if b is not None else None
    r = leaves[-1] if r is not None else None
    u, uw = HALF[x.dtype], HALF[w.dtype]
    y = ot.linear(x, w, b, act=act, residual=r)
    assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (w.shape[0],)
    g = rand(y.shape, x.dtype, 55)
    grads = dict(zip('xwbr' if b is not None and r is not None else 'xwb' if b is not None else 'xwr' if r is not None else 'xw',
                     torch.autograd.grad(y, leaves, g)))
    N, K = w.shape
    X, G = x.detach().double().reshape(-1, K), g.double().reshape(-1, N)
    M = X.shape[0]
    W = (w.detach().to(x.dtype) if uw != u else w.detach()).double()     # an fp32 weight beside bf16 activations is used in bf16
    z = X @ W.t() + (b.detach().double() if b is not None else 0.0)
    ez = (K + 8) * E * (X.abs() @ W.abs().t() + (b.detach().double().abs() if b is not None else 0.0))
    R = r.detach().double().reshape(-1, N) if r is not None else torch.zeros_like(z)
    a = ACT64[act](z)
    want = a + R
    # 1.8: no activation here has a first or second derivative beyond it (selu: 1.76)
    close('y', y.detach().reshape(-1, N), want, 1.8 * ez + 24 * E * (a.abs() + z.abs()) + (u + 4 * E) * want.abs() + 2 * E * R.abs())
    slope = slope64(z, act)
    dz = G * slope
    edz = G.abs() * (1.8 * (ez + u * z.abs()) + 24 * E) if act else torch.zeros_like(dz)
    if act in ('selu', 'relu'):                                          # the slope jumps at 0
        edz = edz + G.abs() * (z.abs() <= ez)
    used = edz + (u * (dz.abs() + edz) if act else 0.0)                  # as an operand of the products
    dx = dz @ W
    close('dx', grads['x'].reshape(-1, K), dx, (used + (N + 8) * E * dz.abs()) @ W.abs() + u * dx.abs())
    dw = dz.t() @ X
    close('dw', grads['w'], dw, (used + (M + 8) * E * dz.abs()).t() @ X.abs() + uw * dw.abs())
    assert grads['w'].dtype == w.dtype
    if b is not None:
        db = dz.sum(0)
        close('db', grads['b'], db, (edz + (M + 8) * E * dz.abs()).sum(0) + HALF[b.dtype] * db.abs())
        assert grads['b'].dtype == b.dtype
    if r is not None:
        assert torch.equal(grads['r'], g)


LINEAR = [(1, 1, 1), (1, 24, 40), (4, 256, 512), (7, 33, 65), (128, 128, 128), (129, 130, 131), (300, 96, 24), (257, 384, 96), (1000, 24, 17), (2, 1000, 2049),
          (65, 8, 2000), (3000, 40, 48), (513, 264, 328)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('M,N,K', LINEAR)
def test_linear_sizes(ot, M, N, K, dtype):
    x, w = rand((M, K), dtype, 1), rand((N, K), dtype, 2, 1.0 / math.sqrt(K))
    check_linear(ot, x, w, rand((N,), dtype, 3), rand((M, N), dtype, 4), 'gelu')
    check_linear(ot, x, w, None, None, None)


# results of hundreds of large tiles in the forward product, in dx and in dw; rows and columns that end inside a tile, contractions that end inside a step
@pytest.mark.gpu
@pytest.mark.parametrize('M,N,K', [(3500, 3592, 72), (3600, 40, 3592), (40, 3592, 3608), (3500, 3590, 200), (3500, 3592, 65)])
def test_linear_large_tiles(ot, M, N, K):
    x, w = rand((M, K), torch.bfloat16, 21), rand((N, K), torch.bfloat16, 22, 1.0 / math.sqrt(K))
    check_linear(ot, x, w, rand((N,), torch.bfloat16, 23), rand((M, N), torch.bfloat16, 24), 'silu')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('act', list(ACT64))
@pytest.mark.parametrize('bias,residual', [(True, False), (False, True), (True, True)])
def test_linear_epilogue(ot, act, bias, residual, dtype):
    x, w = rand((2, 5, 31, 72), dtype, 5, 2.0), rand((88, 72), dtype, 6, 0.3)
    check_linear(ot, x, w, rand((88,), dtype, 7) if bias else None, rand((2, 5, 31, 88), dtype, 8) if residual else None, act)


@pytest.mark.gpu
def test_linear_fp32_parameters_with_bf16_activations(ot):
    x = rand((70, 64), torch.bfloat16, 9)
    check_linear(ot, x, rand((48, 64), torch.float32, 10, 0.1), rand((48,), torch.float32, 11), None, 'silu')
    check_linear(ot, x, rand((48, 64), torch.bfloat16, 10, 0.1), rand((48,), torch.float32, 11), None, 'silu')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_linear_strides(ot, dtype):
    w = rand((40, 48), dtype, 12)
    base = rand((9, 7, 100), dtype, 13)
    forms = [base[..., 4:52], base[..., 3:51], base[:, ::2, 8:56], base[0, 0, :48].expand(9, 48), base.transpose(0, 2)[:48].permute(2, 1, 0),
             base[0, 0, :48]]
    for x in forms:
        x = x.detach().requires_grad_(True)
        y = ot.linear(x, w, act='elu')
        g = rand((40,), dtype, 14).expand(y.shape)                      # a gradient without strides of its own
        (dx,) = torch.autograd.grad(y, x, g)
        c = x.detach().contiguous().requires_grad_(True)
        yc = ot.linear(c, w, act='elu')
        assert torch.equal(y, yc) and torch.equal(dx, torch.autograd.grad(yc, c, g.contiguous())[0])
    wt = rand((48, 40), dtype, 15)
    assert torch.equal(ot.linear(base[..., :48], wt.t()), ot.linear(base[..., :48], wt.t().contiguous()))


@pytest.mark.gpu
def test_linear_large_activation_arguments(ot):
    """saturated arguments give the limits, NaN stays NaN"""
    x = torch.tensor([[1e30], [-1e30], [300.0], [-300.0], [0.0], [math.nan]], device='cuda')
    w = torch.ones(1, 1, device='cuda')
    for act in ACT64:
        xx = x.clone().requires_grad_(True)
        y = ot.linear(xx, w, act=act)
        (dx,) = torch.autograd.grad(y.sum(), xx)
        want, slope = ACT64[act](x.double()), slope64(x.double(), act)
        assert torch.isnan(y[5]).all() and torch.allclose(y[:5].double(), want[:5], rtol=1e-6), act
        ok = slice(0, 4) if act in ('selu', 'relu') else slice(0, 5)
        assert torch.allclose(dx[ok].double(), slope[ok], rtol=1e-6, atol=1e-6), act


@pytest.mark.gpu
def test_linear_infinite_activation_arguments(ot):
    """an infinite bias gives the activations' limits"""
    x, w = torch.zeros(3, 4, device='cuda'), torch.ones(2, 4, device='cuda')
    b = torch.tensor([math.inf, -math.inf], device='cuda')
    for act, low in ((None, -math.inf), ('selu', -1.7580993408473766), ('elu', -1.0), ('relu', 0.0), ('gelu', 0.0), ('silu', 0.0)):
        xx = x.clone().requires_grad_(True)
        y = ot.linear(xx, w, b, act=act)
        (dx,) = torch.autograd.grad(y, xx, torch.ones_like(y))
        assert torch.isinf(y[:, 0]).all() and (y[:, 0] > 0).all(), act
        assert (y[:, 1] == low).all() or torch.allclose(y[:, 1], torch.tensor(low, device='cuda'), rtol=2e-7, atol=0), act
        slope = {None: 2.0, 'selu': 1.0507009873554805}.get(act, 1.0)      # of column 0, and 0 of column 1
        assert torch.allclose(dx, torch.full_like(dx, slope), rtol=2e-7, atol=0), act


# ------------------------------------------------------------------------------------------------ group norm
def check_group_norm(ot, x, G, w, b, act, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    x = leaves[0]
    w, b = (leaves[1] if w is not None else None), (leaves[-1] if b is not None else None)
    u = HALF[x.dtype]
    y = ot.group_norm(x, G, w, b, eps=eps, act=act)
    g = rand(x.shape, x.dtype, 66)
    grads = torch.autograd.grad(y, leaves, g)
    B, C = x.shape[0], x.shape[-1]
    X, Gr = x.detach().double().reshape(B, -1, G, C // G), g.double().reshape(B, -1, G, C // G)
    V, n = X.shape[1], X.shape[1] * (C // G)
    W = (w.detach().double() if w is not None else torch.ones(C, device=x.device, dtype=torch.float64)).view(G, C // G)
    Bt = (b.detach().double() if b is not None else torch.zeros(C, device=x.device, dtype=torch.float64)).view(G, C // G)
    mean, var = X.mean((1, 3), keepdim=True), X.var((1, 3), unbiased=False, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    xh = (X - mean) * rstd
    z = xh * W + Bt
    a, slope = ACT64[act](z), slope64(z, act)
    # statistics: runs of at most 512 fp32 additions of (x - first)^2, joined in 64 bits; then each value in a handful of operations
    spread = ((X - X[:, :1]) ** 2).mean((1, 3), keepdim=True) / (var + eps)
    er = 512 * E * (1 + spread) + 4 * E                                  # relative error of rstd
    em = 512 * E * (X - X[:, :1]).abs().mean((1, 3), keepdim=True) + 2 * E * mean.abs()
    eh = xh.abs() * (er + 4 * E) + rstd * (em + 2 * E * (X.abs() + mean.abs()))
    ez = eh * W.abs() + 4 * E * (z.abs() + (xh * W).abs() + Bt.abs())
    close('y', y.detach(), a.reshape(x.shape), (1.8 * ez + 24 * E * (a.abs() + z.abs()) + (u + 2 * E) * a.abs()).reshape(x.shape))
    du = Gr * slope
    edu = Gr.abs() * (1.8 * ez + 24 * E) if act else torch.zeros_like(du)
    if act in ('selu', 'relu'):
        edu = edu + Gr.abs() * (z.abs() <= ez)
    t, et = du * W, edu * W.abs() + 2 * E * (du * W).abs()
    s = 512 * E
    m1, m2 = t.mean((1, 3), keepdim=True), (t * xh).mean((1, 3), keepdim=True)
    e1 = (et + s * t.abs()).mean((1, 3), keepdim=True)
    e2 = (et * xh.abs() + t.abs() * eh + s * (t * xh).abs()).mean((1, 3), keepdim=True)
    dx = rstd * (t - m1 - xh * m2)
    edx = dx.abs() * (er + 4 * E) + rstd * (et + e1 + eh * m2.abs() + xh.abs() * e2 + 4 * E * (t.abs() + m1.abs() + (xh * m2).abs()))
    close('dx', grads[0], dx.reshape(x.shape), (edx + u * dx.abs()).reshape(x.shape))
    if w is not None:
        dw = (du * xh).sum((0, 1))
        close('dw', grads[1], dw.reshape(C), ((edu * xh.abs() + du.abs() * eh + s * (du * xh).abs()).sum((0, 1)) + HALF[w.dtype] * dw.abs()).reshape(C))
    if b is not None:
        db = du.sum((0, 1))
        close('db', grads[-1], db.reshape(C), ((edu + s * du.abs()).sum((0, 1)) + HALF[b.dtype] * db.abs()).reshape(C))


GROUP_NORM = [((1, 1, 2), 1), ((2, 4), 1), ((2, 3, 5, 8), 2), ((1, 7, 9, 11, 24), 6), ((3, 1000, 64), 8), ((2, 333, 40), 5), ((1, 60, 2500), 4), ((2, 50, 3), 3),
              ((1, 5000, 16), 16), ((2, 100, 2048), 32), ((1, 30, 2056), 1), ((4, 17, 33), 11), ((1, 1, 512), 8), ((2, 4096, 8), 1), ((1, 20, 1200), 2)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape,G', GROUP_NORM)
def test_group_norm_sizes(ot, shape, G, dtype):
    x, C = rand(shape, dtype, 1, 1.5, 0.3), shape[-1]
    if len(shape) == 2 and C // G < 2 or x[0].numel() // G < 2:
        pytest.skip('one value per group')
    check_group_norm(ot, x, G, rand((C,), torch.float32, 2, 0.2, 1.0), rand((C,), torch.float32, 3, 0.2), 'silu')
    check_group_norm(ot, x, G, None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('act', list(ACT64))
def test_group_norm_epilogue(ot, act, dtype):
    x = rand((2, 6, 7, 8, 48), dtype, 4, 1.0, 0.5)
    w, b = rand((48,), dtype, 5, 0.2, 1.0), rand((48,), dtype, 6, 0.2)
    check_group_norm(ot, x, 6, w, b, act)
    check_group_norm(ot, x, 6, None, b, act)
    check_group_norm(ot, x, 6, w.float(), None, act, eps=1e-3)


@pytest.mark.gpu
def test_group_norm_far_from_zero(ot):
    """channels a thousand deviations from zero, each at its own offset"""
    x = rand((2, 500, 24), torch.float32, 7) + 1000.0 * rand((24,), torch.float32, 8)
    check_group_norm(ot, x, 24, None, None, None)
    check_group_norm(ot, x, 6, None, None, 'elu')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_group_norm_constant_input_and_strides(ot, dtype):
    x = torch.full((2, 90, 16), 3.0, device='cuda', dtype=dtype)
    assert (ot.group_norm(x, 4) == 0).all()
    base = rand((2, 91, 17), dtype, 9)
    for v in (base[:, 1:, 1:], base[:, ::3, :16], base.transpose(1, 2), base[:1].expand(3, 91, 17)[..., :16]):
        v = v.detach().requires_grad_(True)
        c = v.detach().contiguous().requires_grad_(True)
        G = v.shape[-1] // (13 if v.shape[-1] == 91 else 4)
        y, yc = ot.group_norm(v, G, act='gelu'), ot.group_norm(c, G, act='gelu')
        assert torch.equal(y, yc)
        g = rand(y.shape, dtype, 10)
        assert torch.equal(torch.autograd.grad(y, v, g)[0], torch.autograd.grad(yc, c, g)[0])


# ------------------------------------------------------------------------------------------------ together
def block(ot, p, x, mask, heads, shared):
    """one transformer block on channels-last tokens (B, T, C)"""
    B, T, C = x.shape
    D = C // heads
    h = ot.group_norm(x, 4, p['g1'], p['b1'])
    qkv = ot.linear(h, p['wqkv'], p['bqkv'])
    q, k, v = qkv.split((C, shared * D, shared * D), dim=-1)
    a = ot.attention(q.unflatten(-1, (heads, D)), k.unflatten(-1, (shared, D)), v.unflatten(-1, (shared, D)), mask=mask)
    x = ot.linear(a.flatten(2), p['wo'], p['bo'], residual=x)
    h = ot.group_norm(x, 4, p['g2'], p['b2'], act='silu')
    h = ot.linear(h, p['w1'], p['bb1'], act='gelu')
    return ot.linear(h, p['w2'], p['bb2'], residual=x)


def block64(p, x, mask, heads, shared):
    B, T, C = x.shape
    D = C // heads
    gn = lambda t, g, b: F.group_norm(t.transpose(1, 2), 4, g, b).transpose(1, 2)  # noqa: E731
    q, k, v = F.linear(gn(x, p['g1'], p['b1']), p['wqkv'], p['bqkv']).split((C, shared * D, shared * D), dim=-1)
    q, k, v = (t.unflatten(-1, (-1, D)).transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(heads // shared, 1) for t in (k, v))
    s = (q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill(~mask, -1e300)
    a = ((torch.softmax(s, -1) * mask) @ v).transpose(1, 2).reshape(B, T, C)
    x = F.linear(a, p['wo'], p['bo']) + x
    h = F.gelu(F.linear(F.silu(gn(x, p['g2'], p['b2'])), p['w1'], p['bb1']))
    return F.linear(h, p['w2'], p['bb2']) + x


def block_parameters(C, heads, shared, dtype):
    D, wide = C // heads, 2 * C
    n = C + 2 * shared * D
    shapes = {'wqkv': (n, C), 'bqkv': (n,), 'wo': (C, C), 'bo': (C,), 'w1': (wide, C), 'bb1': (wide,), 'w2': (C, wide), 'bb2': (C,)}
    p = {k: rand(s, dtype, 30 + i, 1.0 / math.sqrt(s[-1]) if len(s) == 2 else 0.1) for i, (k, s) in enumerate(shapes.items())}
    for i, k in enumerate(('g1', 'g2')):
        p[k], p['b' + k[1]] = rand((C,), torch.float32, 40 + i, 0.1, 1.0), rand((C,), torch.float32, 50 + i, 0.1)
    return {k: t.requires_grad_(True) for k, t in p.items()}


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,tol', [(torch.float32, 2e-5), (torch.bfloat16, 0.05)], ids=['fp32', 'bf16'])
def test_block_forward_and_gradients(ot, dtype, tol):
    """The operators in a row.  Tolerance (2-norm): each of ~12 roundings in a row adds at most one half step in relative 2-norm: 12 x 2^-8 = 0.047 in
    bf16; in fp32 sums of up to 192 terms: 12 x 192 x 2^-24 / sqrt(192) ~ 1e-5."""
    B, T, C, heads, shared = 2, 130, 96, 6, 2
    p = block_parameters(C, heads, shared, dtype)
    x = rand((B, T, C), dtype, 20).requires_grad_(True)
    mask = (torch.rand((B, 1, 1, T), generator=torch.Generator().manual_seed(21)) < 0.8).cuda()
    y = block(ot, p, x, mask, heads, shared)
    g = rand(y.shape, dtype, 22)
    got = [y.detach(), *torch.autograd.grad(y, [x, *p.values()], g)]
    p64 = {k: t.detach().double().requires_grad_(True) for k, t in p.items()}
    x64 = x.detach().double().requires_grad_(True)
    y64 = block64(p64, x64, mask, heads, shared)
    want = [y64.detach(), *torch.autograd.grad(y64, [x64, *p64.values()], g.double())]
    for name, a, b in zip(['y', 'x', *p], got, want):
        err = float((a.double() - b).norm() / b.norm())
        print(f'{name}: {err:.2e}')
        assert err <= tol, (name, err)


@pytest.mark.gpu
def test_gradients_against_differences(ot):
    """directional derivatives of the fp32 operators: (f(x + h d) - f(x - h d)) / 2 h = <gradient, d> up to h^2 and E / h"""
    p = block_parameters(64, 4, 2, torch.float32)
    x = rand((1, 33, 64), torch.float32, 23).requires_grad_(True)
    mask = torch.ones((1, 1, 33, 33), dtype=torch.bool, device='cuda').tril()
    g = rand((1, 33, 64), torch.float32, 24)
    f = lambda t: float((block(ot, p, t, mask, 4, 2).double() * g.double()).sum())  # noqa: E731
    (gx,) = torch.autograd.grad(block(ot, p, x, mask, 4, 2), x, g)
    d = rand(x.shape, torch.float32, 25)
    h = 2.0 ** -8
    with torch.no_grad():
        num = (f(x + h * d) - f(x - h * d)) / (2 * h)
    want = float((gx.double() * d.double()).sum())
    scale = float(gx.double().norm() * d.double().norm())
    assert abs(num - want) <= 2e-3 * scale, (num, want, scale)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_runs_are_bit_equal_on_any_stream(ot, dtype):
    p = block_parameters(64, 4, 1, dtype)
    x = rand((2, 700, 64), dtype, 26).requires_grad_(True)
    mask = torch.ones((1, 1, 700, 700), dtype=torch.bool, device='cuda').tril()
    g = rand(x.shape, dtype, 27)

    def step():
        y = block(ot, p, x, mask, 4, 1)
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], g)]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    third = step()                       # at the same time as the other stream's
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_captured_step_replays(ot, dtype):
    """forward and backward of the block in a graph, replayed on new inputs between eager runs; two graphs alive at once"""
    B, T, C = 2, 300, 64
    mask = torch.ones((1, 1, T, T), dtype=torch.bool, device='cuda').tril()
    g = rand((B, T, C), dtype, 28)
    xs = [rand((B, T, C), dtype, 60 + i) for i in range(4)]

    def step(x, p):
        y = block(ot, p, x, mask, 4, 2)
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], g)]
    p = block_parameters(C, 4, 2, dtype)
    want = [step(x.detach().clone().requires_grad_(True), p) for x in xs]
    graphs = []
    for i in range(2):
        pg = {k: t.detach().clone().requires_grad_(True) for k, t in p.items()}
        x = xs[0].detach().clone().requires_grad_(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, pg)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, pg)
        graphs.append((graph, x, out, pg))                                 # (a graph keeps no input alive)
    for n in (1, 3, 0, 2):
        for i, (graph, x, out, _) in enumerate(graphs):
            at = (n + i) % 4
            with torch.no_grad():
                x.copy_(xs[at])
            graph.replay()
        step(xs[n].detach().clone().requires_grad_(True), p)              # eager work between the replays
        torch.cuda.synchronize()
        for i, (graph, x, out, _) in enumerate(graphs):
            for a, b in zip(out, want[(n + i) % 4]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_capture_with_a_live_eager_graph_is_refused(ot):
    """the accumulation node of a leaf that an eager graph holds belongs to another stream than the capture's"""
    x = torch.randn(8, 32, device='cuda', dtype=torch.bfloat16)
    w = torch.randn(16, 32, device='cuda', requires_grad=True)
    alive = ot.linear(x, w)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match='still alive'):
        with torch.cuda.graph(g, stream=side):
            ot.linear(x, w)
    alive.float().sum().backward()
    want = w.grad.clone()
    del alive
    gc.collect()
    w.grad = None
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        y = ot.linear(x, w)
        y.backward(torch.ones_like(y))
    for _ in range(3):
        w.grad.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(w.grad, want)


@pytest.mark.gpu
def test_weight_gradients_reach_registered_destinations(ot):
    """an fp32 weight's gradient is written where the data-parallel replica wants it; a weight that is used twice gets the sum"""
    import multimodal_3d_image_segmentation_amd as pkg
    x = rand((2, 30, 16), torch.bfloat16, 1)
    w, u = (rand((16, 16), torch.float32, n).requires_grad_(True) for n in (2, 3))

    def grads():
        w.grad = u.grad = None
        y = ot.linear(ot.linear(ot.linear(x, w, act='gelu'), u), w)
        y.backward(rand(y.shape, y.dtype, 4))
        return w.grad, u.grad
    want = [g.clone() for g in grads()]
    flat = torch.full((512,), 7.0, device='cuda')
    old = pkg.ops.set_grad_destinations({w: flat[:256].view(16, 16), u: flat[256:].view(16, 16)})
    try:
        for _ in range(2):
            pkg.ops.new_grad_pass()
            got = grads()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert got[1].data_ptr() == flat[256:].data_ptr()
    finally:
        pkg.ops.set_grad_destinations(None)
        pkg.ops._grad_dest = old


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_empty_batches(ot, dtype):
    """no sample, no token: empty results, and parameters whose gradients are zero"""
    p = lambda *s: torch.randn(s, device='cuda', dtype=dtype).requires_grad_(True)  # noqa: E731
    for B, Tq in ((0, 5), (2, 0)):
        q, k, v = p(B, Tq, 4, 16), p(B, 7, 2, 16), p(B, 7, 2, 24)
        y = ot.attention(q, k, v, causal=True)
        assert y.shape == (B, Tq, 4, 24)
        for t, g in zip((q, k, v), torch.autograd.grad(y, (q, k, v), torch.ones_like(y))):
            assert g.shape == t.shape and (g == 0).all()
        x, w, b = p(B, Tq, 16), p(8, 16), p(8)
        y = ot.linear(x, w, b, act='silu', residual=p(B, Tq, 8))
        assert y.shape == (B, Tq, 8)
        for t, g in zip((x, w, b), torch.autograd.grad(y, (x, w, b), torch.ones_like(y))):
            assert g.shape == t.shape and (g == 0).all()
        gamma, beta = p(16), p(16)
        y = ot.group_norm(x, 4, gamma, beta, act='elu')
        assert y.shape == x.shape
        for t, g in zip((x, gamma, beta), torch.autograd.grad(y, (x, gamma, beta), torch.ones_like(y))):
            assert g.shape == t.shape and g.dtype == t.dtype and (g == 0).all()


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def test_attention_refusals(ot):
    t = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)  # noqa: E731
    q, k = t(1, 4, 4, 32), t(1, 6, 2, 32)
    bad = [((q[0], k, k), {}), ((q, k, t(1, 5, 2, 32)), {}), ((q, t(2, 6, 2, 32), k), {}), ((q, t(1, 6, 2, 16), k), {}), ((q, t(1, 6, 3, 32), t(1, 6, 3, 32)), {}),
           ((t(1, 4, 4, 129), t(1, 6, 2, 129), k), {}), ((q, k, t(1, 6, 2, 129)), {}), ((q.half(), k.half(), k.half()), {}), ((q, k.bfloat16(), k), {}),
           ((q.double(), k.double(), k.double()), {}), ((q, k, k), {'scale': 0.0}), ((q, k, k), {'scale': -1.0}), ((q, k, k), {'scale': 1e-31}), ((q, k, k), {'scale': 1e31}), ((q, k, k), {'scale': math.inf}),
           ((q, k, k), {'scale': math.nan}), ((q, k, k), {'mask': t(4, 6)}), ((q, k, k), {'mask': t(4, 5).bool()}), ((q, k, k), {'mask': t(1, 1, 1, 4, 6).bool()}),
           ((q, k, k), {'kv_lens': t(2).int()}), ((q, k, k), {'kv_lens': t(1)}), ((t(1, 4, 4, 0), t(1, 6, 2, 0), k), {}), ((t(1, 4, 0, 32), k, k), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            ot.attention(*args, **kw)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ot.attention(q, k, k)


def test_linear_refusals(ot):
    t = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)  # noqa: E731
    x, w = t(3, 8), t(5, 8)
    bad = [((x, t(5, 7)), {}), ((x, t(5, 8, 1)), {}), ((x, t(0, 8)), {}), ((t(3, 0), t(5, 0)), {}), ((x.half(), w.half()), {}), ((x, w.bfloat16()), {}),
           ((x, w, t(4)), {}), ((x, w, t(5).half()), {}), ((x, w), {'act': 'tanh'}), ((x, w), {'act': torch.tanh}), ((x, w), {'residual': t(5)}),
           ((x, w), {'residual': t(3, 5).bfloat16()}), ((x.bfloat16(), w.half()), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            ot.linear(*args, **kw)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ot.linear(x, w)


def test_group_norm_refusals(ot):
    t = lambda *s: torch.zeros(s)  # noqa: E731
    bad = [((t(8), 2), {}), ((t(2, 8), 3), {}), ((t(2, 8), 0), {}), ((t(2, 0), 1), {}), ((t(2, 8), 2, t(7)), {}), ((t(2, 8), 2, t(8).half()), {}),
           ((t(2, 8).half(), 2), {}), ((t(2, 8), 2), {'eps': -1.0}), ((t(2, 8), 2), {'eps': math.nan}), ((t(2, 8), 2), {'act': 'softmax'})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            ot.group_norm(*args, **kw)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ot.group_norm(t(2, 8), 2)


def test_entry_points_check_before_any_launch():
    import ctypes

    import multimodal_3d_image_segmentation_amd as pkg
    L = pkg._lib.lib()
    a = pkg._lib.AttnArgs()
    ok = dict(dtype=1, B=1, Tq=4, Tk=4, H=2, Hk=1, Dk=32, Dv=32, scale=1.0, q=4096, k=4096, v=4096)

    def attn(ws=0, out=4096, **kw):
        for k, v in {**ok, **kw}.items():
            setattr(a, k, v)
        return L.hno_attn_fwd(ctypes.byref(a), out, None, None, None, ws, None)
    for kw in ({'dtype': 2}, {'Tq': 0}, {'Tk': -1}, {'H': 3, 'Hk': 2}, {'scale': 0.0}, {'scale': float('nan')}, {'q': None}, {'k': None}, {'out': None}, {'out': 4098}):
        assert attn(**kw) == -1, kw
    assert attn(Dk=36) == -1 and attn(q=4100) == -1
    assert attn(Dk=136) == -2 and attn(B=70000000) == -2
    assert L.hno_attn_fwd(None, None, None, None, None, 0, None) == -1
    assert attn(Tk=100000, Tq=1) == -1 and b'workspace' in L.hno_last_error()
    assert L.hno_attn_bwd(ctypes.byref(a), 4096, None, 4096, 4096, None, 4096, None, 4096, 1 << 40, None) == -1      # dk without dv
    assert L.hno_linear_fwd(0, 4096, 8, 4096, None, 0, None, None, 4096, 0, 8, 8, 0, None, 0, None) == -1
    assert L.hno_linear_fwd(0, 4096, 7, 4096, None, 0, None, None, 4096, 8, 8, 8, 0, None, 0, None) == -1
    assert L.hno_linear_fwd(0, 4096, 8, 4096, None, 0, None, None, 4096, 8, 8, 8, 3, None, 0, None) == -1            # sigmoid is not one of theirs
    assert L.hno_linear_fwd(0, 4096, 100000, 4096, None, 0, None, None, 4096, 8, 8, 100000, 0, None, 0, None) == -1 and b'workspace' in L.hno_last_error()
    assert L.hno_linear_bwd(0, 4096, None, 4096, 8, 4096, 4096, 4096, 0, None, 0, 8, 8, 8, 5, 4096, 1 << 40, None) == -1   # gelu without z
    assert L.hno_gncl_fwd(0, 4096, None, None, 4096, 4096, 4096, 0, 1, 8, 8, 2, 1e-5, 0, None) == -1 and b'workspace' in L.hno_last_error()
    assert L.hno_gncl_fwd(0, 4096, None, None, 4096, 4096, 4096, 1 << 40, 1, 8, 8, 3, 1e-5, 0, None) == -1
    assert L.hno_gncl_bwd(0, 4096, 4096, None, None, 4096, None, None, None, 4096, 1 << 40, 1, 8, 8, 2, 0, None) == -1


def test_sizes_beyond_32_bits_are_refused(ot):
    """a row count of 2^32 + 1 would reach the library as 1"""
    m = lambda *s: torch.empty(s, device='meta', dtype=torch.bfloat16)  # noqa: E731
    n = 2 ** 32 + 1
    for call in (lambda: ot.linear(m(n, 8), m(4, 8)), lambda: ot.linear(m(2 ** 16, 2 ** 16, 8), m(4, 8)), lambda: ot.linear(m(2, 8), m(n, 8)),
                 lambda: ot.attention(m(n, 2, 1, 8), m(n, 2, 1, 8), m(n, 2, 1, 8)), lambda: ot.attention(m(1, 2, 1, 8), m(1, n, 1, 8), m(1, n, 1, 8)),
                 lambda: ot.group_norm(m(n, 2, 8), 2), lambda: ot.group_norm(m(2, 2, n - 1), 2)):
        with pytest.raises(ValueError, match='size'):
            call()
    import ctypes

    import multimodal_3d_image_segmentation_amd as pkg
    L = pkg._lib.lib()
    # more threads than a grid holds, and statistics whose index passes 32 bits
    a = pkg._lib.AttnArgs()
    for kw in (dict(B=1, Tq=1 << 28, H=2), dict(B=1 << 20, Tq=1, H=16), dict(B=1 << 20, Tq=400, H=1)):
        for k, v in {**dict(dtype=1, Tk=4, Hk=1, Dk=32, Dv=32, scale=1.0, q=4096, k=4096, v=4096), **kw}.items():
            setattr(a, k, v)
        assert L.hno_attn_fwd(ctypes.byref(a), 4096, None, None, None, 0, None) == -2
    assert L.hno_linear_fwd(0, 4096, 8, 4096, None, 0, None, None, 4096, 1 << 30, 512, 8, 0, None, 0, None) == -2
    assert L.hno_gncl_fwd(0, 4096, None, None, 4096, 4096, 4096, 1 << 62, 65535, 1, 32768, 32768, 1e-5, 0, None) == -2


def test_meta_tensors_give_shapes(ot):
    m = lambda *s: torch.empty(s, device='meta', dtype=torch.bfloat16)  # noqa: E731
    assert ot.attention(m(2, 5, 4, 32), m(2, 7, 2, 32), m(2, 7, 2, 16)).shape == (2, 5, 4, 16)
    assert ot.linear(m(2, 5, 8), m(3, 8)).shape == (2, 5, 3) and ot.group_norm(m(2, 5, 8), 4).dtype == torch.bfloat16


@pytest.mark.gpu
def test_no_second_derivative(ot):
    x = rand((2, 9, 8), torch.float32, 1).requires_grad_(True)
    for y in (ot.group_norm(x, 2, act='silu'), ot.linear(x, rand((4, 8), torch.float32, 2), act='gelu'),
              ot.attention(x.unflatten(2, (1, 8)), x.unflatten(2, (1, 8)), x.unflatten(2, (1, 8)))):
        with pytest.raises(RuntimeError, match='twice'):
            torch.autograd.grad(y.sum(), x, create_graph=True)


# ------------------------------------------------------------------------------------------------ the attention network's softmax
def softmax_mha64(op, x):
    """the operator of reference nets/hartley_mha.py:136-222 on one input without the transform, its activation a softmax over the keys, in float64"""
    from oracle import hno_oracle as O
    wq, wk, wv, wo = (w.detach().double() for w in (op.weight_query, op.weight_key, op.weight_value, op.weight_out))
    q, k, v = (torch.einsum('zoi,bidhw->bzodhw', w, x) for w in (wq, wk, wv))
    if op.patch_size is not None:
        q, k, v = (O._group3d(t, op.patch_size) for t in (q, k, v))
    shape = q.shape[3:]
    q, k, v = (t.flatten(3) for t in (q, k, v))
    att = torch.softmax(torch.einsum('bzcq,bzck->bzqk', q, k) / math.sqrt(k.shape[2]), dim=-1)
    out = torch.einsum('bzqk,bzck->bzcq', att, v).unflatten(3, shape)
    if op.patch_size is not None:
        out = O._ungroup3d(out, wv.shape[1], op.patch_size)
    return torch.einsum('oi,bidhw->bodhw', wo, out.flatten(1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize('patch', [None, (2, 2, 2), (1, 2, 1)])
def test_hartley_attention_with_softmax(patch):
    import functools

    from multimodal_3d_image_segmentation_amd.nets.hartley_mha import HartleyMultiHeadAttention
    torch.manual_seed(3)
    op = HartleyMultiHeadAttention(12, 12, 4, (2, 3, 4), patch, attention_activation=functools.partial(F.softmax, dim=-1), use_transform=False).cuda()
    x = rand((2, 12, 4, 6, 8), torch.float32, 4, 3.0).requires_grad_(True)
    y = op(x)
    g = rand(y.shape, torch.float32, 5)
    grads = torch.autograd.grad(y, [x, *op.parameters()], g)
    x64 = x.detach().double().requires_grad_(True)
    want = softmax_mha64(op, x64)
    wx, = torch.autograd.grad(want, x64, g.double())
    # four products of at most 192 terms and a softmax of scores below 32: some 500 E in the worst case
    for a, b in ((y.detach(), want.detach()), (grads[0], wx)):
        assert float((a.double() - b).abs().max() / b.abs().max()) < 500 * E
    h = 2.0 ** -7                                        # the parameters' gradients against differences, along one direction each
    with torch.no_grad():
        for p, gp in zip(op.parameters(), grads[1:]):
            d, keep = rand(p.shape, torch.float32, 6), p.detach().clone()
            f = []
            for sign in (1, -1):
                p.copy_(keep + sign * h * d)
                f.append(float((softmax_mha64(op, x64) * g.double()).sum()))
            p.copy_(keep)
            num, got = (f[0] - f[1]) / (2 * h), float((gp.double() * d.double()).sum())
            assert abs(num - got) <= 1e-2 * float(gp.double().norm() * d.double().norm()), (num, got)


@pytest.mark.gpu
def test_attention_network_trains_with_softmax():
    import functools

    import multimodal_3d_image_segmentation_amd as pkg
    from multimodal_3d_image_segmentation_amd.nets import custom_losses
    torch.manual_seed(0)
    make = lambda dev: pkg.nets.HartleyMHASeg(2, 3, 8, 2, 2, (3, 4, 4), (1, 2, 2), attention_activation=torch.nn.Softmax(dim=-1), device=dev)  # noqa: E731
    model = make(None).cuda()
    x = rand((1, 2, 24, 20, 28), torch.float32, 7)
    lab = torch.randint(0, 3, (1, 1, 24, 20, 28), device='cuda').float()
    loss = custom_losses.PCCLoss()(model(x), pkg.ops.labels_prepare(lab, 3))
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert make('meta')(torch.empty(1, 2, 24, 20, 28, device='meta')).shape == (1, 3, 24, 20, 28)


def test_softmax_over_keys_is_recognised():
    import functools

    from multimodal_3d_image_segmentation_amd.nets.hartley_mha import softmax_over_keys as s
    assert s(functools.partial(F.softmax, dim=-1)) and s(functools.partial(torch.softmax, dim=3)) and s(torch.nn.Softmax(-1))
    assert not any(s(f) for f in (F.softmax, functools.partial(F.softmax, dim=1), functools.partial(F.softmax, dim=-1, dtype=torch.float64),
                                  functools.partial(F.log_softmax, dim=-1), torch.nn.Softmax(1), F.selu, None))


class TokenNet(torch.nn.Module):
    """a transformer block over the voxels of an image, its classes behind a softmax"""

    def __init__(self, ot, cin, classes, width, heads):
        super().__init__()
        self.ot, self.heads = ot, heads
        p = lambda *s: torch.nn.Parameter(torch.randn(s) * s[-1] ** -0.5)  # noqa: E731
        self.win, self.qkv, self.wo, self.out = p(width, cin), p(3 * width, width), p(width, width), p(classes, width)
        self.gamma, self.beta = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))

    def __deepcopy__(self, memo):
        new = TokenNet.__new__(TokenNet)
        torch.nn.Module.__init__(new)
        new.ot, new.heads = self.ot, self.heads
        for n, q in self.named_parameters():
            setattr(new, n, torch.nn.Parameter(q.detach().clone()))
        return new

    def forward(self, x):
        ot = self.ot
        t = ot.linear(x.flatten(2).transpose(1, 2), self.win, act='gelu')
        q, k, v = ot.linear(ot.group_norm(t, 2, self.gamma, self.beta), self.qkv).unflatten(2, (3, self.heads, -1)).unbind(2)
        t = ot.linear(ot.attention(q, k, v).flatten(2), self.wo, residual=t)
        return torch.softmax(ot.linear(t, self.out), -1).transpose(1, 2).unflatten(2, x.shape[2:])


@pytest.mark.gpu
@pytest.mark.parametrize('net', ['tokens', 'hartley'])
@pytest.mark.parametrize('split', ['0', '1'])
def test_captured_training_step(ot, monkeypatch, net, split):
    """the training loop's captured step over the token operators: loss and gradients of the eager step, on every replay"""
    import multimodal_3d_image_segmentation_amd as pkg
    from multimodal_3d_image_segmentation_amd import ops
    from multimodal_3d_image_segmentation_amd.experiments import train_test as tt
    from multimodal_3d_image_segmentation_amd.nets import custom_losses
    monkeypatch.setenv('HNO_SPLIT_STREAMS', split)
    monkeypatch.setenv('HNO_TRAIN_GRAPH_QUIET', '1')
    torch.manual_seed(9)
    if net == 'tokens':
        model = TokenNet(ot, 2, 3, 16, 2).cuda()
    else:
        model = pkg.nets.HartleyMHASeg(2, 3, 8, 2, 2, (3, 4, 4), (1, 2, 2), attention_activation=torch.nn.Softmax(dim=-1)).cuda()
    loss_fn = custom_losses.PCCLoss()
    x = rand((2, 2, 16, 20, 16), torch.float32, 17)
    y = torch.randint(0, 3, (2, 1, 16, 20, 16), device='cuda').float()
    params = list(model.parameters())

    def eager():
        lab = ops.labels_prepare(y, 3)
        loss = loss_fn(model(x), lab)
        loss.backward()
        res = float(loss.detach()), [p.grad.clone() for p in params]
        for p in params:
            p.grad = None
        return res
    want, grads = eager()
    cap = tt.CapturedStep(model, loss_fn, 3)
    assert cap.step(x, y) is None                          # the first sight of a shape runs eagerly
    for _ in range(3):
        loss = cap.step(x, y)
        assert loss is not None
        torch.cuda.synchronize()
        assert abs(float(loss) - want) < 2e-6
        for p, g in zip(params, grads):                    # the halves of a split batch are summed in another order
            assert float((p.grad - g).norm()) <= 2e-4 * float(g.norm()) + 1e-9
        eager_again = model(x)                             # eager work between the replays
        del eager_again
