"""Token operators over the ``hno_attn_*`` / ``hno_linear_*`` / ``hno_gncl_*`` entry points of include/hno.h: softmax attention, the matrix
product with bias, activation and residual in its epilogue, and group norm with an activation -- on channels-last tokens, in fp32 or bf16, with
their backward passes.

Tensors are torch containers; no product, sum, norm or activation goes through ATen, and there is no CPU path (meta tensors get shape inference only).
What ATen does beside allocations: copies of operands whose layout the kernels do not take, and conversions of lengths and norm parameters of another type.
Parameters may stay fp32 next to bf16 activations: the matrix product then rounds its weight to bf16, as the bf16 convolutions do, and returns an fp32 gradient.
Gradients of gradients and forward-mode derivatives are refused.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from ._lib import check
from .ops import _m

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}                     # HNO_F32, HNO_BF16
_ACTS = {None: 0, 'none': 0, 'selu': 1, 'elu': 2, 'relu': 4, 'gelu': 5, 'silu': 6}
MAX_HEAD = 128


def act_id(act):
    """id of an activation of the token operators: None, 'none', 'selu', 'elu', 'relu', 'gelu' (exact), 'silu', or the torch function of that name"""
    if callable(act):
        act = getattr(act, '__name__', act)
    if act not in _ACTS:
        raise ValueError(f'activation {act!r} is not supported by the token operators ({", ".join(k for k in _ACTS if k)})')
    return _ACTS[act]


def _dtype(t, what):
    if t.dtype not in _DTYPES:
        raise ValueError(f'{what}: dtype {t.dtype} is not provided by the HIP path (torch.float32 or torch.bfloat16)')
    return _DTYPES[t.dtype]


def _sizes(what, *sizes):
    """the library takes sizes as 32-bit integers"""
    if max(sizes) > 0x7fffffff:
        raise ValueError(f'{what}: a size of {max(sizes)} is not provided')


def _same_device(what, first, *others):
    if not first.is_cuda:
        raise _lib.HnoError('the HIP path needs CUDA/HIP tensors; there is no CPU fallback (use oracle/ for CPU checks)')
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f'{what}: tensors on {first.device} and {t.device}')


def _call(fn, *args):
    """fn.run(...) -> result, kept; as a node of the autograd graph where a gradient can be asked for (4 us of host time: a call for one token took 24
    with a node that nobody asks, 20 without), and where a tensor may be dual: the node refuses it (forward-mode derivatives are not provided).
    The device of the first argument is the current one meanwhile: launches and workspaces go by it and its current stream."""
    if args[0].device.index != torch.cuda.current_device():
        with torch.cuda.device(args[0].device):
            return _call(fn, *args)
    if torch.is_grad_enabled():
        for t in args:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return _leaves(fn.apply(*args))
    return fn.apply(*args) if forward_ad._current_level >= 0 else fn.run(False, *args)[0]


def _leaves(y):
    """Refuses a capture that the backward pass could not survive.  A leaf's accumulation node belongs to the stream on which it was made and lives as long as
    any graph that holds it: one left over from another stream would join that stream to the capture in the backward pass, which ends the process."""
    stream = _stream(y)
    for node, _ in y.grad_fn.next_functions:
        if node is not None and hasattr(node, 'variable'):
            if node.metadata.setdefault('hno_stream', stream) != stream and torch.cuda.is_current_stream_capturing():
                raise RuntimeError('a graph of the same leaf, made on another stream before the capture, is still alive: delete its outputs first')
    return y


def _stream(t):
    """the current stream of the tensor's device, as the library takes it (torch.cuda.current_stream() builds a Stream object: 4 us of a 20 us call)"""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _once():
    """called by every backward pass: a graph of the gradients (create_graph) would hold nothing of these kernels"""
    if torch.is_grad_enabled():
        raise RuntimeError('the token operators cannot be differentiated twice')


def _p(t):
    return None if t is None else t.data_ptr()


def _ws(nbytes, device):
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


# ----------------------------------------------------------------------------------------------- attention
def _heads(t, esize):
    """a (B, T, H, D) operand as the kernels take it: unit stride along D, D a multiple of 8, rows 16-byte aligned and less than 2^24 elements apart --
    the tensor itself where it is so, else a copy padded with zeros (which change no score; padded channels of the result are cut off)"""
    D, step = t.shape[3], 16 // esize
    sb, st, sh, sd = t.stride()
    if not (D % 8 or sd != 1 or t.data_ptr() % 16 or sb % step or st % step or sh % step or st >= 1 << 24):
        return t
    if D % 8 == 0:
        return t.clone(memory_format=torch.contiguous_format)
    return torch.nn.functional.pad(t.contiguous(), (0, -D % 8))          # (pad keeps the order of the strides)


def _attn_args(q, k, v, mask, kv_lens, causal, scale):
    a = _lib.AttnArgs()
    B, Tq, H, Dk = q.shape
    a.dtype, a.B, a.Tq, a.Tk, a.H, a.Hk, a.Dk, a.Dv = _DTYPES[q.dtype], B, Tq, k.shape[1], H, k.shape[2], Dk, v.shape[3]
    a.causal, a.scale = int(causal), scale
    a.q, a.k, a.v, a.mask, a.kv_lens = _p(q), _p(k), _p(v), _p(mask), _p(kv_lens)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    if mask is not None:
        a.mask_stride[:] = [0 if n == 1 else s for n, s in zip(mask.shape, mask.stride())]
    return a


class AttentionFn(torch.autograd.Function):
    """out = softmax(scale q k^T) v over the visible keys; the backward pass recomputes the probabilities from lse (``attention`` has the
    contract)."""

    @staticmethod
    def run(train, q, k, v, mask, kv_lens, causal, scale):
        Dk, Dv = q.shape[3], v.shape[3]
        q, k, v = (_heads(t, t.element_size()) for t in (q, k, v))
        B, Tq, H, _ = q.shape
        out = torch.empty((B, Tq, H, v.shape[3]), device=q.device, dtype=q.dtype)
        lse = torch.empty((B, Tq, H), device=q.device, dtype=torch.float32) if train else None
        res = torch.empty_like(out) if train and q.dtype == torch.bfloat16 else None
        if out.numel():
            L = _lib.lib()
            a = _attn_args(q, k, v, mask, kv_lens, causal, scale)
            ref = ctypes.byref(a)
            n = L.hno_attn_workspace_bytes(ref, 0)
            ws = _ws(n, q.device)
            check(L.hno_attn_fwd(ref, _p(out), _p(res), _p(lse), _p(ws), n, _stream(q)), 'hno_attn_fwd')
        return out if out.shape[3] == Dv else out[..., :Dv].contiguous(), (q, k, v, mask, kv_lens, out, res, lse), (causal, scale, Dk, Dv)

    @staticmethod
    def forward(ctx, *args):
        y, kept, ctx.cfg = AttentionFn.run(True, *args)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    def backward(ctx, g):
        _once()
        q, k, v, mask, kv_lens, out, res, lse = ctx.saved_tensors
        causal, scale, Dk, Dv = ctx.cfg
        need_q, need_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        new = torch.empty if out.numel() else torch.zeros
        dq = new(q.shape, device=q.device, dtype=q.dtype) if need_q else None
        dk, dv = (new(t.shape, device=q.device, dtype=q.dtype) if need_kv else None for t in (k, v))
        if out.numel() and (need_q or k.shape[1]):                         # (without keys dk and dv are empty: there may be nothing to write)
            L = _lib.lib()
            g = _heads(g, g.element_size()).contiguous()
            a = _attn_args(q, k, v, mask, kv_lens, causal, scale)
            ref = ctypes.byref(a)
            n = L.hno_attn_workspace_bytes(ref, 1)
            ws = _ws(n, q.device)
            check(L.hno_attn_bwd(ref, _p(out), _p(res), _p(lse), _p(g), _p(dq), _p(dk), _p(dv), _p(ws), n, _stream(q)), 'hno_attn_bwd')
        dq, dk, dv = (t if t is None or t.shape[3] == D else t[..., :D] for t, D in ((dq, Dk), (dk, Dk), (dv, Dv)))
        return dq, dk if ctx.needs_input_grad[1] else None, dv if ctx.needs_input_grad[2] else None, None, None, None, None


def attention(q, k, v, *, causal=False, mask=None, kv_lens=None, scale=None):
    """Softmax attention on tokens: q (B, Tq, H, Dk), k (B, Tk, Hk, Dk), v (B, Tk, Hk, Dv) -> (B, Tq, H, Dv); all fp32 or all bf16.

    H is a multiple of Hk: query head h reads key head h // (H // Hk).  Head sizes 1 ... 128.  Any strides; rows that are not
    16-byte aligned or contiguous, and head sizes that are no multiple of 8, are copied.  ``scale`` (positive, default Dk ** -0.5) multiplies the scores.
    Visible to query i are the keys j < L with L = ``kv_lens[b]`` (integers (B,) on the device, clamped to 0 ... Tk; default Tk);
    with ``causal`` those with j <= i + L - Tq (the last query is aligned with the last key);
    with ``mask`` (bool, broadcastable to (B, H, Tq, Tk)) those that it marks True.  A query that sees no key gives zeros and has no gradient.
    Keys and values from L on, and those that a mask of shape (B, 1, 1, Tk) hides, may hold anything (inf, NaN); all others have to be finite, also
    where a mask hides them.  Additive (floating) masks are refused.  fp32 products are formed from three bf16 terms per value, so an
    infinity comes out as NaN.
    The relative error of a weight is about 2^-24 of the row's largest |scale q k| (in bf16 beside its rounding), in both passes; scores from 2^20 on are not provided.
    Differentiable in q, k, v; the probabilities are recomputed in the backward pass, memory grows with Tq + Tk only."""
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError('attention: q, k, v must be (batch, tokens, heads, channels)')
    B, Tq, H, Dk = q.shape
    _, Tk, Hk, Dv = v.shape
    if tuple(k.shape) != (B, Tk, Hk, Dk) or v.shape[0] != B:
        raise ValueError(f'attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not belong together')
    if Hk == 0 or H % Hk or H == 0:
        raise ValueError(f'attention: {H} query heads do not share {Hk} key heads evenly')
    if not 1 <= Dk <= MAX_HEAD or not 1 <= Dv <= MAX_HEAD:
        raise ValueError(f'attention: head sizes {Dk}, {Dv} are outside 1 ... {MAX_HEAD}')
    _sizes('attention', B, Tq, Tk, H)
    _dtype(q, 'attention')
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f'attention: q, k, v are {q.dtype}, {k.dtype}, {v.dtype}: one type is needed')
    scale = 1.0 / math.sqrt(Dk) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError('attention: scale must be positive, from 1e-30 to 1e30')
    if mask is not None:
        if mask.dtype != torch.bool:
            raise ValueError('attention: mask must be bool (True: visible); additive masks are not provided')
        if mask.ndim > 4 or any(m not in (1, n) for m, n in zip(reversed(mask.shape), (Tk, Tq, H, B))):
            raise ValueError(f'attention: mask {tuple(mask.shape)} does not broadcast to {(B, H, Tq, Tk)}')
        mask = mask[(None,) * (4 - mask.ndim)]
    if kv_lens is not None:
        if tuple(kv_lens.shape) != (B,) or kv_lens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f'attention: kv_lens must be {B} integers')
    if q.is_meta:
        return _m((B, Tq, H, Dv), q.dtype)
    _same_device('attention', q, k, v, mask, kv_lens)
    if kv_lens is not None and (kv_lens.dtype != torch.int32 or not kv_lens.is_contiguous()):
        kv_lens = kv_lens.clamp(0, Tk).to(torch.int32).contiguous()
    return _call(AttentionFn, q, k, v, mask, kv_lens, bool(causal), scale)


# ----------------------------------------------------------------------------------------------- linear
def _rows(x):
    """x (..., K) as (M, K) with unit stride along K -> (view or copy, row stride)"""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 and x2.shape[1] != 1:
        x2 = x2.contiguous()
    ld = x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]
    if ld < x2.shape[1]:          # rows that share memory (expanded views)
        x2 = x2.contiguous()
        ld = x2.shape[1]
    return x2, ld


def _bf16_weight(w):
    out = torch.empty(w.shape, device=w.device, dtype=torch.bfloat16)
    check(_lib.lib().hno_cast_f32_bf16(_p(w), _p(out), w.numel(), _stream(w)), 'hno_cast_f32_bf16')
    return out


class LinearFn(torch.autograd.Function):
    """y = act(x W^T + b) + r with the whole epilogue in the product's kernel (``linear`` has the contract)."""

    @staticmethod
    def run(train, x, weight, bias, residual, act):
        N, K = weight.shape
        y = torch.empty(tuple(x.shape[:-1]) + (N,), device=x.device, dtype=x.dtype)
        z, w, x2 = None, weight.contiguous(), x
        if y.numel():
            L = _lib.lib()
            x2, ldx = _rows(x)
            M = x2.shape[0]
            if w.dtype != x.dtype:
                w = _bf16_weight(w)
            b = None if bias is None else bias.contiguous()
            r = None if residual is None else residual.contiguous()
            z = torch.empty((M, N), device=x.device, dtype=x.dtype) if train and act else None
            dt = _DTYPES[x.dtype]
            n = L.hno_linear_workspace_bytes(dt, M, N, K, act, 0)
            ws = _ws(n, x.device)
            check(L.hno_linear_fwd(dt, _p(x2), ldx, _p(w), _p(b), 0 if b is None else _DTYPES[b.dtype], _p(r), _p(z), _p(y), M, N, K, act, _p(ws), n,
                                   _stream(x)), 'hno_linear_fwd')
        return y, (x2, w, z, weight), (act, x.shape, None if bias is None else bias.dtype)

    @staticmethod
    def forward(ctx, *args):
        y, kept, ctx.cfg = LinearFn.run(True, *args)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    def backward(ctx, g):
        _once()
        x, w, z, weight = ctx.saved_tensors
        act, xshape, bias_dtype = ctx.cfg
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        N, K = w.shape
        if not g.numel():
            zeros = lambda shape, dt: torch.zeros(shape, device=g.device, dtype=dt)  # noqa: E731
            return (zeros(xshape, g.dtype) if need_x else None, zeros((N, K), weight.dtype) if need_w else None,
                    zeros((N,), bias_dtype) if need_b else None, g if need_r else None, None)
        dx = dw = db = None
        if need_x or need_w or need_b:
            L = _lib.lib()
            gc = g.contiguous()
            x2, ldx = _rows(x)
            M = x2.shape[0]
            if need_x:
                dx = torch.empty(xshape, device=g.device, dtype=g.dtype)
            if need_w:
                own = weight.is_leaf and weight.dtype == torch.float32 and weight.is_contiguous()
                dw = ops._grad_buffer(weight) if own else torch.empty((N, K), device=g.device, dtype=weight.dtype)
            if need_b:
                db = torch.empty(N, device=g.device, dtype=bias_dtype)
            dt = _DTYPES[g.dtype]
            n = L.hno_linear_workspace_bytes(dt, M, N, K, act, 1)
            ws = _ws(n, g.device)
            check(L.hno_linear_bwd(dt, _p(gc), _p(z), _p(x2), ldx, _p(w), _p(dx), _p(dw), 0 if dw is None else _DTYPES[dw.dtype], _p(db),
                                   0 if db is None else _DTYPES[db.dtype], M, N, K, act, _p(ws), n, _stream(g)), 'hno_linear_bwd')
        return dx, dw, db, g if need_r else None, None


def linear(x, weight, bias=None, *, act=None, residual=None):
    """act(x W^T + bias) + residual: x (..., K), weight (N, K), bias (N,), residual (..., N) -> (..., N), in x's type (fp32 or bf16).

    ``act``: see ``act_id``.  weight is of x's type, or fp32 next to a bf16 x (rounded to bf16 for the product; its gradient is fp32); bias is of either
    type.  residual has the result's shape and type.  x may be any view; rows of equal stride are read where they lie.
    fp32 products of more than four rows are formed from three bf16 terms per value (errors as in fp32; infinities and NaN as in fp32).
    Differentiable in all four; with an activation the backward pass keeps the product's result, in x's type."""
    a = act_id(act)
    if x.ndim < 1 or weight.ndim != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f'linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not belong together')
    N, K = weight.shape
    if N == 0 or K == 0:
        raise ValueError('linear: empty weight')
    _sizes('linear', math.prod(x.shape[:-1]), N, K)
    _dtype(x, 'linear')
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f'linear: weight is {weight.dtype}, x is {x.dtype}')
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f'linear: bias must be ({N},) of {x.dtype} or fp32')
    if residual is not None and (tuple(residual.shape) != tuple(x.shape[:-1]) + (N,) or residual.dtype != x.dtype):
        raise ValueError(f'linear: residual must have the shape and type of the result, {tuple(x.shape[:-1]) + (N,)} {x.dtype}')
    if x.is_meta:
        return _m(tuple(x.shape[:-1]) + (N,), x.dtype)
    _same_device('linear', x, weight, bias, residual)
    return _call(LinearFn, x, weight, bias, residual, a)


# ----------------------------------------------------------------------------------------------- group norm
class GroupNormClFn(torch.autograd.Function):
    """act(GroupNorm(G, C)(x)) on channels-last tokens (``group_norm`` has the contract)."""

    @staticmethod
    def run(train, x, weight, bias, groups, eps, act):
        x = x.contiguous()
        y = torch.empty_like(x)
        B, C = x.shape[0], x.shape[-1]
        w, b = (None if t is None else (t if t.dtype == torch.float32 else t.float()).contiguous() for t in (weight, bias))
        mr = torch.empty((B, groups, 2), device=x.device, dtype=torch.float32)
        if x.numel():
            L = _lib.lib()
            V = x.numel() // (B * C)
            n = L.hno_gncl_workspace_bytes(B, V, C, groups)
            ws = _ws(n, x.device)
            check(L.hno_gncl_fwd(_DTYPES[x.dtype], _p(x), _p(w), _p(b), _p(y), _p(mr), _p(ws), n, B, V, C, groups, eps, act, _stream(x)), 'hno_gncl_fwd')
        return y, (x, w, b, mr), (groups, act, None if weight is None else weight.dtype, None if bias is None else bias.dtype)

    @staticmethod
    def forward(ctx, *args):
        y, kept, ctx.cfg = GroupNormClFn.run(True, *args)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    def backward(ctx, g):
        _once()
        x, w, b, mr = ctx.saved_tensors
        groups, act, wt, bt = ctx.cfg
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        B, C = x.shape[0], x.shape[-1]
        new = torch.empty if x.numel() else torch.zeros
        dx = torch.empty_like(x) if need_x else None
        dw, db = (new(C, device=x.device, dtype=torch.float32) if n else None for n in (need_w, need_b))
        if x.numel():
            L = _lib.lib()
            g = g.contiguous()
            V = x.numel() // (B * C)
            n = L.hno_gncl_workspace_bytes(B, V, C, groups)
            ws = _ws(n, x.device)
            check(L.hno_gncl_bwd(_DTYPES[x.dtype], _p(g), _p(x), _p(w), _p(b), _p(mr), _p(dx), _p(dw), _p(db), _p(ws), n, B, V, C, groups, act, _stream(x)),
                  'hno_gncl_bwd')
        return dx, dw if wt in (None, torch.float32) or dw is None else dw.to(wt), db if bt in (None, torch.float32) or db is None else db.to(bt), None, None, None


def group_norm(x, num_groups, weight=None, bias=None, *, eps=1e-5, act=None):
    """act(gamma (x - mean) / sqrt(var + eps) + beta) on channels-last x (B, ..., C), fp32 or bf16, statistics per sample and group of
    C / num_groups neighbouring channels over all positions; weight, bias (C,) fp32 or x's type; at most 65535 samples.  ``act``: see ``act_id``.
    Statistics: means and squared distances from them, in fp32 and, over more than a few thousand values, joined in 64 bits.  Differentiable in x,
    weight, bias; the backward pass keeps x and the statistics."""
    a = act_id(act)
    num_groups, eps = int(num_groups), float(eps)
    if x.ndim < 2:
        raise ValueError('group_norm: x must be (batch, ..., channels)')
    C = x.shape[-1]
    if num_groups < 1 or C == 0 or C % num_groups:
        raise ValueError(f'group_norm: {C} channels do not fall into {num_groups} groups')
    if not eps >= 0.0:
        raise ValueError('group_norm: eps must not be negative')
    _sizes('group_norm', x.shape[0], C)
    _dtype(x, 'group_norm')
    for t in (weight, bias):
        if t is not None and (tuple(t.shape) != (C,) or t.dtype not in (x.dtype, torch.float32)):
            raise ValueError(f'group_norm: weight and bias must be ({C},) of {x.dtype} or fp32')
    if x.is_meta:
        return _m(x.shape, x.dtype)
    _same_device('group_norm', x, weight, bias)
    return _call(GroupNormClFn, x, weight, bias, num_groups, eps, a)
