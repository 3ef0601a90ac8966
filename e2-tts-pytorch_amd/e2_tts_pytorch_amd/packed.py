"""Attention over packed documents and layer norm for autograd: the front end of the packed_attn / attn_decode / layernorm kernels.

The reference pads a batch of utterances to the longest one (collate_fn, trainer.py:61-82) and masks the rest; packed, the utterances of a batch lie one behind
the other and no row is padding.  Distance biases stand in for, or beside, rotary embeddings: `slopes` (linear in the distance) or RelativePositionBias
(learned, by buckets of distance)."""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import Function, forward_ad

from . import ops

__all__ = ['packed_attention', 'attn_decode', 'RelativePositionBias', 'LayerNorm', 'layer_norm']


def _no_tangents(what, *ts):
    """refuses forward-mode duals, which a call that goes past autograd (or hides an input in its options) would drop without a word"""
    if forward_ad._current_level < 0:             # (no dual level is open: nothing to unpack)
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ops.E2KError(f'{what}: no forward-mode gradients')


class _PackedAttnFn(Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, kw):
        train = any(ctx.needs_input_grad[:4])
        if not train:
            return ops.packed_attn_fwd(q, k, v, cu_q, cu_k, table=table, **kw)
        out, st = ops.packed_attn_fwd(q, k, v, cu_q, cu_k, table=table, train=True, **kw)
        # every tensor of the state goes through save_for_backward (changed in place it raises; hooks may pack it away), the numbers beside it
        ctx.save_for_backward(*(getattr(st, n) for n in st.TENSORS))
        ctx.numbers = {n: getattr(st, n) for n in st.NUMBERS}
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        st = ops.PackedAttnState(**dict(zip(ops.PackedAttnState.TENSORS, ctx.saved_tensors)), **ctx.numbers)
        need = ctx.needs_input_grad
        dq, dk, dv, dtable = ops.packed_attn_bwd(st, dout, need_table=need[3])
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dtable if need[3] else None, None, None, None


def packed_attention(q, k, v, cu_q, cu_k=None, *, len_q=None, len_k=None, prefix=None, max_q=0, max_k=0, causal=False, scale=None, softcap=0., slopes=None,
                     bias=None):
    """ops.packed_attn_fwd with gradients for q, k, v and the bias: q (Tq,H,64), k / v (Tk,Hkv,64) bf16, documents at the offsets cu_q / cu_k; `bias` a
    RelativePositionBias.  `slopes` are constants: a tensor that wants a gradient is refused.  Into a HIP graph capture a training pass with
    torch.autograd.grad (or the ops calls): accumulating into .grad of leaves that an eager graph still holds on another stream cannot be captured.
    -> (Tq,H,64) bf16"""
    if slopes is not None and slopes.requires_grad:
        raise ops.E2KError('packed_attention: slopes get no gradient; pass slopes.detach(), or learn a RelativePositionBias')
    table, buckets = (None, None) if bias is None else (bias.weight, bias.buckets)
    _no_tangents('packed_attention', q, k, v, slopes, table)
    kw = dict(len_q=len_q, len_k=len_k, prefix=prefix, max_q=max_q, max_k=max_k, causal=causal, scale=scale, softcap=softcap, slopes=slopes, buckets=buckets)
    if not torch.is_grad_enabled():              # (nothing is kept for a backward)
        return ops.packed_attn_fwd(q, k, v, cu_q, cu_k, table=table, **kw)
    return _PackedAttnFn.apply(q, k, v, table, cu_q, cu_k, kw)


def attn_decode(q, k_cache, v_cache, lens, *, scale=None, softcap=0., slopes=None, bias=None, out=None):
    """ops.attn_decode with a RelativePositionBias as its `bias` (no gradients: serving)"""
    _no_tangents('attn_decode', q, k_cache, v_cache, slopes, None if bias is None else bias.weight)
    table, buckets = (None, None) if bias is None else (bias.weight.detach(), bias.buckets)
    return ops.attn_decode(q.detach(), k_cache.detach(), v_cache.detach(), lens, scale=scale, softcap=softcap, slopes=slopes, table=table, buckets=buckets, out=out)


class RelativePositionBias(nn.Module):
    """learned bias per head and bucket of the distance key - query: `weight` (num_buckets, heads) fp32; one bucket per distance up close, logarithmically
    wider ones up to max_distance (ops.rel_buckets); causal: all buckets for keys before the query"""

    def __init__(self, heads, num_buckets=32, max_distance=128, causal=False):
        super().__init__()
        self.weight = nn.Parameter(torch.zeros(num_buckets, heads))
        nn.init.normal_(self.weight, std=0.02)
        self.register_buffer('buckets', ops.rel_buckets(num_buckets, max_distance, causal), persistent=False)

    @property
    def reach(self):
        return self.buckets.numel() // 2

    def forward(self, nq, nk):
        """the bias as a matrix (heads, nq, nk) of a document whose last query stands on its last key (what the kernels add, for inspection)"""
        d = torch.arange(nk, device=self.weight.device)[None] - torch.arange(nk - nq, nk, device=self.weight.device)[:, None]
        return self.weight[self.buckets.long()[d.clamp(-self.reach, self.reach) + self.reach]].permute(2, 0, 1)


def _ln_input(x):
    """x as rows that the kernels can read in place, a copy where its last dimension is strided or its rows overlap"""
    rows = x.reshape(-1, x.shape[-1])
    M, D = rows.shape
    return rows.contiguous() if (D > 1 and rows.stride(1) != 1) or (M > 1 and rows.stride(0) < D) else rows


class _LayerNormFn(Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, gamma_off, rows_per_batch, eps):
        y, mean, rstd = ops.layernorm_fwd(_ln_input(x), gamma, beta, gamma_off, rows_per_batch, eps)
        ctx.save_for_backward(x, gamma, mean, rstd)
        ctx.args = gamma_off, rows_per_batch, None if gamma is None else gamma.shape, None if beta is None else beta.shape
        return y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, gamma, mean, rstd = ctx.saved_tensors
        off, rpb, gs, bs = ctx.args
        need = ctx.needs_input_grad
        D = x.shape[-1]
        dx, dg, db = ops.layernorm_bwd(dy.reshape(-1, D).to(x.dtype), _ln_input(x), mean, rstd, gamma, off, rpb, need_weights=need[1] or need[2])

        def shaped(t, shape):            # rows of gamma / beta beyond the last batch element are not read: zero gradient
            if t.shape[0] == (1 if len(shape) == 1 else shape[0]):
                return t.view(shape)
            return torch.cat([t, t.new_zeros(shape[0] - t.shape[0], D)])
        return dx.view(x.shape) if need[0] else None, shaped(dg, gs) if need[1] else None, shaped(db, bs) if need[2] else None, None, None, None


def layer_norm(x, gamma=None, beta=None, gamma_off=0., rows_per_batch=0, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * (gamma + gamma_off) + beta over the last dimension, bf16 or fp32, with gradients; gamma / beta fp32 (D,), or (nb,D) with
    row m of x (counted over all leading dimensions) taking row m // rows_per_batch: the scale and shift of an adaptive norm"""
    return _LayerNormFn.apply(x, gamma, beta, float(gamma_off), int(rows_per_batch), float(eps))


class LayerNorm(nn.Module):
    """nn.LayerNorm over the last dimension on this package's kernels: same parameter names, fp32 parameters, bf16 or fp32 input"""

    def __init__(self, dim, eps=1e-5, elementwise_affine=True, bias=True):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(dim)) if elementwise_affine and bias else None
        self.dim = dim

    def forward(self, x):
        if x.shape[-1] != self.dim:
            raise ops.E2KError(f'LayerNorm({self.dim}): got rows of {x.shape[-1]}')
        return layer_norm(x, self.weight, self.bias, eps=self.eps)
