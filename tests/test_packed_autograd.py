"""packed_attention, attn_decode and layer_norm under autograd's other machinery: forward-mode duals, saved-tensor hooks, recomputation, inputs as views."""
import pytest
import torch
from torch.autograd import forward_ad

from test_packed_attn import offsets

bf16, f32 = torch.bfloat16, torch.float32


def attn_inputs(dev, heads=2):
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(33, heads, 64, generator=g).to(bf16).to(dev) for _ in range(4))
    return q, k, v, do, offsets([20, 13], dev)


@pytest.mark.parametrize('grad', [True, False], ids=['grad', 'no_grad'])
def test_forward_mode_is_refused(emu, grad):
    """a tangent has no way through these operators: it is refused wherever it sits, never dropped"""
    import e2_tts_pytorch_amd as pkg
    q, k, v, do, cu = attn_inputs('cpu')
    bias = pkg.RelativePositionBias(2, 8, 16)
    slopes, n = torch.ones(2), torch.tensor([20], dtype=torch.int32)
    kc = k[None]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: pkg.packed_attention(dual(q), k, v, cu), lambda: pkg.packed_attention(q, dual(k), v, cu), lambda: pkg.packed_attention(q, k, dual(v), cu),
                 lambda: pkg.packed_attention(q, k, v, cu, slopes=dual(slopes)), lambda: pkg.attn_decode(dual(q[:1]), kc, kc, n),
                 lambda: pkg.attn_decode(q[:1], dual(kc), kc, n), lambda: pkg.attn_decode(q[:1], kc, dual(kc), n),
                 lambda: pkg.attn_decode(q[:1], kc, kc, n, slopes=dual(slopes)), lambda: pkg.layer_norm(dual(slopes[None])), ]
        weight = bias.weight.detach()
        del bias.weight
        bias.weight = dual(weight)
        calls += [lambda: pkg.packed_attention(q, k, v, cu, bias=bias), lambda: pkg.attn_decode(q[:1], kc, kc, n, bias=bias)]
        for i, f in enumerate(calls):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()
                print('not refused:', i)
        assert pkg.packed_attention(q, k, v, cu, slopes=slopes).shape == q.shape and pkg.attn_decode(q[:1], kc, kc, n).shape == (1, 2, 64)


@pytest.mark.parametrize('table', [False, True], ids=['plain', 'table'])
def test_saved_tensors_go_through_the_hooks(dev, table, monkeypatch):
    """all that the backward reads can be packed away: nothing of it stays alive beside the hooks, and what they unpack is what counts"""
    import gc
    import weakref

    import e2_tts_pytorch_amd as pkg
    from e2_tts_pytorch_amd import ops
    q, k, v, do, cu = attn_inputs(dev)
    bias = pkg.RelativePositionBias(2, 8, 16).to(dev) if table else None
    extra = [bias.weight] if table else []
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(pkg.packed_attention(*leaves, cu, bias=bias), leaves + extra, do)
    kept, plain = [], ops.packed_attn_fwd

    def watched(*a, **kw):
        out, st = plain(*a, **kw)
        kept.extend(weakref.ref(t) for t in (st.q, st.k, st.v, st.lo, st.lse2))
        return out, st
    monkeypatch.setattr(ops, 'packed_attn_fwd', watched)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (t.detach().cpu().clone(), t.device), lambda p: p[0].to(p[1])):
        ins = [t * 1 for t in leaves]
        ins[1] = torch.cat([ins[1], ins[1]], 2)[..., :64]                    # (read in place, rows 128 apart)
        ins[2] = ins[2].transpose(1, 2).contiguous().transpose(1, 2)        # (a copy is made)
        out = pkg.packed_attention(*ins, cu, bias=bias)
    del ins
    gc.collect()
    assert len(kept) == 5 and all(r() is None for r in kept), [i for i, r in enumerate(kept) if r() is not None]
    with torch.no_grad():
        out.data.zero_()                                                     # (the packed output is another tensor)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves + extra, do), want))


def test_recomputed_in_the_backward(dev):
    """under non-reentrant checkpointing: the same gradients"""
    from torch.utils.checkpoint import checkpoint

    import e2_tts_pytorch_amd as pkg
    q, k, v, do, cu = attn_inputs(dev)
    bias = pkg.RelativePositionBias(2, 8, 16).to(dev)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)] + [bias.weight]
    f = lambda q, k, v: pkg.packed_attention(q, k, v, cu, bias=bias, causal=True)  # noqa: E731
    want = torch.autograd.grad(f(*leaves[:3]), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(checkpoint(f, *leaves[:3], use_reentrant=False), leaves, do), want))


def test_layer_norm_of_views(dev):
    """transposed, expanded and column-strided inputs of two and three dimensions, an input gradient that is one of them: as the contiguous copy"""
    import e2_tts_pytorch_amd as pkg
    g = torch.Generator().manual_seed(1)
    gam, bet = (torch.randn(8, generator=g).to(dev) for _ in range(2))
    base = torch.randn(8, 6, 8, generator=g).to(dev)
    for make in (lambda b: b[0, :6, :6].t().contiguous().t()[:, :6], lambda b: b[:, 0].t(), lambda b: b[0, :1].expand(5, 8), lambda b: b[:, :, ::2], lambda b: b[0, :, ::2],
                 lambda b: b.transpose(0, 2), lambda b: b[0, 0], lambda b: b[0, 0].expand(2, 3, 8), lambda b: b[0, 0, :1].expand(8), lambda b: b[:0, 0].expand(0, 8)):
        for dt in (f32, bf16):
            x = make(base.to(dt))
            D = x.shape[-1]
            dy = make(torch.randn(8, 6, 8, generator=torch.Generator().manual_seed(2)).to(dev).to(dt))
            outs = []
            for xi, dyi in ((x, dy), (x.contiguous(), dy.contiguous())):
                xi = xi.detach().requires_grad_()
                w, b = gam[:D].clone().requires_grad_(), bet[:D].clone().requires_grad_()
                y = pkg.layer_norm(xi, w, b)
                outs.append([y, *torch.autograd.grad(y, [xi, w, b], dyi)])
            assert outs[0][0].shape == x.shape and outs[0][1].shape == x.shape
            assert all(torch.equal(s, t) for s, t in zip(*outs)), (tuple(x.shape), x.stride(), dt)
