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
