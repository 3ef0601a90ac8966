"""Layer norm kernels (csrc/layernorm.hip) against the definition in 64 bits."""
import pytest
import torch

from conftest import gpu_shapes

bf16, f32, f64 = torch.bfloat16, torch.float32, torch.float64
U32 = 2. ** -24                     # half a step of fp32, relative


def inputs(M, D, nb, dt, seed=0, shift=1., affine=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, D, generator=g) + shift * torch.randn(M, 1, generator=g)).to(dt)
    dy = torch.randn(M, D, generator=g).to(dt)
    gamma = torch.randn(nb, D, generator=g) * 0.3 if affine else None
    beta = torch.randn(nb, D, generator=g) * 0.3 if affine else None
    return x, dy, gamma, beta


def exact(x, dy, gamma, beta, off, rpb, eps):
    M, D = x.shape
    nb = -(-M // rpb)
    x = x.to(f64).requires_grad_()
    w = torch.zeros(nb, D, dtype=f64) + (1. - off) if gamma is None else gamma[:nb].to(f64)
    b = torch.zeros(nb, D, dtype=f64) if beta is None else beta[:nb].to(f64)
    w.requires_grad_(), b.requires_grad_()
    row = torch.arange(M) // rpb
    m = x.mean(1, keepdim=True)
    xc = x - m
    r = (xc.square().mean(1, keepdim=True) + eps).rsqrt()
    y = xc * r * (w[row] + off) + b[row]
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy.to(f64))
    return y.detach(), dx, dw, db, m.detach(), r.detach(), (xc * r).detach()


def out_half_step(dt):
    return torch.finfo(dt).eps / 2


def check(dev, M, D, nb=1, dt=bf16, off=0., eps=1e-5, shift=1., affine=True, pad=0, accumulate=False):
    from e2_tts_pytorch_amd import ops
    rpb = -(-M // nb)
    x, dy, gamma, beta = inputs(M, D, nb, dt, seed=M * 131 + D, shift=shift, affine=affine)
    y64, dx64, dw64, db64, m64, r64, xh64 = exact(x, dy, gamma, beta, off, rpb, eps)
    xd = torch.full((M, D + pad), float('nan'), dtype=dt, device=dev)[:, :D]
    xd.copy_(x)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y, mean, rstd = ops.layernorm_fwd(xd, to(gamma), to(beta), off, rpb, eps=eps)
    d0 = torch.randn(2, nb, D) if accumulate else None
    dg, db = (d0.clone().to(dev).unbind(0)) if accumulate else (None, None)
    dx, dg, db = ops.layernorm_bwd(to(dy), xd, mean, rstd, to(gamma), off, rpb, dg, db)
    assert y.dtype == dt and dx.dtype == dt and dg.shape == (nb, D) and y.is_contiguous()
    # fp32 error of xh: the mean of D terms and x - mean are off by a few half steps of |x|, the mean's sum by log-depth times that; relative to 1 / r.
    # 24 half steps cover the lane-serial part of the sums (at most 32 terms a lane, then 6 + 2 levels).  The square sum adds the same relative to xh
    n = 24 * U32
    exh = n * (x.to(f64).abs().amax(1, keepdim=True) * r64 + xh64.abs() + 1)
    row = torch.arange(M) // rpb
    w = (torch.ones(nb, D, dtype=f64) if gamma is None else gamma.to(f64) + off)[row]
    b = (torch.zeros(nb, D, dtype=f64) if beta is None else beta.to(f64))[row]
    ey = exh * w.abs() + 4 * U32 * ((xh64 * w).abs() + b.abs())
    h = out_half_step(dt)
    bound = y64.abs() * h + (1 + h) * ey
    assert ((y.cpu().to(f64) - y64).abs() <= bound).all(), ((y.cpu().to(f64) - y64).abs() / bound).max()
    # dx = r (g - c1 - xh c2): errors of xh enter through c2 (|c2| <= max |g| max |xh|) and through the product xh c2
    g = dy.to(f64) * w
    c2 = (g * xh64).mean(1, keepdim=True)
    gm, xm = g.abs().amax(1, keepdim=True), xh64.abs().amax(1, keepdim=True)
    em = exh.amax(1, keepdim=True)
    edx = r64 * (n * (g.abs() + gm + xh64.abs() * gm * xm + (xh64 * c2).abs()) + em * c2.abs() + xh64.abs() * (g.abs().mean(1, keepdim=True) * em))
    bound = dx64.abs() * h + (1 + h) * edx * 2
    assert ((dx.cpu().to(f64) - dx64).abs() <= bound).all(), ((dx.cpu().to(f64) - dx64).abs() / bound).max()
    # column sums: rpb terms; any fixed order is off by at most (number of additions on a term's path) half steps of the sum of magnitudes
    add = U32 * (rpb / 8 + 32)
    for got, want, mag, err in ((dg, dw64, (dy.to(f64) * xh64).abs(), dy.to(f64).abs() * exh), (db, db64, dy.to(f64).abs(), 0 * exh.expand(M, D))):
        lim = torch.zeros(nb, D, dtype=f64).index_add_(0, row, mag * add + err) + 1e-30
        start = 0. if d0 is None else (d0[0] if got is dg else d0[1]).to(f64)
        lim = lim + (0 if d0 is None else 2 * U32 * (start.abs() + want.abs()))
        assert ((got.cpu().to(f64) - want - start).abs() <= lim).all(), ((got.cpu().to(f64) - want - start).abs() / lim).max()


@pytest.mark.parametrize('dt', [bf16, f32], ids=['bf16', 'f32'])
@pytest.mark.parametrize('M,D', [(1, 1), (3, 7), (9, 64), (5, 512), (17, 1003), (12, 1024), (4, 1600), (5, 2048), (3, 2056), (3, 4099), (2, 8192)])
def test_layer_norm(dev, M, D, dt):
    check(dev, M, D, dt=dt)


@pytest.mark.parametrize('dt', [bf16, f32], ids=['bf16', 'f32'])
def test_layer_norm_per_batch_element(dev, dt):
    check(dev, 12, 256, nb=4, dt=dt, off=1.)
    check(dev, 11, 100, nb=3, dt=dt, off=1., accumulate=True)         # a short last batch element


def test_layer_norm_forms(dev):
    check(dev, 6, 128, affine=False)
    check(dev, 6, 96, dt=f32, affine=False, accumulate=True)
    check(dev, 7, 64, pad=8)                                            # row stride wider than the row, still 16-byte rows
    check(dev, 7, 64, pad=3)                                            # ... and not
    check(dev, 6, 512, dt=f32, shift=300.)                              # a mean far from 0: the centred squares do not cancel
    check(dev, 5, 33, dt=f32, shift=0., eps=0.1)


def test_layer_norm_constant_rows(dev):
    """variance 0: y = beta exactly, and a finite gradient through eps"""
    from e2_tts_pytorch_amd import ops
    x = torch.full((3, 256), 2.5, dtype=bf16, device=dev)
    beta = torch.randn(1, 256).to(dev)
    y, mean, rstd = ops.layernorm_fwd(x, None, beta)
    assert torch.equal(y.cpu(), beta.cpu().to(bf16).expand(3, 256)) and torch.equal(mean.cpu(), torch.full((3,), 2.5))
    dx, _, _ = ops.layernorm_bwd(torch.randn(3, 256).to(dev).to(bf16), x, mean, rstd, None)
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize('M,D,nb,dt', [(8448, 1024, 8, bf16), (4099, 1003, 1, f32), (2000, 2048, 1, bf16), (700, 6144, 7, f32), (300, 600, 300, bf16)])
def test_layer_norm_large(M, D, nb, dt):
    check('cuda', M, D, nb=nb, dt=dt, off=1.)


def test_layer_norm_same_bits(dev):
    from e2_tts_pytorch_amd import ops
    M, D = (5000, 1024) if gpu_shapes(dev) else (40, 200)
    x, dy, gamma, beta = (t.to(dev) for t in inputs(M, D, 1, bf16))
    y, m, r = ops.layernorm_fwd(x, gamma, beta)
    a = ops.layernorm_bwd(dy, x, m, r, gamma)
    b = ops.layernorm_bwd(dy, x, m, r, gamma)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_layer_norm_gradient_against_differences(emu):
    """the fp32 kernels' gradient against central differences of their own forward"""
    from e2_tts_pytorch_amd import ops
    x, dy, gamma, beta = inputs(2, 10, 1, f32, seed=3)
    loss = lambda x, g, b: (ops.layernorm_fwd(x, g, b)[0].to(f64) * dy.to(f64)).sum().item()  # noqa: E731
    y, m, r = ops.layernorm_fwd(x, gamma, beta)
    dx, dg, db = ops.layernorm_bwd(dy, x, m, r, gamma)
    h = 2. ** -7           # truncation h^2 / 6 f''' ~ 1e-5 |f'''|, rounding 24 * 2^-24 * |loss| / h ~ 2e-4: 5e-3 covers both
    for t, grad, i in ((x, dx, (1, 4)), (x, dx, (0, 9)), (gamma, dg, (0, 2)), (beta, db, (0, 7))):
        old = t[i].item()
        t[i] = old + h
        up = loss(x, gamma, beta)
        t[i] = old - h
        down = loss(x, gamma, beta)
        t[i] = old
        assert abs((up - down) / (2 * h) - grad[i].item()) < 5e-3


def test_layer_norm_empty(dev):
    from e2_tts_pytorch_amd import ops
    x = torch.zeros(0, 64, dtype=bf16, device=dev)
    y, m, r = ops.layernorm_fwd(x, None, None)
    dx, dg, db = ops.layernorm_bwd(x, x, m, r, None)
    assert y.shape == (0, 64) and dx.shape == (0, 64)


def test_layer_norm_refusals(emu):
    from e2_tts_pytorch_amd import ops
    x = torch.zeros(4, 64, dtype=bf16)
    w = torch.ones(1, 64)
    bad = [lambda: ops.layernorm_fwd(x.half(), w, w), lambda: ops.layernorm_fwd(x[0], w, w), lambda: ops.layernorm_fwd(x.t(), w, w),
           lambda: ops.layernorm_fwd(torch.zeros(2, 8193, dtype=bf16), None, None), lambda: ops.layernorm_fwd(x, torch.ones(1, 63), w),
           lambda: ops.layernorm_fwd(x, w.to(bf16), w), lambda: ops.layernorm_fwd(x, w, w, 0., 2), lambda: ops.layernorm_fwd(x, w, w, eps=-1.),
           lambda: ops.layernorm_fwd(x, w, w, eps=float('nan')), lambda: ops.layernorm_fwd(x.expand(4, 64)[:1].expand(4, 64), w, w)]
    y, m, r = ops.layernorm_fwd(x, w, w)
    bad += [lambda: ops.layernorm_bwd(x.float(), x, m, r, w), lambda: ops.layernorm_bwd(x[:2], x, m, r, w), lambda: ops.layernorm_bwd(x, x, m[:2], r, w),
            lambda: ops.layernorm_bwd(x, x, m, r, w, 0., 0, torch.zeros(1, 64)), lambda: ops.layernorm_bwd(x, x, m, r, w, 0., 0, torch.zeros(1, 64), torch.zeros(1, 32)),
            lambda: ops.layernorm_bwd(x, x, m, r, w, 0., 0, torch.zeros(1, 64), torch.zeros(1, 64), need_weights=False)]
    for i, f in enumerate(bad):
        with pytest.raises(ops.E2KError):
            f()
            print('not refused:', i)


def test_layer_norm_broadcast_columns(dev):
    """scale and shift expanded over the batch elements, or with strides of their own, are read as they stand"""
    from e2_tts_pytorch_amd import ops
    x, dy, gamma, beta = (t.to(dev) for t in inputs(8, 96, 1, f32))
    want = ops.layernorm_fwd(x, gamma, beta, 1., 0)[0]
    wide = torch.zeros(4, 200, device=dev)
    wide[:, :96] = beta
    assert torch.equal(ops.layernorm_fwd(x, gamma.expand(4, 96), wide[:, :96], 1., 2)[0], want)
    y, m, r = ops.layernorm_fwd(x, gamma.expand(4, 96), beta.expand(4, 96), 1., 2)
    assert torch.equal(y, want)
    dx, dg, db = ops.layernorm_bwd(dy, x, m, r, gamma.expand(4, 96), 1., 2)
    one = ops.layernorm_bwd(dy, x, m, r, gamma, 1., 0)
    assert torch.equal(dx, one[0]) and (dg.sum(0) - one[1][0]).abs().max() < 1e-4
    with pytest.raises(ops.E2KError):
        ops.layernorm_bwd(dy, x, m, r, gamma, 1., 2, torch.zeros(1, 96, device=dev).expand(4, 96), torch.zeros(1, 96, device=dev).expand(4, 96))
