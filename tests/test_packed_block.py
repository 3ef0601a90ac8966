"""Layer norm, packed attention with a learned distance bias, and the single-token form, used together as a block uses them."""
import pytest
import torch
import torch.nn.functional as F

from conftest import gpu_shapes
from test_packed_attn import offsets

bf16, f32, f64 = torch.bfloat16, torch.float32, torch.float64


class Block(torch.nn.Module):
    """x + W_o attention(W_qkv norm(x)) over packed rows, grouped key heads"""

    def __init__(self, dim=128, heads=2, kv_heads=1):
        super().__init__()
        import e2_tts_pytorch_amd as pkg
        self.heads, self.kv = heads, kv_heads
        self.norm = pkg.LayerNorm(dim)
        self.bias = pkg.RelativePositionBias(heads, num_buckets=8, max_distance=20)
        self.qkv = torch.nn.Parameter(torch.randn((heads + 2 * kv_heads) * 64, dim) * dim ** -0.5)
        self.out = torch.nn.Parameter(torch.randn(dim, heads * 64) * (heads * 64) ** -0.5)
        with torch.no_grad():
            self.norm.weight.normal_(1., 0.2)
            self.norm.bias.normal_(0., 0.2)
            self.bias.weight.normal_()

    def project(self, x):
        y = F.linear(self.norm(x), self.qkv.to(x.dtype)).view(-1, self.heads + 2 * self.kv, 64)
        return y.split([self.heads, self.kv, self.kv], 1)

    def forward(self, x, cu, **kw):
        import e2_tts_pytorch_amd as pkg
        q, k, v = self.project(x)
        o = pkg.packed_attention(q, k, v, cu, softcap=30., bias=self.bias, **kw)
        return x + F.linear(o.flatten(1), self.out.to(x.dtype))

    def exact(self, x, lens, causal, prefix):
        """the same block in 64 bits, from the definitions"""
        y = F.layer_norm(x, x.shape[-1:], self.norm.weight.to(f64), self.norm.bias.to(f64), 1e-5)
        q, k, v = F.linear(y, self.qkv.to(f64)).view(-1, self.heads + 2 * self.kv, 64).split([self.heads, self.kv, self.kv], 1)
        outs, at = [], 0
        for n, p in zip(lens, prefix):
            Q, K, V = (t[at:at + n].transpose(0, 1) for t in (q, k, v))
            at += n
            K, V = (t.repeat_interleave(self.heads // self.kv, 0) for t in (K, V))
            z = 30. * torch.tanh(Q @ K.transpose(1, 2) / 8 / 30.) + self.bias(n, n).to(f64)
            if causal:
                i, j = torch.arange(n)[:, None], torch.arange(n)[None]
                z = z.masked_fill((j > i) & (j >= p), -torch.inf)
            outs.append((z.softmax(-1) @ V).transpose(0, 1))
        return x + F.linear(torch.cat(outs).flatten(1), self.out.to(f64))


@pytest.mark.parametrize('causal', [False, True], ids=['full', 'prefix'])
def test_block_forward_and_gradients(dev, causal):
    torch.manual_seed(0)
    lens, prefix = ([300, 41, 130], [50, 41, 0]) if gpu_shapes(dev) else ([40, 9, 23], [10, 9, 0])
    blk = Block()
    for p in blk.parameters():
        p.data = p.data.to(bf16).to(f32)                         # what the products round to anyway
    x0, dy = torch.randn(sum(lens), 128).to(bf16), torch.randn(sum(lens), 128).to(bf16)
    x64 = x0.to(f64).requires_grad_()
    y64 = blk.exact(x64, lens, causal, prefix)
    names = [n for n, _ in blk.named_parameters()]
    want = torch.autograd.grad(y64, [x64] + list(blk.parameters()), dy.to(f64))
    blk = blk.to(dev)
    x = x0.to(dev).requires_grad_()
    kw = dict(max_q=max(lens), causal=causal)
    if causal:
        kw['prefix'] = torch.tensor(prefix, dtype=torch.int32, device=dev)
    y = blk(x, offsets(lens, dev), **kw)
    got = torch.autograd.grad(y, [x] + list(blk.parameters()), dy.to(dev))
    # bf16 roundings between x and y: norm, projection, probabilities, attention, product, sum: six, each at most 2^-8 of its tensor (in norm the
    # random signs make it about a third of that); the way back has as many again plus dS and the gradients of q, k, v
    rel = lambda a, b: ((a.detach().cpu().to(f64) - b.detach()).norm() / b.detach().norm()).item()  # noqa: E731
    assert rel(y, y64) < 6 * 2. ** -8
    for n, a, b in zip(['x'] + names, got, want):
        assert rel(a, b) < 14 * 2. ** -8, (n, rel(a, b))


def test_block_token_by_token(dev):
    """a causal pass over a document and the same document decoded token by token from a cache agree to their roundings"""
    import e2_tts_pytorch_amd as pkg
    torch.manual_seed(1)
    n = 70 if gpu_shapes(dev) else 37
    blk = Block(heads=4, kv_heads=2).to(dev)
    x = torch.randn(n, 128).to(bf16).to(dev)
    with torch.no_grad():
        q, k, v = blk.project(x)
        full = pkg.packed_attention(q, k, v, offsets([n], dev), causal=True, softcap=30., bias=blk.bias)
        kc, vc = (torch.zeros(1, 80, 2, 64, dtype=bf16, device=dev) for _ in range(2))
        for i in range(n):
            kc[:, i], vc[:, i] = k[i], v[i]
            one = pkg.attn_decode(q[i:i + 1].contiguous(), kc, vc, torch.tensor([i + 1], dtype=torch.int32, device=dev), softcap=30., bias=blk.bias)
            # both round probabilities (2^-8 each) and output (2^-8) of the same fp32 scores; |o| <= max |v|
            lim = 2 * 2. ** -8 * (one[0].abs() + v[:i + 1].abs().amax()) + 1e-6
            assert ((one[0].float() - full[i].float()).abs() <= lim.float()).all(), i


def test_autograd_forms(dev):
    """which gradients are asked for, an input changed in place, a second backward, refusals"""
    import e2_tts_pytorch_amd as pkg
    from e2_tts_pytorch_amd import ops
    torch.manual_seed(2)
    cu = offsets([20, 13], dev)
    bias = pkg.RelativePositionBias(2, 8, 16).to(dev)
    q, k, v = (torch.randn(33, 2, 64).to(bf16).to(dev).requires_grad_() for _ in range(3))
    out = pkg.packed_attention(q, k, v, cu, bias=bias)
    g = torch.randn(33, 2, 64).to(bf16).to(dev)
    a = torch.autograd.grad(out, [q, k, v, bias.weight], g, retain_graph=True)
    b = torch.autograd.grad(out, [q, k, v, bias.weight], g)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    bias.weight.requires_grad_(False)                                                 # a frozen table: the other gradients, to their rounding
    c = torch.autograd.grad(pkg.packed_attention(q, k, v, cu, bias=bias), [q, k, v], g)
    assert all((s.float() - t.float()).norm() < 0.02 * s.float().norm() for s, t in zip(a[:3], c))
    only = torch.autograd.grad(pkg.packed_attention(q.detach(), k, v.detach(), cu, bias=bias), [k], g)
    assert torch.equal(only[0], c[1])
    k2 = k.detach().clone().requires_grad_()
    w = k2 * 1
    out = pkg.packed_attention(q, w, v, cu)
    w.mul_(2)
    with pytest.raises(RuntimeError):
        out.sum().backward()
    with pytest.raises(ops.E2KError):
        pkg.packed_attention(q, k, v, cu, slopes=torch.ones(2, device=dev, requires_grad=True))
    with torch.no_grad():
        assert not pkg.packed_attention(q, k, v, cu, bias=bias).requires_grad
    ln = pkg.LayerNorm(64).to(dev)
    with pytest.raises(ops.E2KError):
        ln(torch.zeros(2, 32, dtype=bf16, device=dev))
    x = torch.randn(3, 5, 64, device=dev, requires_grad=True)
    gam, bet = (torch.randn(4, 64, device=dev, requires_grad=True) for _ in range(2))
    y = pkg.layer_norm(x, gam, bet, 1., 5)                                            # one more row of scale / shift than batch elements
    dx, dg, db = torch.autograd.grad(y.sum(), [x, gam, bet])
    assert dx.shape == x.shape and dg.shape == (4, 64) and (dg[3] == 0).all() and (db[:3] == 5).all() and (db[3] == 0).all()
    ref = torch.nn.LayerNorm(64).to(dev)
    ref.load_state_dict(ln.state_dict())
    assert (ln(x) - ref(x)).abs().max() < 1e-5


@pytest.mark.gpu
def test_captured_and_replayed():
    """two captured graphs (a training pass, a decode step) replayed in turn with eager work between, against the eager results; both on a stream
    other than the one that made their inputs"""
    import e2_tts_pytorch_amd as pkg
    from e2_tts_pytorch_amd import _lib, ops
    from emu.install import install
    install(None, False)
    _lib.get()
    torch.manual_seed(3)
    lens = [200, 333, 65]
    cu = offsets(lens, 'cuda')
    bias = pkg.RelativePositionBias(4, 32, 128).cuda()
    T = sum(lens)
    x = torch.randn(T, 256, device='cuda').to(bf16)
    q, k, v, g = (torch.randn(T, 4, 64, device='cuda').to(bf16) for _ in range(4))
    kc, vc = (torch.randn(3, 2000, 4, 64, device='cuda').to(bf16) for _ in range(2))
    n = torch.tensor([2000, 1, 777], dtype=torch.int32, device='cuda')
    w = torch.randn(256, device='cuda')

    def train():
        out, st = ops.packed_attn_fwd(q, k, v, cu, train=True, table=bias.weight.detach(), buckets=bias.buckets, max_q=333)
        y, m, r = ops.layernorm_fwd(x, w, w)
        return [out, *ops.packed_attn_bwd(st, g), y, *ops.layernorm_bwd(x, x, m, r, w)]

    def step():
        return [ops.attn_decode(q[:3], kc, vc, n, table=bias.weight.detach(), buckets=bias.buckets)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for f in (train, step):
            f()
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                res = f()
            graphs.append((gr, res, f))
    for i in range(4):
        q.normal_()
        k.normal_()
        kc.normal_()
        n[1] = 50 * i + 1
        torch.cuda.synchronize()
        eager = [[t.clone() for t in f()] for _, _, f in graphs]
        for gr, _, _ in graphs:
            gr.replay()
        junk = [torch.full((1 << 20,), float('nan'), device='cuda') for _ in range(4)]
        del junk
        for gr, _, _ in reversed(graphs):
            gr.replay()
        torch.cuda.synchronize()
        for (_, res, _), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(res, want)), i


@pytest.mark.gpu
def test_recorded_in_a_launch_plan():
    """the entry points record into a launch plan like every compute call and replay to the same bits"""
    from e2_tts_pytorch_amd import _lib, ops
    from emu.install import install
    install(None, False)
    L = _lib.get()
    torch.manual_seed(4)
    q, k, v = (torch.randn(150, 2, 64, device='cuda').to(bf16) for _ in range(3))
    cu = offsets([100, 50], 'cuda')
    x = torch.randn(64, 256, device='cuda')
    want = ops.packed_attn_fwd(q, k, v, cu), ops.layernorm_fwd(x, None, None)[0]
    ops.begin_recording()
    out, y = ops.packed_attn_fwd(q, k, v, cu), ops.layernorm_fwd(x, None, None)[0]
    assert ops.recorded() == 2
    h = ops.end_recording()
    out.zero_(), y.zero_()
    ops.run_plan(h, 0, 2, q.device)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(y, want[1])
    L.e2k_plan_free(h)


@pytest.mark.gpu
def test_two_streams_and_next_to_lds_dma_gemms():
    """the kernels on two streams at once, beside a third that runs LDS-DMA GEMMs: the bits of the same calls alone, every time"""
    from e2_tts_pytorch_amd import _lib, ops
    from emu.install import install
    install(None, False)
    _lib.get()
    torch.manual_seed(5)
    T, H = 1500, 8
    cu = offsets([700, 96, 704], 'cuda')
    buckets = ops.rel_buckets(32, 128, device='cuda')
    table, slopes = torch.randn(32, H, device='cuda'), torch.rand(H, device='cuda')
    q, k, v, g = (torch.randn(T, H, 64, device='cuda').to(bf16) for _ in range(4))
    kc, vc = (torch.randn(4, 3000, H, 64, device='cuda').to(bf16) for _ in range(2))
    n = torch.tensor([3000, 10, 1111, 2222], dtype=torch.int32, device='cuda')
    x, w = torch.randn(T, 1024, device='cuda').to(bf16), torch.randn(1024, device='cuda')

    def first():
        out, st = ops.packed_attn_fwd(q, k, v, cu, train=True, table=table, buckets=buckets, softcap=30.)
        y, m, r = ops.layernorm_fwd(x, w, w)
        return [out, *ops.packed_attn_bwd(st, g), y, *ops.layernorm_bwd(x, x, m, r, w)]

    def second():
        out, st = ops.packed_attn_fwd(q, k[:, ::4], v[:, ::4], cu, train=True, causal=True, slopes=slopes)
        return [out, *ops.packed_attn_bwd(st, g)[:3], ops.packed_attn_fwd(q[:40], k, v, cu.new_tensor([0, 40]), cu.new_tensor([0, T])),
                ops.attn_decode(q[:4], kc, vc, n, slopes=slopes)]

    want = first(), second()
    a, b = torch.randn(4096, 1024, device='cuda').to(bf16), torch.randn(4096, 1024, device='cuda').to(bf16)
    torch.cuda.synchronize()
    s1, s2, s3 = (torch.cuda.Stream() for _ in range(3))
    bad = 0
    for _ in range(30):
        got = [[], []]
        for _ in range(3):
            with torch.cuda.stream(s3):
                for _ in range(6):
                    ops.gemm_nt(a, b)
            for s, f, o in ((s1, first, got[0]), (s2, second, got[1])):
                with torch.cuda.stream(s):
                    o.append(f())
        torch.cuda.synchronize()
        for res, ref in zip(got, want):
            bad += sum(not torch.equal(t, u) for one in res for t, u in zip(one, ref))
    assert bad == 0, bad


@pytest.mark.gpu
def test_autograd_captured():
    """forward and torch.autograd.grad of the block in one captured graph, replayed on changed inputs"""
    from e2_tts_pytorch_amd import _lib
    from emu.install import install
    install(None, False)
    _lib.get()
    torch.manual_seed(6)
    lens = [150, 70]
    cu = offsets(lens, 'cuda')
    blk = Block(heads=4, kv_heads=2).cuda()
    ps = list(blk.parameters())
    x = torch.randn(sum(lens), 128, device='cuda').to(bf16).requires_grad_()
    dy = torch.randn(sum(lens), 128, device='cuda').to(bf16)

    def f():
        y = blk(x, cu, max_q=150, causal=True)
        return [y.detach(), *torch.autograd.grad(y, [x] + ps, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            f()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        res = f()
    for i in range(3):
        with torch.no_grad():
            x.normal_()
            dy.normal_()
        want = f()
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        # (the projections' library products may take another kernel inside the graph: bf16 roundings of the same values)
        for a, b in zip(res, want):
            assert (a.float() - b.float()).norm() <= 0.02 * b.float().norm(), i
