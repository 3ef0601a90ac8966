"""Attention over packed documents (csrc/packed_attn.hip) against the definition in 64 bits."""
import math

import pytest
import torch

from conftest import gpu_shapes

bf16, f32, f64 = torch.bfloat16, torch.float32, torch.float64
HALF = 2. ** -8                       # half a step of bf16, relative
U = 2. ** -24                         # half a step of fp32, relative


@pytest.fixture(params=[0, 1], ids=['dma_early', 'dma_late'])
def landing(request, dev, monkeypatch):
    """the kernels stage their tiles with LDS-DMA into a two-stage ring: on the host model both landing extremes (at issue / at the counted wait)"""
    if dev == 'cuda' and request.param:
        pytest.skip('LDS-DMA landing extremes exist on the host model only')
    monkeypatch.setenv('E2K_EMU_GLDS_LATE', str(request.param))
    return request.param


def offsets(lens, dev='cpu'):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


class Case:
    """inputs of one call, on the CPU; ql / kl: rows of each document's slot, nq / nk: how many of them count"""

    def __init__(self, ql, kl=None, H=2, Hkv=None, nq=None, nk=None, mask='full', prefix=None, cap=0., bias='none', buckets=8, reach=24, scale=None, gain=1.5, seed=0,
                 tail=0, causal_map=None):
        g = torch.Generator().manual_seed(seed)
        self.ql, self.kl = ql, kl or ql
        self.nq, self.nk = nq or self.ql, nk or self.kl
        self.H, self.Hkv, self.mask, self.cap, self.bias, self.tail = H, Hkv or H, mask, cap, bias, tail
        self.prefix = prefix if mask == 'prefix' else None
        self.scale = scale or 0.125
        Tq, Tk = sum(self.ql) + tail, sum(self.kl) + tail
        self.q = (torch.randn(Tq, H, 64, generator=g) * gain).to(bf16)
        self.k = torch.randn(Tk, self.Hkv, 64, generator=g).to(bf16)
        self.v = torch.randn(Tk, self.Hkv, 64, generator=g).to(bf16)
        self.dout = torch.randn(Tq, H, 64, generator=g).to(bf16)
        self.slopes = torch.tensor([0.5 ** (i + 1) for i in range(H)]) if bias == 'alibi' else None
        self.table = torch.randn(buckets, H, generator=g) if bias == 'table' else None
        self.reach = reach
        if bias == 'table':
            from e2_tts_pytorch_amd import ops
            self.map = ops.rel_buckets(buckets, reach, causal=mask == 'causal' if causal_map is None else causal_map)
        else:
            self.map = None

    def args(self, dev):
        to = lambda t: None if t is None else t.to(dev)  # noqa: E731
        kw = dict(causal=self.mask != 'full', scale=self.scale, softcap=self.cap, slopes=to(self.slopes), table=to(self.table), buckets=to(self.map))
        if self.nq != self.ql:
            kw['len_q'] = torch.tensor(self.nq, dtype=torch.int32, device=dev)
        if self.nk != self.kl:
            kw['len_k'] = torch.tensor(self.nk, dtype=torch.int32, device=dev)
        if self.prefix is not None:
            kw['prefix'] = torch.tensor(self.prefix, dtype=torch.int32, device=dev)
        return [to(self.q), to(self.k), to(self.v), offsets(self.ql, dev), offsets(self.kl, dev)], kw

    def exact(self):
        """definition in 64 bits with, beside each result, the sum of magnitudes that its error bound is a multiple of"""
        H, G = self.H, self.H // self.Hkv
        q, k, v, do = (t.to(f64) for t in (self.q, self.k, self.v, self.dout))
        r = dict(out=torch.zeros_like(q), dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        b = {n: torch.zeros_like(t) for n, t in r.items()}
        if self.table is not None:
            r['dtable'], b['dtable'] = torch.zeros(self.table.shape, dtype=f64), torch.zeros(self.table.shape, dtype=f64)
        qs, ks = offsets(self.ql).tolist(), offsets(self.kl).tolist()
        for d, (nq, nk) in enumerate(zip(self.nq, self.nk)):
            if not nq or not nk:
                continue
            A, B = slice(qs[d], qs[d] + nq), slice(ks[d], ks[d] + nk)
            pos, at = torch.arange(nq)[:, None] + nk - nq, torch.arange(nk)[None]
            see = torch.ones(nq, nk, dtype=torch.bool) if self.mask == 'full' else at <= pos
            if self.prefix is not None:
                see = see | (at < self.prefix[d])
            rel = at - pos
            for h in range(H):
                Q, K, V, dO = q[A, h], k[B, h // G], v[B, h // G], do[A, h]
                z = Q @ K.t() * self.scale
                mag = Q.abs() @ K.abs().t() * self.scale
                th = torch.tanh(z / self.cap) if self.cap else torch.zeros_like(z)
                t = self.cap * th if self.cap else z
                bias = torch.zeros_like(t)
                if self.slopes is not None:
                    bias = -self.slopes[h].to(f64) * rel.abs()
                if self.table is not None:
                    bias = self.table[:, h].to(f64)[self.map.long()[rel.clamp(-self.reach, self.reach) + self.reach]]
                seen = see & (bias > -1e30)                   # (a bias that hides is a mask: such a pair has no score, and no error of one)
                bias = torch.where(seen, bias, torch.zeros_like(bias))
                t = torch.where(seen, t + bias, torch.tensor(-math.inf, dtype=f64))
                top = t.amax(1, keepdim=True)
                e = torch.where(top > -math.inf, torch.exp(t - torch.where(top > -math.inf, top, torch.zeros_like(top))), torch.zeros_like(t))
                l = e.sum(1, keepdim=True)
                p = torch.where(l > 0, e / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(e))
                # error of a score in fp32: 64 products (64 half steps of their magnitudes), the tanh (2^-22 of the cap: one exp2, one reciprocal, one
                # subtraction from 1), the bias and the reference point (8 half steps of everything that is added up)
                et = 64 * U * mag + 4 * U * self.cap + 8 * U * (t.abs().nan_to_num(posinf=0.) + bias.abs() + top.abs().nan_to_num(posinf=0.) + 10)
                et = torch.where(seen, et, torch.zeros_like(et))
                ep = et + (p * et).sum(1, keepdim=True) + 16 * U               # of a probability, relative (its own score, the row's sum)
                o = p @ V
                r['out'][A, h] = o
                # out: rounded once (HALF of itself), its probabilities rounded to bf16 (HALF each) and off by ep
                b['out'][A, h] = HALF * o.abs() + (p * (HALF + ep)) @ V.abs()
                dP = dO @ V.t()
                mdP = dO.abs() @ V.abs().t()
                dl = (dO * o).sum(1, keepdim=True)
                edl = (dO.abs() * b['out'][A, h]).sum(1, keepdim=True)           # dO.o is taken from the output as the forward left it
                ds = p * (dP - dl)
                eds = p * (ep * (dP - dl).abs() + 64 * U * (mdP + dl.abs()) + edl)
                cap1 = 1 - th * th
                dz, edz = ds * cap1 * self.scale, (eds * cap1 + ds.abs() * (4 * U + 2 * et / self.cap if self.cap else 4 * U)) * self.scale
                r['dq'][A, h] = dz @ K
                b['dq'][A, h] = HALF * r['dq'][A, h].abs() + (HALF * dz.abs() + edz) @ K.abs()
                r['dk'][B, h // G] += dz.t() @ Q
                b['dk'][B, h // G] += (HALF * dz.abs() + edz).t() @ Q.abs()
                r['dv'][B, h // G] += p.t() @ dO
                b['dv'][B, h // G] += (p * (HALF + ep)).t() @ dO.abs()
                if self.table is not None:
                    # the table's gradient: dO.o is good to 2^-16 of its terms or better (three-term probabilities, fp32 remainder of the output); fp32 sums over the document's pairs
                    edl = ((dO.abs() * ((p * (2. ** -16 + ep)) @ V.abs() + 2. ** -16 * o.abs())).sum(1, keepdim=True))
                    eds = p * (ep * (dP - dl).abs() + 64 * U * (mdP + dl.abs()) + edl) + 64 * U * ds.abs()
                    where = self.map.long()[rel.clamp(-self.reach, self.reach) + self.reach]
                    r['dtable'][:, h].index_add_(0, where.flatten(), ds.flatten())
                    b['dtable'][:, h].index_add_(0, where.flatten(), eds.flatten())
        for n in ('dk', 'dv'):
            b[n] += HALF * r[n].abs()
        return r, b


def held(got, want, bound, what):
    got = got.detach().cpu().to(f64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    # (a quotient of 0 / 0 where a row is exactly zero on both sides)
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    bad = off > bound * 1.001 + 1e-37
    assert not bad.any(), (what, int(bad.sum()), (off / bound.clamp_min(1e-37)).max().item())


def run(c, dev, train=True, **more):
    from e2_tts_pytorch_amd import ops
    a, kw = c.args(dev)
    kw.update(more)
    out, st = ops.packed_attn_fwd(*a, train=True, **kw)
    dq, dk, dv, dtable = ops.packed_attn_bwd(st, c.dout.to(dev))
    got = dict(out=out, dq=dq, dk=dk, dv=dv)
    if dtable is not None:
        got['dtable'] = dtable
    return got


def check(c, dev, **more):
    got = run(c, dev, **more)
    want, bound = c.exact()
    for n in want:
        held(got[n], want[n], bound[n], n)
    from e2_tts_pytorch_amd import ops
    a, kw = c.args(dev)
    plain = ops.packed_attn_fwd(*a, **{**kw, **more})         # the inference form keeps nothing for a backward and rounds its probabilities once
    held(plain, want['out'], bound['out'], 'out (inference)')
    return got


BIASES = ['none', 'alibi', 'table']


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('mask', ['full', 'causal', 'prefix'])
@pytest.mark.parametrize('cap', [0., 20.])
def test_packed_attention(dev, landing, mask, bias, cap):
    """documents of one token, odd lengths, across tile borders, an empty one"""
    lens = [1, 37, 0, 70, 150] if gpu_shapes(dev) else [1, 37, 0, 70]
    check(Case(lens, mask=mask, prefix=[1, 5, 0, 40, 64][:len(lens)], bias=bias, cap=cap), dev)


@pytest.mark.parametrize('bias', BIASES)
def test_packed_attention_grouped_heads(dev, bias):
    check(Case([33, 65], H=4, Hkv=2, mask='causal', bias=bias, cap=30. if bias == 'alibi' else 0.), dev)
    check(Case([40], H=3, Hkv=1, bias=bias), dev)


@pytest.mark.parametrize('mask', ['full', 'causal', 'prefix'])
def test_packed_attention_other_keys(dev, mask):
    """fewer queries than keys (a prompt behind a cache), more (rows whose mask leaves nothing), none on either side"""
    check(Case([5, 40, 3, 0, 20], kl=[69, 8, 0, 12, 20], mask=mask, prefix=[0, 2, 0, 1, 30], bias='alibi'), dev)
    c = Case([40], kl=[8], mask='causal')
    got = check(c, dev)
    assert (got['out'][:32] == 0).all() and (got['dq'][:32] == 0).all()


def test_packed_attention_capped_far(dev):
    """scores far into the cap (the exp2 form of the tanh) and beside its border"""
    check(Case([50], cap=4., gain=6.), dev)
    check(Case([50], cap=12., gain=2., bias='table', reach=5, buckets=4), dev)


@pytest.mark.parametrize('reach', [3, 24, 128, 130, 512])
def test_packed_attention_table_reach(dev, reach):
    n = 200 if gpu_shapes(dev) else 100
    check(Case([n, 17], H=2, bias='table', reach=reach, buckets=4), dev)


def test_packed_attention_slots(dev):
    """documents shorter than their slots, rows behind the last document: outputs there are zero, or left alone in the caller's own buffer; what lies
    there (NaN, inf) reaches nobody"""
    from e2_tts_pytorch_amd import ops
    c = Case([48, 40, 8, 33], kl=[64, 40, 8, 40], nq=[37, 40, 0, 33], nk=[64, 33, 8, 40], tail=5, bias='table', mask='causal')
    want, bound = c.exact()
    for t, slots, n in ((c.q, c.ql, c.nq), (c.dout, c.ql, c.nq), (c.k, c.kl, c.nk), (c.v, c.kl, c.nk)):
        at = offsets(slots).tolist()
        for d in range(len(n)):
            t[at[d] + n[d]:at[d + 1]] = float('nan') if d % 2 else float('inf')
        t[at[-1]:] = float('nan')
    got = run(c, dev)
    for n in want:
        held(got[n], want[n], bound[n], n)
    a, kw = c.args(dev)
    buf = torch.full((c.q.shape[0], c.H, 64), 7., dtype=bf16, device=dev)
    out = ops.packed_attn_fwd(*a, out=buf, **kw)
    assert out is buf
    rows = torch.zeros(c.q.shape[0], dtype=torch.bool)
    for d, s in enumerate(offsets(c.ql).tolist()[:-1]):
        rows[s:s + c.nq[d]] = True
    assert (buf.cpu()[~rows] == 7.).all()
    held(buf.cpu()[rows], want['out'][rows], bound['out'][rows], 'out')


def test_packed_attention_masking_biases(dev):
    """biases of -inf and of fp32's lowest value hide their keys; a row whose keys are all hidden is empty"""
    from e2_tts_pytorch_amd import ops
    for low in (-math.inf, torch.finfo(f32).min):
        c = Case([45], bias='table', buckets=8, reach=24, mask='causal', causal_map=True)
        c.table[0] = low                                    # distance 0: nobody sees itself; the first query sees nobody
        got = run(c, dev)
        c.table[0] = -math.inf
        want, bound = c.exact()
        for n in ('out', 'dq', 'dk', 'dv'):
            held(got[n], want[n], bound[n].nan_to_num(nan=0., posinf=0.) + 1e-2 * want[n].abs() + 1e-3, n)
        assert (got['out'][0] == 0).all() and (got['dq'][0] == 0).all() and (got['dtable'][0] == 0).all()


def test_packed_attention_strides(dev):
    """q, k, v as columns of one projection, an output and a dout with strides of their own, an expanded dout"""
    from e2_tts_pytorch_amd import ops
    c = Case([37, 20], H=2, Hkv=2, bias='alibi')
    want, bound = c.exact()
    a, kw = c.args(dev)
    T = c.q.shape[0]
    qkv = torch.stack([c.q, c.k, c.v], 1).reshape(T, 3 * 2 * 64).to(dev)
    wide = torch.zeros(T, 3 * 2 * 64 + 24, dtype=bf16, device=dev)
    wide[:, :3 * 2 * 64] = qkv
    q, k, v = (wide[:, i * 128:(i + 1) * 128].view(T, 2, 64) for i in range(3))
    buf = torch.zeros(2, T, 64, dtype=bf16, device=dev)                    # head-major
    out, st = ops.packed_attn_fwd(q, k, v, a[3], out=buf.transpose(0, 1), train=True, **kw)
    held(out, want['out'], bound['out'], 'out')
    dq, dk, dv, _ = ops.packed_attn_bwd(st, c.dout.to(dev).transpose(0, 1).contiguous().transpose(0, 1))
    for n, t in (('dq', dq), ('dk', dk), ('dv', dv)):
        held(t, want[n], bound[n], n)
    one = ops.packed_attn_bwd(st, torch.ones((), dtype=bf16, device=dev).expand(T, 2, 64))
    two = ops.packed_attn_bwd(st, torch.ones(T, 2, 64, dtype=bf16, device=dev))
    assert all(torch.equal(x, y) for x, y in zip(one[:3], two[:3]))
    odd = torch.zeros(T, 2 * 64 + 3, dtype=bf16, device=dev)[:, 3:].view(T, 2, 64)          # rows that are not 16-byte aligned are copied
    odd.copy_(q)
    assert torch.equal(ops.packed_attn_fwd(odd, k, v, a[3], **kw), ops.packed_attn_fwd(q, k, v, a[3], **kw))


def test_packed_attention_hints(dev):
    """the sizing hints change nothing but the grid: too small, exact, none"""
    c = Case([150, 30], kl=[140, 160], bias='table', mask='causal')
    base = run(c, dev)
    for mq, mk in ((1, 1), (128, 128), (150, 160), (10 ** 6, 10 ** 6)):
        got = run(c, dev, max_q=mq, max_k=mk)
        for n in ('out', 'dq', 'dk', 'dv'):
            assert torch.equal(base[n], got[n]), (n, mq)
        assert torch.allclose(base['dtable'], got['dtable'], rtol=0, atol=2e-5 * base['dtable'].abs().max().item() + 1e-5)      # other partial sums
    assert all(torch.equal(base[n], run(c, dev)[n]) for n in base)                   # the same call twice: the same bits


def test_packed_attention_table_gradient_accumulates(dev):
    from e2_tts_pytorch_amd import ops
    c = Case([60, 9], bias='table')
    a, kw = c.args(dev)
    out, st = ops.packed_attn_fwd(*a, train=True, **kw)
    fresh = ops.packed_attn_bwd(st, c.dout.to(dev))[3]
    start = torch.randn_like(fresh)
    buf = start.clone()
    assert ops.packed_attn_bwd(st, c.dout.to(dev), dtable=buf)[3] is buf
    assert torch.equal(buf, start + fresh)
    assert ops.packed_attn_bwd(st, c.dout.to(dev), need_table=False)[3] is None
    with pytest.raises(ops.E2KError):
        ops.packed_attn_bwd(st, c.dout.to(dev), dtable=buf, need_table=False)


def test_packed_attention_table_gradient_against_differences(emu):
    """differences of the 64-bit loss in the table's entries: the gradient's formula, without its code"""
    c = Case([30], bias='table', buckets=4, reach=6, H=1)
    got = run(c, 'cpu')['dtable'].to(f64)
    do = c.dout.to(f64)
    h = 2. ** -6
    for b in range(4):
        old = c.table[b, 0].item()
        c.table[b, 0] = old + h
        up = (c.exact()[0]['out'] * do).sum()
        c.table[b, 0] = old - h
        down = (c.exact()[0]['out'] * do).sum()
        c.table[b, 0] = old
        # truncation h^2 / 6 of the third derivative, which is at most a few times the sum of |dO.v| p: 30 rows x 8 x 4e-5 < 2e-2
        assert abs((up - down) / (2 * h) - got[b, 0]) < 2e-2 + 1e-3 * abs(got[b, 0])


def test_rel_buckets():
    from e2_tts_pytorch_amd import ops
    m = ops.rel_buckets(32, 128)
    assert m.numel() == 257 and m[128] == 0 and m[128 - 7] == 7 and m[128 + 7] == 23 and m[0] == 15 and m[256] == 31
    # the borders of the logarithmic buckets lie where 8 (128 / 8)^(j / 8) does: 8, 11.3, 16, 22.6, 32, 45.3, 64, 90.5
    assert [int((m[:129].flip(0) == b).nonzero()[0]) for b in range(8, 16)] == [8, 12, 16, 23, 32, 46, 64, 91]
    c = ops.rel_buckets(16, 100, causal=True)
    assert (c[100:] == 0).all() and c[0] == 15 and sorted(set(c.tolist())) == list(range(16))
    for bad in ((2, 128), (32, 8), (32, 513)):
        with pytest.raises(ops.E2KError):
            ops.rel_buckets(*bad)


def test_packed_attention_no_rows(dev):
    from e2_tts_pytorch_amd import ops
    z = lambda *s: torch.zeros(*s, dtype=bf16, device=dev)  # noqa: E731
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    assert ops.packed_attn_fwd(z(0, 2, 64), z(0, 2, 64), z(0, 2, 64), cu(0)).shape == (0, 2, 64)
    out, st = ops.packed_attn_fwd(z(3, 2, 64) + 1, z(0, 2, 64), z(0, 2, 64), cu(0, 3), cu(0, 0), train=True)
    assert (out == 0).all()
    assert all((t == 0).all() for t in ops.packed_attn_bwd(st, z(3, 2, 64) + 1)[:3])
    out, st = ops.packed_attn_fwd(z(0, 2, 64), z(5, 2, 64) + 1, z(5, 2, 64) + 1, cu(0, 0), cu(0, 5), train=True)
    assert out.numel() == 0 and all((t == 0).all() for t in ops.packed_attn_bwd(st, z(0, 2, 64))[:3])
    out = ops.packed_attn_fwd(z(3, 2, 64) + 1, z(3, 2, 64), z(3, 2, 64), cu(0))        # no document at all: zeros
    assert (out == 0).all()


def test_packed_attention_bad_offsets(dev):
    """offsets outside the tensors are cut off: nothing is read or written out of range, and the documents inside are right"""
    from e2_tts_pytorch_amd import ops
    c = Case([30, 20])
    a, kw = c.args(dev)
    good = ops.packed_attn_fwd(*a, **kw)
    big = torch.tensor([0, 30, 10 ** 9], dtype=torch.int32, device=dev)
    assert torch.equal(ops.packed_attn_fwd(a[0], a[1], a[2], big, big, **kw), good)
    low = torch.tensor([-5, 30, 50], dtype=torch.int32, device=dev)
    assert torch.equal(ops.packed_attn_fwd(a[0], a[1], a[2], low, low, **kw), good)


def test_packed_attention_refusals(emu):
    from e2_tts_pytorch_amd import ops
    c = Case([10, 6], bias='table')
    (q, k, v, cu, _), kw = c.args('cpu')
    f = ops.packed_attn_fwd
    out, st = f(q, k, v, cu, train=True, **kw)
    no = dict(scale=0.125)
    bad = [
        lambda: f(q.float(), k, v, cu), lambda: f(q[..., :32], k, v, cu), lambda: f(q, k, v[:8], cu), lambda: f(q, k[:, :1].expand(16, 3, 64), v, cu),
        lambda: f(torch.cat([q, q], 1)[:, :3], k, v, cu), lambda: f(q, k, v, cu.long()), lambda: f(q, k, v, cu[None]), lambda: f(q, k, v, cu, cu[:2]),
        lambda: f(q[:4], k, v, cu), lambda: f(q, k, v, cu, len_q=cu), lambda: f(q, k, v, cu, prefix=cu[:2]), lambda: f(q, k, v, cu, scale=0.),
        lambda: f(q, k, v, cu, scale=float('nan')), lambda: f(q, k, v, cu, softcap=-1.), lambda: f(q, k, v, cu, slopes=torch.ones(2), **{n: kw[n] for n in ('table', 'buckets')}),
        lambda: f(q, k, v, cu, slopes=torch.ones(3)), lambda: f(q, k, v, cu, table=kw['table']), lambda: f(q, k, v, cu, buckets=kw['buckets']),
        lambda: f(q, k, v, cu, table=kw['table'].to(bf16), buckets=kw['buckets']), lambda: f(q, k, v, cu, table=kw['table'], buckets=kw['buckets'][:-1]),
        lambda: f(q, k, v, cu, table=kw['table'], buckets=torch.zeros(1027, dtype=torch.int32)), lambda: f(q, k, v, cu, out=torch.zeros(16, 2, 64)),
        lambda: f(q, k, v, cu, out=torch.zeros(16, 1, 64, dtype=bf16).expand(16, 2, 64)), lambda: f(q, k, v, cu, max_q=-1),
        lambda: f(q, k, v, cu, out=torch.zeros(16 * 2 * 64 + 1, dtype=bf16)[1:].view(16, 2, 64)),
        lambda: ops.packed_attn_bwd(st, c.dout[:4]), lambda: ops.packed_attn_bwd(st, c.dout, dtable=torch.zeros(3, 2)),
        lambda: ops.packed_attn_bwd(f(q, k, v, cu, train=True, **no)[1], c.dout, dtable=torch.zeros(8, 2)),
    ]
    for i, g in enumerate(bad):
        with pytest.raises(ops.E2KError):
            g()
            print('not refused:', i)


@pytest.mark.gpu
@pytest.mark.parametrize('c', [dict(ql=[700, 1056, 33], H=4, bias='table', buckets=32, reach=128), dict(ql=[900], H=8, Hkv=2, mask='causal', cap=50., bias='alibi'),
                               dict(ql=[513, 600], kl=[2000, 600], H=4, mask='prefix', prefix=[77, 300], cap=30., bias='table', buckets=16, reach=200),
                               dict(ql=[1300], H=2)], ids=['table', 'causal', 'prefix', 'plain'])
def test_packed_attention_large(c):
    from e2_tts_pytorch_amd import _lib
    from emu.install import install
    install(None, False)
    _lib.get()
    check(Case(**c), 'cuda')


# ------------------------------------------------------------------------------------------------ one query token per sequence

def decode_case(lens, cap_n, H=4, Hkv=None, cap=0., bias='none', buckets=8, reach=24, seed=0, gain=1.5):
    """-> (q, k, v, lens, keyword arguments), exact output and its error bound: each sequence is a one-query document over its cached keys"""
    Hkv = Hkv or H
    B = len(lens)
    c = Case([1] * B, kl=[cap_n] * B, H=H, Hkv=Hkv, mask='causal', cap=cap, bias=bias, buckets=buckets, reach=reach, seed=seed, gain=gain,
             nk=[min(max(n, 0), cap_n) for n in lens])
    want, bound = c.exact()
    # two further roundings-free joins (waves, workgroups) of fp32 partial sums: 2 x 128 additions at most, far below the probabilities' bf16 rounding
    return c, want['out'], bound['out'] * (1 + 256 * U / HALF)


def decode(c, lens, cap_n, dev, **more):
    from e2_tts_pytorch_amd import ops
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    B = len(lens)
    k, v = (t.view(B, cap_n, c.Hkv, 64).clone() for t in (c.k, c.v))
    for b, n in enumerate(lens):                 # what lies behind a sequence's keys is never read
        k[b, max(n, 0):], v[b, max(n, 0):] = float('nan'), float('inf')
    kw = dict(softcap=c.cap, slopes=to(c.slopes), table=to(c.table), buckets=to(c.map))
    kw.update(more)
    return ops.attn_decode(c.q.to(dev), k.to(dev), v.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), **kw)


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('cap', [0., 20.])
def test_attn_decode(dev, landing, bias, cap):
    lens, cap_n = [1, 33, 0, 200, 150, 64], 200
    c, want, bound = decode_case(lens, cap_n, cap=cap, bias=bias)
    held(decode(c, lens, cap_n, dev), want, bound, 'out')


def test_attn_decode_grouped_heads(dev):
    for H, Hkv in ((4, 2), (3, 1), (40, 1)):                     # (more query heads than an MFMA has columns: two passes over the keys)
        c, want, bound = decode_case([70, 40], 80, H=H, Hkv=Hkv, bias='alibi')
        held(decode(c, [70, 40], 80, dev), want, bound, 'out')


def test_attn_decode_cut_lengths(dev):
    """lengths outside 0 .. capacity are cut off"""
    c, want, bound = decode_case([-3, 10 ** 6], 50)
    held(decode(c, [-3, 10 ** 6], 50, dev), want, bound, 'out')


def test_attn_decode_strides(dev):
    """a head-major cache, a slice of a longer one, strided q and out"""
    from e2_tts_pytorch_amd import ops
    lens, n = [50, 61], 64
    c, want, bound = decode_case(lens, n, H=2)
    B = 2
    k, v = (t.view(B, n, 2, 64) for t in (c.k, c.v))
    kh = k.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    vl = torch.full((B, 3 * n, 2, 64), float('nan'), dtype=bf16, device=dev)
    vl[:, n:2 * n] = v.to(dev)
    L = torch.tensor(lens, dtype=torch.int32, device=dev)
    buf = torch.full((B, 3, 64), 7., dtype=bf16, device=dev)
    qs = torch.zeros(B, 2, 3, 64, dtype=bf16, device=dev)[:, :, 1]
    qs.copy_(c.q)
    out = ops.attn_decode(qs, kh, vl[:, n:2 * n], L, out=buf[:, 1:])
    held(out, want, bound, 'out')
    assert (buf[:, 0] == 7.).all()


def test_attn_decode_matches_packed(dev):
    """the same scores as a packed call with one query per document"""
    from e2_tts_pytorch_amd import ops
    lens, n = [90, 13], 96
    c, want, bound = decode_case(lens, n, bias='table', cap=25.)
    a, kw = c.args(dev)
    held(ops.packed_attn_fwd(*a, **kw), want, bound, 'packed')
    held(decode(c, lens, n, dev), want, bound, 'decode')


def test_attn_decode_refusals(emu):
    from e2_tts_pytorch_amd import ops
    q, k, L = torch.zeros(2, 4, 64, dtype=bf16), torch.zeros(2, 8, 2, 64, dtype=bf16), torch.ones(2, dtype=torch.int32)
    f = ops.attn_decode
    assert f(q, k, k, L).shape == (2, 4, 64)
    assert f(q[:0], k[:0], k[:0], L[:0]).shape == (0, 4, 64)
    bad = [lambda: f(q.float(), k, k, L), lambda: f(q, k[:1], k[:1], L), lambda: f(q, k, k[:, :4], L), lambda: f(q, k[..., :32], k[..., :32], L),
           lambda: f(q[:, :3], k, k, L), lambda: f(q, k, k, L.long()), lambda: f(q, k, k, L[:1]), lambda: f(q, k.transpose(2, 3), k.transpose(2, 3), L),
           lambda: f(q, torch.zeros(2 * 8 * 2 * 64 + 1, dtype=bf16)[1:].view(2, 8, 2, 64), k, L), lambda: f(q, k, k, L, softcap=-1.),
           lambda: f(q, k, k, L, slopes=torch.ones(2)), lambda: f(q, k, k, L, out=torch.zeros(2, 4, 64)), lambda: f(q, k.float(), k.float(), L)]
    for i, g in enumerate(bad):
        with pytest.raises(ops.E2KError):
            g()
            print('not refused:', i)


@pytest.mark.gpu
@pytest.mark.parametrize('lens,n,kw', [([4128, 2000, 1, 3333], 4128, dict(H=16, bias='table', buckets=32, reach=128)),
                                       ([30000, 17], 30011, dict(H=8, Hkv=2, bias='alibi', cap=50.)), ([640], 640, dict(H=16))], ids=['batch', 'long', 'one'])
def test_attn_decode_large(lens, n, kw):
    from e2_tts_pytorch_amd import _lib
    from emu.install import install
    install(None, False)
    _lib.get()
    c, want, bound = decode_case(lens, n, **kw)
    out = decode(c, lens, n, 'cuda')
    held(out, want, bound, 'out')
    assert torch.equal(out, decode(c, lens, n, 'cuda'))


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('mask', ['full', 'causal'])
def test_packed_attention_split_sweep(dev, mask, bias):
    """few key heads, long sweeps: dK / dV in parts (the borders of the parts lie inside a head's tiles), gaps between the documents left zero"""
    from e2_tts_pytorch_amd import _lib
    c = Case([600, 100], kl=[70, 100], H=3 if dev == 'cpu' else 6, Hkv=1, nq=[513, 100], nk=[65, 100], mask=mask, bias=bias, tail=4)
    assert _lib.get().e2k_query_packed_attn_bwd_ws_floats(2, c.q.shape[0], c.k.shape[0], c.H, 1, 600, 0, 0) > 0
    got = check(c, dev, max_q=600)
    assert (got['dk'][65:70] == 0).all() and (got['dv'][170:] == 0).all()
    again = run(c, dev, max_q=600)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('mask', ['full', 'causal'])
def test_packed_attention_split_keys(dev, mask, bias):
    """inference with few queries over many keys: a row's keys in parts, some of them empty; queries that see nothing; gaps between the documents"""
    from e2_tts_pytorch_amd import _lib, ops
    c = Case([70, 8, 10], kl=[700, 3, 40], H=2, nq=[65, 8, 10], nk=[650, 3, 40], mask=mask, bias=bias, cap=20., tail=3)
    assert _lib.get().e2k_query_packed_attn_fwd_ws_floats(c.q.shape[0], c.k.shape[0], c.H, 700) > 0
    want, bound = c.exact()
    a, kw = c.args(dev)
    out = ops.packed_attn_fwd(*a, max_k=700, **kw)
    held(out, want['out'], bound['out'], 'out')
    assert (out[65:70] == 0).all() and (out[88:] == 0).all() and (mask == 'full' or (out[70:75] == 0).all())
    assert torch.equal(out, ops.packed_attn_fwd(*a, max_k=700, **kw))
    buf = torch.full((c.q.shape[0], 2, 64), 7., dtype=bf16, device=dev)
    ops.packed_attn_fwd(*a, max_k=700, out=buf, **kw)
    assert (buf[65:70] == 7).all() and (buf[88:] == 7).all() and torch.equal(buf[:65], out[:65])


def test_packed_attention_many_documents(dev):
    """more documents x heads than the grid has tiles for: a workgroup takes several tiles of its document (the sums by distance too)"""
    from e2_tts_pytorch_amd import _lib, ops
    n = 70000 if gpu_shapes(dev) else 9000
    lens = [0] * n
    lens[5], lens[n - 3] = 300, 40
    H = 2 if gpu_shapes(dev) else 16
    c = Case([300, 40], H=H, bias='table')
    want, bound = c.exact()
    a, kw = c.args(dev)
    cu = torch.zeros(n + 1, dtype=torch.int32)
    cu[6:], cu[n - 2:] = 300, 340
    cu = cu.to(dev)
    out, st = ops.packed_attn_fwd(a[0], a[1], a[2], cu, train=True, **kw)
    dq, dk, dv, dtable = ops.packed_attn_bwd(st, c.dout.to(dev))
    for name, t in (('out', out), ('dq', dq), ('dk', dk), ('dv', dv), ('dtable', dtable)):
        held(t, want[name], bound[name], name)


def test_packed_attention_longest_first(dev):
    """more workgroups than slots: documents are taken by length (ties, empty ones, 64 and 65 of them); heads in eights and not"""
    for lens, H in (([40, 0, 70, 40, 130, 1], 8), ([3] * 63 + [50], 1), ([2] * 64 + [33], 1), ([5, 90, 5], 3)):
        c = Case(lens, H=H, bias='table', mask='causal')
        base = run(c, dev)                                   # (no hint: the grid is sized for the total, most of it empty)
        want, bound = c.exact()
        for n in want:
            held(base[n], want[n], bound[n], n)
        big = run(c, dev, max_q=100 * 128, max_k=100 * 128)
        assert all(torch.equal(base[n], big[n]) for n in ('out', 'dq', 'dk', 'dv'))
