"""What a training forward of packed attention hands to its backward (output and what rounding cut off it, log-sum-exps), and the gradients of q and k that
rest on it, held to the bits they are kept in: bounds far below the bf16 rounding of the output itself.  Peaked rows above all: one probability near 1, whose
own rounding is then the row sum's."""
import math

import pytest
import torch

from conftest import gpu_shapes
from test_packed_attn import BIASES, HALF, U, Case, held

bf16, f32, f64 = torch.bfloat16, torch.float32, torch.float64
TWO = 2. ** -16                       # what two bf16 terms leave of a value


def sharp(c):
    """-> (values, bounds) of out + lo (Tq,H,64), lse2 (H,Tq), dq, dk in 64 bits; documents as wide as their slots, every row sees something"""
    H, G = c.H, c.H // c.Hkv
    q, k, v, do = (t.to(f64) for t in (c.q, c.k, c.v, c.dout))
    r = dict(out=torch.zeros_like(q), lse2=torch.zeros(H, q.shape[0], dtype=f64), dq=torch.zeros_like(q), dk=torch.zeros_like(k))
    b = {n: torch.zeros_like(t) for n, t in r.items()}
    q0 = k0 = 0
    for nq, nk in zip(c.ql, c.kl):
        A, B = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        rel = torch.arange(nk)[None] - (torch.arange(nq)[:, None] + nk - nq)
        see = torch.ones(nq, nk, dtype=torch.bool) if c.mask == 'full' else rel <= 0
        for h in range(H):
            Q, K, V, dO = q[A, h], k[B, h // G], v[B, h // G], do[A, h]
            z = Q @ K.t() * c.scale
            th = torch.tanh(z / c.cap) if c.cap else torch.zeros_like(z)
            bias = torch.zeros_like(z)
            if c.slopes is not None:
                bias = -c.slopes[h].to(f64) * rel.abs()
            if c.table is not None:
                bias = c.table[:, h].to(f64)[c.map.long()[rel.clamp(-c.reach, c.reach) + c.reach]]
            t = ((c.cap * th if c.cap else z) + bias).masked_fill(~see, -math.inf)
            lse = t.logsumexp(1, keepdim=True)
            p = (t - lse).exp()
            # a score: 64 products in fp32; the tanh (three-term polynomial up to 0.3: 1.2e-6 of the product, beyond it 2^-22 of the cap); the bias, the
            # reference point (at most 2^60 from the row's sum: 42) and the argument they end in
            et = 64 * U * (Q.abs() @ K.abs().t()) * c.scale + (1.2e-6 * z.abs() + 4 * U * c.cap if c.cap else 0.)
            et = torch.where(see, et + 8 * U * (t.abs().nan_to_num(posinf=0.) + bias.abs() + lse.abs() + 42), torch.zeros_like(z))
            # a row's sum: nk / 4 additions one after the other in each of four accumulators, exp2, the join; a product's accumulator: nk / 16 + 64
            es = (p * et).sum(1, keepdim=True) + (nk / 4 + 16) * U
            ep = et + es
            o = p @ V
            r['out'][A, h], b['out'][A, h] = o, TWO * o.abs() + (p * (TWO + ep + (nk / 16 + 64) * U)) @ V.abs()
            r['lse2'][h, A] = lse[:, 0] / math.log(2.)
            b['lse2'][h, A] = (es[:, 0] + 8 * U * (lse[:, 0].abs() + 42)) / math.log(2.)
            dP, dl = dO @ V.t(), (dO * o).sum(1, keepdim=True)
            edl = (dO.abs() * b['out'][A, h]).sum(1, keepdim=True)
            eds = p * (ep * (dP - dl).abs() + 64 * U * (dO.abs() @ V.abs().t() + (dO * o).abs().sum(1, keepdim=True)) + edl)
            dz = p * (dP - dl) * (1 - th * th) * c.scale
            edz = (eds * (1 - th * th) + (p * (dP - dl)).abs() * (4 * U + (2 * et / c.cap if c.cap else 0.))) * c.scale
            edz = edz + HALF * (dz.abs() + edz)                       # dS is one bf16 term
            r['dq'][A, h], b['dq'][A, h] = dz @ K, edz @ K.abs() + HALF * (dz @ K).abs()
            r['dk'][B, h // G] += dz.t() @ Q
            b['dk'][B, h // G] += edz.t() @ Q.abs()
    b['dk'] += HALF * r['dk'].abs()
    return r, b


def check(c, dev):
    from e2_tts_pytorch_amd import ops
    a, kw = c.args(dev)
    out, st = ops.packed_attn_fwd(*a, train=True, **kw)
    dq, dk, _, _ = ops.packed_attn_bwd(st, c.dout.to(dev))
    want, bound = sharp(c)
    got = dict(out=st.out.cpu().to(f64) + st.lo.cpu().to(f64), lse2=st.lse2, dq=dq, dk=dk)
    for n in want:
        held(got[n], want[n], bound[n], n)


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('mask', ['full', 'causal'])
@pytest.mark.parametrize('cap', [0., 30.])
def test_training_forward_keeps_its_bits(dev, mask, bias, cap):
    lens = [300, 65] if gpu_shapes(dev) else [100, 33]
    check(Case(lens, mask=mask, bias=bias, cap=cap), dev)


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('gain', [12., 48.])
def test_training_forward_of_steep_scores(dev, bias, gain):
    check(Case([256 if gpu_shapes(dev) else 128], gain=gain, bias=bias, seed=1), dev)


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('cap', [0., 50.])
def test_training_forward_of_one_dominating_key(dev, bias, cap):
    """every query points at one key of a later block than its row's first: its probability is all but 1, and the exact gradient of q all but 0"""
    c = Case([128], bias=bias, cap=cap, seed=2)
    at = torch.randint(70, 128, (128,), generator=torch.Generator().manual_seed(3))
    c.q = (c.k[at].to(f32) * torch.linspace(2.3, 3.3, 128)[:, None, None]).to(bf16)
    check(c, dev)


def test_training_forward_grouped_heads(dev):
    check(Case([90], H=4, Hkv=2, mask='causal', bias='alibi', gain=8.), dev)


@pytest.mark.parametrize('bias', BIASES)
@pytest.mark.parametrize('cap', [1e-3, 1e-9, 1e-20, 1e-28, 1e29])
def test_caps_far_from_the_scores(dev, bias, cap):
    """a cap of next to nothing leaves the bias alone, one far above every score changes nothing; whole blocks of scores that are exactly zero among them"""
    from e2_tts_pytorch_amd import ops
    c = Case([70, 9], cap=cap, bias=bias)
    c.q[:64] = 0
    want, _ = c.exact()
    a, kw = c.args(dev)
    out, st = ops.packed_attn_fwd(*a, train=True, **kw)
    got = dict(zip(('dq', 'dk', 'dv'), ops.packed_attn_bwd(st, c.dout.to(dev)))) | dict(out=out, inference=ops.packed_attn_fwd(*a, **kw))
    kc, vc = a[1][None, :70], a[2][None, :70]
    got['decode'] = ops.attn_decode(a[0][:1], kc, vc, torch.tensor([1], dtype=torch.int32, device=dev), softcap=cap, slopes=kw['slopes'], table=kw['table'], buckets=kw['buckets'])
    want['inference'], want['decode'] = want['out'], a[2][:1].cpu().to(f64)
    for n, t in got.items():
        # P, dS, dO.o and the result are each rounded to bf16: four half steps of sums of magnitudes below 4 |v| |k| sqrt(79)
        held(t, want[n], 4 * HALF * (want[n].abs() + 1), n)


def test_caps_out_of_range_are_refused(emu):
    from e2_tts_pytorch_amd import ops
    c = Case([8])
    a, _ = c.args('cpu')
    n = torch.tensor([8], dtype=torch.int32)
    for scale, cap in ((0.125, 1e-38), (1e20, 1e-12), (0.125, 1e-42)):
        with pytest.raises(ops.E2KError):
            ops.packed_attn_fwd(*a, scale=scale, softcap=cap)
        with pytest.raises(ops.E2KError):
            ops.attn_decode(a[0][:1], a[1][None], a[2][None], n, scale=scale, softcap=cap)
