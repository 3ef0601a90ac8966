"""Which memory the packed operators may share, and which tensors they take as they lie: outputs that overlap an input, tensors off the 16-byte grid, calls
with nothing on one side."""
import random

import pytest
import torch

from test_packed_attn import Case, held, offsets

bf16, f32, f64 = torch.bfloat16, torch.float32, torch.float64


def test_rows_meet():
    """against the elements' addresses, for random views of one buffer"""
    from e2_tts_pytorch_amd import ops
    rng = random.Random(0)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        views = []
        for dims in (2, rng.choice([2, 3])):
            n = [rng.randint(1, 4) for _ in range(dims)]
            st, inner = [], 4                                # nested strides, in any order of the dimensions
            for m in n:
                st.append(inner + rng.choice([0, 0, 1, 4, 8]) if rng.random() < 0.7 else 4 * rng.randint(1, 12))
                inner = max(inner, (m - 1) * st[-1] + inner)
            order = rng.sample(range(dims), dims)
            views.append(([n[i] for i in order], [st[i] for i in order], rng.randint(0, 60)))
        buf = torch.zeros(4000)
        a, b = (buf.as_strided(n + [4], st + [1], at) for n, st, at in views)
        if ops._row_dims(a) is None or ops._row_dims(b) is None:
            continue

        def cells(t):
            idx = torch.zeros(4000)
            idx.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(1.)
            return idx
        want = bool((cells(a) * cells(b)).any())
        seen[want] += 1
        assert ops._rows_meet(a, b) == want, views
    assert min(seen.values()) > 300
    assert ops._row_dims(torch.zeros(1, 4).expand(3, 4)) is None and not ops._rows_meet(torch.zeros(3, 4), torch.zeros(3, 4))


def test_packed_attention_out_beside_its_inputs(dev):
    """an `out` in the buffer of q, k and v, and q itself as `out`: the same bits as an `out` of its own"""
    from e2_tts_pytorch_amd import ops
    for kw in (dict(ql=[37, 40], H=2), dict(ql=[9, 4], kl=[700, 30], H=2)):                # (the second in parts)
        c = Case(**kw)
        a, kw = c.args(dev)
        T, S = c.q.shape[0], c.k.shape[0]
        want = ops.packed_attn_fwd(*a, **kw)
        buf = torch.zeros(max(T, S), 4, 2, 64, dtype=bf16, device=dev)
        q, k, v, out = buf[:T, 0], buf[:S, 1], buf[:S, 2], buf[:T, 3]
        q.copy_(a[0]), k.copy_(a[1]), v.copy_(a[2])
        assert torch.equal(ops.packed_attn_fwd(q, k, v, *a[3:], out=out, **kw), want)
        assert torch.equal(ops.packed_attn_fwd(q, k, v, *a[3:], out=q, **kw), want) and torch.equal(q, want)
    c = Case([1] * 3, kl=[40] * 3, H=8, Hkv=2, mask='causal')
    q, k, v = c.q.to(dev), c.k.view(3, 40, 2, 64).to(dev), c.v.view(3, 40, 2, 64).to(dev)
    n = torch.tensor([40, 7, 33], dtype=torch.int32, device=dev)
    want = ops.attn_decode(q, k, v, n)
    assert torch.equal(ops.attn_decode(q, k, v, n, out=q), want) and torch.equal(q, want)


def test_overlapping_outputs_are_refused(emu):
    from e2_tts_pytorch_amd import ops
    z = lambda *s: torch.zeros(*s, dtype=bf16)  # noqa: E731
    cu = offsets([10, 6])
    f = ops.packed_attn_fwd
    buf, wide = z(17, 3, 2, 64), z(16, 4, 64)
    q, k, v = buf[:16].unbind(1)
    two = z(2, 16, 2, 64)
    bad = [lambda: f(q, k, v, cu, out=k), lambda: f(q, k, v, cu, out=v), lambda: f(q, k, v, cu, out=buf[1:, 0]), lambda: f(q, k, v, cu, out=buf[1:, 1]),
           lambda: f(q, k, v, cu, out=q, train=True), lambda: f(wide[:, :2], k, v, cu, out=wide[:, 1:3]), lambda: f(q, wide[:, :2], v, cu, out=wide[:, 1:3]),
           lambda: f(two[0].reshape(2, 16, 64).transpose(0, 1), k, v, cu, out=two[0]), lambda: f(q, k, v, cu, out=z(40, 64).as_strided((16, 2, 64), (128, 128, 1))),
           lambda: f(q, k, v, cu, out=z(40, 64).as_strided((16, 2, 64), (128, 64, 1), 64).as_strided((16, 2, 64), (128, 192, 1)))]
    bad += [lambda: f(q, q, v, cu, out=q), lambda: f(q, k, q, cu, out=q), lambda: f(q, q, q, cu, out=q)]             # (q is k or v too)
    kc, L = z(3, 8, 2, 64), torch.ones(3, dtype=torch.int32)
    d, qs = ops.attn_decode, z(4, 2, 64)
    bad += [lambda: d(qs[:3], kc, kc.clone(), L, out=kc[:, 3]), lambda: d(qs[:3], kc.clone(), kc, L, out=kc[:, 7]), lambda: d(qs[:3], kc, kc, L, out=qs[1:]),
            lambda: d(qs[:3], kc, kc, L, out=z(9, 64).as_strided((3, 2, 64), (64, 64, 1)))]
    for i, g in enumerate(bad):
        with pytest.raises(ops.E2KError):
            g()
            print('not refused:', i)
    assert d(qs[:3], kc, kc, L, out=z(3, 3, 64)[:, 1:]).shape == (3, 2, 64)

def test_contiguous_but_misaligned_tensors_are_copied(dev):
    """q, k, v, dout and a decode q at an odd element of a flat buffer; a single row with a stride that no row of it uses"""
    from e2_tts_pytorch_amd import ops

    def moved(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)
    c = Case([37, 20], H=2, bias='alibi')
    a, kw = c.args(dev)
    out, st = ops.packed_attn_fwd(*a, train=True, **kw)
    want = [out, *ops.packed_attn_bwd(st, c.dout.to(dev))[:3]]
    out, st = ops.packed_attn_fwd(*(moved(t) for t in a[:3]), *a[3:], train=True, **kw)
    got = [out, *ops.packed_attn_bwd(st, moved(c.dout.to(dev)))[:3]]
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(ops.packed_attn_fwd(*(moved(t) for t in a[:3]), *a[3:], **kw), ops.packed_attn_fwd(*a, **kw))
    q, k, v = a[0][:2].contiguous(), a[1][:40].view(2, 20, 2, 64), a[2][:40].view(2, 20, 2, 64)
    n = torch.tensor([20, 7], dtype=torch.int32, device=dev)
    assert torch.equal(ops.attn_decode(moved(q), k, v, n), ops.attn_decode(q, k, v, n))
    one = torch.zeros(2 * 64 + 64, dtype=bf16, device=dev).as_strided((1, 2, 64), (131, 64, 1))
    one.copy_(q[:1])
    cu = offsets([1], dev)
    assert torch.equal(ops.packed_attn_fwd(one, one, one, cu), ops.packed_attn_fwd(q[:1], q[:1], q[:1], cu))
    assert torch.equal(ops.attn_decode(one, k[:1], v[:1], n[:1]), ops.attn_decode(q[:1], k[:1], v[:1], n[:1]))


def test_backward_without_queries_checks_its_keys(emu):
    """the C entry with no query rows still writes dk and dv: pointers, strides and sizes are held to the same rules (the missing ones after the others: each
    is refused before a kernel could follow it)"""
    from e2_tts_pytorch_amd import _lib, ops
    k = torch.zeros(6, 2, 64, dtype=bf16)
    dk, dv, cu = torch.ones_like(k), torch.ones_like(k), torch.zeros(2, dtype=torch.int32)
    cuk = torch.tensor([0, 6], dtype=torch.int32)
    names = 'dO sg hg Q sq hq K sk hk V sv hv cu_q cu_k len_q len_k prefix nd Tq Tk H Hkv max_q max_k causal scale softcap slopes table buckets nbuckets reach O so ho Olo lse2 delta dQ dK dV dtable accumulate ws fill stream'.split()
    good = dict.fromkeys(names, 0) | dict.fromkeys('dO Q len_q len_k prefix slopes table buckets O Olo lse2 delta dQ dtable ws stream'.split(), None)
    good |= dict(sg=128, hg=64, sq=128, hq=64, K=k.data_ptr(), sk=128, hk=64, V=k.data_ptr(), sv=128, hv=64, cu_q=cu.data_ptr(), cu_k=cuk.data_ptr(), nd=1, Tk=6, H=2,
                 Hkv=2, scale=0.125, softcap=0., so=128, ho=64, dK=dk.data_ptr(), dV=dv.data_ptr(), fill=1)

    def call(**other):
        _lib.get().e2k_packed_attn_bwd(*(good | other).values())
    call()
    assert (dk == 0).all() and (dv == 0).all()
    for other in (dict(sk=127), dict(hv=60), dict(K=k.data_ptr() + 2), dict(scale=0.), dict(softcap=-1.), dict(H=3, Hkv=2), dict(nd=-1), dict(cu_q=None), dict(cu_k=None), dict(K=None),
                  dict(V=None), dict(dK=None)):
        with pytest.raises(ops.E2KError):
            call(**other)
            print('not refused:', other)


def test_workspace_of_the_table_gradient(emu):
    """sized by the rows and documents there are: a hint that is missing costs nothing"""
    from e2_tts_pytorch_amd import _lib
    f = _lib.get().e2k_query_packed_attn_bwd_ws_floats
    for max_q in (0, 1024, 16384):
        for nd, T, H, reach in ((64, 16384, 16, 512), (128, 16384, 16, 512), (1, 16384, 16, 128), (70000, 340, 2, 128)):
            join = f(nd, T, T, H, H, max_q, 0, 0)
            assert f(nd, T, T, H, H, max_q, reach, 1) - join <= H * (T // 128 + min(nd, T) + 1) * (2 * reach + 1) + 3


@pytest.mark.parametrize('hint', [0, 130, 1])
def test_table_gradient_over_tiles_and_documents(dev, hint):
    """documents that start anywhere in a tile, empty ones, more than 64 of them, slots longer than their documents: the same sums whatever the hint (to
    their order), and the same bits twice"""
    for kw in (dict(ql=[130, 0, 126, 1, 0, 255, 128, 3]), dict(ql=[1, 0, 2] * 43 + [200]), dict(ql=[140, 300, 20], kl=[150, 290, 20], nq=[129, 130, 0], nk=[150, 3, 20])):
        c = Case(H=1, bias='table', buckets=6, reach=10, **kw)
        from test_packed_attn import run
        got = run(c, dev, max_q=hint)
        want, bound = c.exact()
        for n in want:
            held(got[n], want[n], bound[n], n)
        assert torch.equal(got['dtable'], run(c, dev, max_q=hint)['dtable'])


def test_gradient_buffers_that_share_memory_are_refused(emu):
    """a table's gradient added into the table (still read by the kernel that follows), a scale's and a shift's into one buffer"""
    from e2_tts_pytorch_amd import ops
    c = Case([10], bias='table')
    a, kw = c.args('cpu')
    out, st = ops.packed_attn_fwd(*a, train=True, **kw)
    with pytest.raises(ops.E2KError):
        ops.packed_attn_bwd(st, c.dout, dtable=kw['table'])
    x, w = torch.randn(6, 8), torch.ones(3, 8)
    y, m, r = ops.layernorm_fwd(x, w, w, 0., 2)
    both = torch.zeros(4, 2, 8)
    for dg, db in ((both[:3, 0], both[:3, 0]), (both[:3, 0], both[1:, 0]), (both.view(8, 8)[:3], both.view(8, 8)[2:5])):
        with pytest.raises(ops.E2KError):
            ops.layernorm_bwd(x, x, m, r, w, 0., 2, dg, db)
    want = ops.layernorm_bwd(x, x, m, r, w, 0., 2)
    got = ops.layernorm_bwd(x, x, m, r, w, 0., 2, both[:3, 0], both[:3, 1])
    assert all(torch.equal(s, t) for s, t in zip(got, want)) and (both[3] == 0).all()
