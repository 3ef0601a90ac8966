"""Rows that lie more than 2^32 elements apart: packed attention, single-token attention and layer norm read and write them like close ones."""
import pytest
import torch

from test_packed_attn import offsets

bf16, f32 = torch.bfloat16, torch.float32
FAR = (1 << 23) - 64                  # elements from row to row: the longest token stride the kernels read in place


@pytest.fixture()
def rows():
    """(620 rows, 4, 2, 64) bf16 whose rows are FAR apart: 10 GB, 5.2e9 elements"""
    from e2_tts_pytorch_amd import _lib
    from emu.install import install
    install(None, False)
    _lib.get()
    buf = torch.empty(620 * FAR, dtype=bf16, device='cuda').as_strided((620, 4, 2, 64), (FAR, 128, 64, 1))
    assert 619 * FAR > 1 << 32
    buf.copy_(torch.randn(620, 4, 2, 64, generator=torch.Generator('cuda').manual_seed(0), device='cuda'))
    yield buf
    del buf
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize('bias', ['none', 'alibi', 'table'])
def test_packed_attention_far_rows(rows, bias):
    from e2_tts_pytorch_amd import ops
    kw = {}
    if bias == 'alibi':
        kw = dict(slopes=torch.tensor([0.5, 0.1], device='cuda'))
    if bias == 'table':
        kw = dict(table=torch.randn(8, 2, generator=torch.Generator('cuda').manual_seed(1), device='cuda'), buckets=ops.rel_buckets(8, 24, device='cuda'))
    q, k, v, do = rows.unbind(1)
    near = [t.contiguous() for t in (q, k, v)]
    cu = offsets([300, 0, 310], 'cuda')                       # the last ten rows belong to nobody
    want, ws = ops.packed_attn_fwd(*near, cu, train=True, causal=True, softcap=30., **kw)
    wants = [want, *ops.packed_attn_bwd(ws, do.contiguous())]
    got, st = ops.packed_attn_fwd(q, k, v, cu, train=True, causal=True, softcap=30., **kw)
    gots = [got, *ops.packed_attn_bwd(st, do)]
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(gots, wants))
    for mask in (dict(), dict(causal=True)):
        want = ops.packed_attn_fwd(*near, cu, **kw, **mask)
        assert torch.equal(ops.packed_attn_fwd(q, k, v, cu, **kw, **mask), want)
        few = offsets([16], 'cuda'), offsets([620], 'cuda')   # in parts, written to far rows
        want = ops.packed_attn_fwd(near[0][-16:], *near[1:], *few, **kw, **mask)
        out = ops.packed_attn_fwd(q[-16:], k, v, *few, out=do[-16:], **kw, **mask)
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_attn_decode_far_rows(rows):
    from e2_tts_pytorch_amd import ops
    k, v = rows[:, 1][None], rows[:, 2][None]
    q = rows[:1, 0].contiguous()
    for n in (620, 601, 33):
        lens = torch.tensor([n], dtype=torch.int32, device='cuda')
        assert torch.equal(ops.attn_decode(q, k, v, lens), ops.attn_decode(q, k.contiguous(), v.contiguous(), lens))
    per = 310                                                 # two sequences, the second one's cache 2.6e9 elements behind the first
    kb, vb = (rows[:, i].unflatten(0, (2, per)) for i in (1, 2))
    q2, lens = rows[:2, 0].contiguous(), torch.tensor([300, 310], dtype=torch.int32, device='cuda')
    assert torch.equal(ops.attn_decode(q2, kb, vb, lens, slopes=torch.tensor([0.1, 0.], device='cuda')),
                       ops.attn_decode(q2, kb.contiguous(), vb.contiguous(), lens, slopes=torch.tensor([0.1, 0.], device='cuda')))


@pytest.mark.gpu
def test_layer_norm_far_rows(rows):
    from e2_tts_pytorch_amd import ops
    for x in (rows.flatten(1), rows.flatten(1)[:, 1:500], rows.flatten(1)[:, 3:4]):
        w, b, dy = (torch.randn(s, generator=torch.Generator('cuda').manual_seed(2), device='cuda') for s in (x.shape[1], x.shape[1], x.shape))
        outs = []
        for t in (x, x.contiguous()):
            y, m, r = ops.layernorm_fwd(t, w, b)
            outs.append([y, m, r, *ops.layernorm_bwd(dy.to(bf16), t, m, r, w)])
        assert all(torch.equal(s, t) for s, t in zip(*outs))
