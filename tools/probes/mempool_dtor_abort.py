"""Probe (GPU): a dead module's plan pool survives the cycle collector inside another module's recording.

`torch.cuda.MemPool.__del__` empties its pool through the allocator, which must not happen while any other pool context is open
(torch.cuda.use_mem_pool counts as a capture under way, c10/hip/HIPCachingAllocator.cpp).  A launch plan of this package records
inside `use_mem_pool`, and a plan of a dead module is cyclic garbage, i.e. its pool dies whenever Python's cycle collector happens
to run.  `backbone._PlanPool` therefore parks dying pools until no pool context is open.

One child process (a regression would end it, not its parent) forces the collector to run inside the next module's recording;
exit code 0 and 'survived' are expected.

  python tools/probes/mempool_dtor_abort.py [out.json]
"""
import json
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent.parent

PRODUCT = r'''
import gc, random, sys
sys.path[:0] = [%(pkg)r, %(root)r]
import torch
from e2_tts_pytorch_amd import Transformer, ops
random.seed(0); torch.manual_seed(0)

def steps(m, n):
    for i in range(n):
        x = torch.randn(2, 24, 256, device='cuda', requires_grad=True)
        m(x, times=torch.rand(2, device='cuda'), text_embed=torch.randn(2, 24, 128, device='cuda')).sum().backward()

gc.disable()
a = Transformer(dim=256, depth=2, heads=2, dropout=0., max_seq_len=64).cuda()
steps(a, 3)                               # first sighting, recording, replay: `a` owns a plan and its pool
assert any(not isinstance(v, str) for v in a._plans.values())
a.__dict__['_me'] = a                     # cyclic garbage: only the collector can free it
del a
b = Transformer(dim=256, depth=2, heads=2, dropout=0., max_seq_len=64).cuda()
orig = ops.begin_recording
def hooked(meta=None):
    orig(meta)
    gc.collect()                          # the collector strikes inside b's recording = inside a use_mem_pool context
ops.begin_recording = hooked
steps(b, 3)
torch.cuda.synchronize()
print('survived')
'''


def run(code):
    r = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=600)
    err = [ln for ln in r.stderr.strip().splitlines() if ln.strip()]
    key = [ln for ln in err if 'INTERNAL ASSERT' in ln or 'terminate called' in ln or 'captures_underway' in ln]
    return dict(rc=r.returncode, stdout=r.stdout.strip()[-200:], stderr_key_lines=key[:4], stderr_tail=err[-3:])


def main():
    out = dict(product=run(PRODUCT % dict(pkg=str(ROOT / 'e2-tts-pytorch_amd'), root=str(ROOT))))
    print(json.dumps(out, indent=1))
    if len(sys.argv) > 1:
        Path(sys.argv[1]).write_text(json.dumps(out, indent=1))


if __name__ == '__main__':
    main()
