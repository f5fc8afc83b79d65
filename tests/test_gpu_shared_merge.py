"""GPU: short calls of shared prefix attention, whose states the last workgroup or wave merges, give the
bits of the same call with a second launch.  Every case is one that takes a single launch."""
import pytest
import torch

from test_gpu_shared_attn import BF16, DEV, F16, Case
from test_shared_plan import launches

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,r,hq,hkv,shared,own,sink,recent,dtype", [
    # every number of rows of a sequence, one to eight states, own tokens a wave's range or a workgroup's
    (5, 5, 4, 4, 48, 0, 0, 0, F16), (1, 16, 4, 4, 1024, 500, 0, 33, BF16), (2, 8, 6, 3, 16, 200, 64, 3, F16),
    (5, 4, 24, 8, 3200, 200, 16, 0, F16), (9, 2, 9, 3, 16, 500, 16, 600, BF16), (1, 2, 32, 8, 1024, 17, 16, 64, F16),
    (2, 3, 20, 4, 1920, 1, 0, 3, BF16), (5, 2, 20, 4, 3200, 500, 16, 600, F16), (2, 2, 56, 8, 1920, 9, 16, 33, BF16),
    (5, 1, 14, 2, 1920, 500, 64, 600, F16), (5, 1, 33, 3, 1440, 9, 64, 0, F16), (2, 1, 88, 8, 0, 0, 16, 200, F16),
    (5, 1, 32, 2, 1920, 500, 0, 600, BF16), (3, 1, 48, 3, 1024, 0, 0, 33, F16)])
def test_one_launch_gives_the_bits_of_two(groups, r, hq, hkv, shared, own, sink, recent, dtype, monkeypatch):
    from heterokv import ops
    print("case: %d x %d, %d/%d heads, %d shared, %d own, %d + %d" % (groups, r, hq, hkv, shared, own, sink, recent), flush=True)
    assert launches(groups, r, hq, hkv, shared, own, sink, recent) == 1
    n = groups * r
    c = Case(70 + n, groups, r, hq, hkv, shared, [own - (i * 7) % (own + 1) if i else own for i in range(n)], sink,
             [recent - (i * 5) % (recent + 1) if i else recent for i in range(n)], dtype)
    c.check()
    lens = [torch.tensor([x if (i + j) % 4 else (x * j) // 5 for i, x in enumerate(c.lens.tolist())], dtype=torch.int32, device=DEV)
            for j in range(4)]
    counts = [None] + [torch.tensor([(i * 5 + j) * (shared // 16) // 7 for i in range(groups)], dtype=torch.int32, device=DEV)
                       for j in range(3)]
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)

    def run():
        outs = []
        for x in lens:
            for y in counts:
                ws.fill_(255)
                outs.append(c.run(int4_lens=x, shared_counts=y, workspace=ws))
        return outs

    with monkeypatch.context() as m:
        m.setattr(ops, "_arrivals", lambda *a: None)
        two = run()
    assert all(bool(torch.isfinite(t).all()) for t in two)
    for _ in range(8):
        assert all(torch.equal(a, b) for a, b in zip(run(), two))
    torch.cuda.synchronize()
    assert all(int(t.abs().sum()) == 0 for t in ops._ARRIVALS.values())
