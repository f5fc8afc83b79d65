"""GPU: attention over a shared prefix by sequences that do not hold all of it, being shorter, or of a
group whose count is below the bound: right, and without one wave that reads a prefix alone."""
import random

import pytest
import torch

from test_gpu_shared_attn import BF16, DEV, F16, Case

pytestmark = pytest.mark.gpu


def _lens(c, r):
    """Lengths around every border: none, one token, the groups' counts, the bound, all."""
    full = [c.shared + n for n in c.own]
    counts = [r.choice([c.shared // 16, r.randrange(c.shared // 16 + 1), 0]) for _ in range(c.groups)]
    keep = []
    for b in range(c.B):
        at = 16 * counts[b // c.r]
        x = r.choice([0, 1, at - 1, at, at + 1, c.shared - 1, c.shared, r.randrange(full[b] + 1), full[b], full[b]])
        keep.append(min(max(x, 0), full[b]))
    return keep, counts


@pytest.mark.parametrize("groups,r,hq,hkv,shared,own,sink,recent,dtype", [
    # one row tile a group, of every number of rows a sequence: merged in the launch
    (2, 3, 8, 8, 96, 40, 0, 20, F16), (3, 2, 21, 3, 1008, 9, 16, 3, BF16), (2, 4, 12, 4, 336, 0, 0, 0, F16),
    (1, 2, 35, 5, 48, 600, 0, 100, F16), (4, 1, 22, 2, 160, 33, 0, 0, BF16), (1, 1, 16, 1, 512, 70, 0, 0, F16),
    # rows of a sequence in two workgroups' tiles, two to four tiles, many groups
    (1, 23, 21, 3, 400, 20, 0, 0, F16), (1, 30, 28, 4, 1600, 50, 16, 30, BF16), (2, 11, 40, 8, 736, 7, 0, 40, F16),
    (7, 9, 32, 8, 240, 30, 0, 0, F16), (1, 130, 4, 4, 64, 5, 0, 0, F16), (3, 40, 2, 1, 304, 90, 0, 0, BF16),
    # more ranges than one wave merges
    (1, 5, 16, 2, 40000, 100, 0, 0, F16), (1, 19, 8, 2, 20000, 40, 0, 33, BF16)])
def test_parity(groups, r, hq, hkv, shared, own, sink, recent, dtype):
    print("case: %d x %d, %d/%d heads, %d shared, %d own, %d + %d fp16, %s" %
          (groups, r, hq, hkv, shared, own, sink, recent, dtype), flush=True)
    n, rng = groups * r, random.Random(shared + hq)
    c = Case(60 + n, groups, r, hq, hkv, shared, [own - i % (own + 1) for i in range(n)], sink,
             [recent - i % (recent + 1) for i in range(n)], dtype)
    for step in range(4):
        keep, counts = _lens(c, rng)
        lens = torch.tensor(keep, dtype=torch.int32, device=DEV)
        print("  counts %s, lengths %s" % (counts, keep[:12]), flush=True)
        a = c.check(keep=keep, int4_lens=lens, shared_counts=torch.tensor(counts, dtype=torch.int32, device=DEV))
        assert torch.equal(a, c.run(int4_lens=lens, shared_counts=counts))
        c.check(keep=keep, int4_lens=lens)
    c.check(shared_counts=[0] * groups, int4_lens=None if own == 0 else c.lens)


def _us(f):
    for _ in range(5):
        f()
    best = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        for _ in range(4):
            f()
        b.record()
        b.synchronize()
        best.append(a.elapsed_time(b) * 250)
    return min(best)


def test_time_of_prefixes_read_alone():
    """2 x 16 sequences, 28608 shared tokens: the two prefixes are 63 MB, and one read alone is half of
    that.  One sequence that is a token short of its prefix reads 1.5 times as much, a group without
    shared blocks 8.5 times as much (more than the time of a small one grows)."""
    c = Case(61, 2, 16, 32, 8, 28608, 200, 64, [256] * 32)
    usual = _us(c.run)
    lens = c.lens.clone()
    lens[5] = c.shared - 1
    short = _us(lambda: c.run(int4_lens=lens))
    counts = torch.tensor([c.shared // 16, 0], dtype=torch.int32, device=DEV)
    alone = _us(lambda: c.run(shared_counts=counts))
    print("  %.1f us, one short %.1f us, one group of none %.1f us" % (usual, short, alone), flush=True)
    assert short <= 3 * usual and alone <= 8.5 * usual


def test_captured_and_replayed_with_other_lengths():
    c = Case(62, 2, 6, 32, 8, 960, 40, 16, [30] * 12)
    lens, counts = c.lens.clone(), torch.tensor([60, 60], dtype=torch.int32, device=DEV)
    out = torch.empty_like(c.q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out, int4_lens=lens, shared_counts=counts)
    rng = random.Random(4)
    for step in range(5):
        keep, n = _lens(c, rng)
        lens.copy_(torch.tensor(keep, dtype=torch.int32))
        counts.copy_(torch.tensor(n, dtype=torch.int32))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.check(keep=keep, int4_lens=lens, shared_counts=counts))


def test_two_graphs_of_one_workspace():
    c, d = Case(63, 1, 16, 32, 8, 3200, 50), Case(64, 2, 3, 28, 4, 640, 60, 16, [20] * 6, dtype=BF16)
    rng, ws, graphs = random.Random(5), torch.empty(64 << 20, dtype=torch.uint8, device=DEV), []
    outs = torch.empty_like(c.q), torch.empty_like(d.q)
    args = [dict(zip(("int4_lens", "shared_counts"), (torch.tensor(x, dtype=torch.int32, device=DEV) for x in _lens(y, rng)))) for y in (c, d)]
    want = [x.check(keep=a["int4_lens"].tolist(), **a) for x, a in zip((c, d), args)]
    torch.cuda.synchronize()
    for x, a, out in zip((c, d), args, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            x.run(out=out, workspace=ws, **a)
    for step in range(4):
        ws.fill_(255)
        for g in graphs if step % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        for out in outs:
            out.zero_()
